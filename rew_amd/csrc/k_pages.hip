// The block tables of a serving step, and the write of its keys and values
// into their pages (PageTablesArgs and PageWriteArgs in kernels.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"

namespace rew {

namespace {
constexpr int kThreads = 256;
constexpr int kResident = 256 * 8;  // workgroups of the tables kernel on 256 CUs

__device__ __forceinline__ int64_t blocks_of(int64_t n, int log_page) {
  return (n + (1ll << log_page) - 1) >> log_page;
}

// Sum of x over the workgroup, in every thread.
__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t* tmp) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = x;
  __syncthreads();
  int64_t s = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += tmp[w];
  return s;
}
}  // namespace

// Workgroup (r, y) sums the new tokens and pages of the requests before r
// itself (reading n counts costs less than a launch that scans them first)
// and writes share y of request r's table row and tokens; r = n: the totals,
// and the tokens that no request has.  1000 requests with tables of 2048
// entries: 7 us, most of it the sums (with 8 shares a request, 15 us).
__global__ void __launch_bounds__(kThreads) page_tables_kernel(PageTablesArgs a) {
  __shared__ int64_t tmp[kThreads / 64];
  const int64_t r = blockIdx.x;
  const int64_t page = 1ll << a.log_page;
  int64_t tok = 0, take = 0;
  for (int64_t i = threadIdx.x; i < r; i += kThreads) {
    const int64_t c = max(a.cached[i], 0), f = max(a.fresh[i], 0);
    tok += f;
    take += blocks_of(c + f, a.log_page) - blocks_of(c, a.log_page);
  }
  tok = block_sum(tok, tmp);
  take = block_sum(take, tmp);
  const int64_t first = blockIdx.y * kThreads + threadIdx.x, step = (int64_t)gridDim.y * kThreads;
  const int64_t start = min(tok, a.tokens);
  if (r == a.n) {
    if (first == 0) {
      a.starts[r] = (int32_t)start;
      a.taken[0] = (int32_t)min(take, (int64_t)0x7fffffff);
    }
    for (int64_t t = start + first; t < a.tokens; t += step) {
      a.slots[t] = -1;
      a.positions[t] = 0;
    }
    return;
  }
  const int64_t c = max(a.cached[r], 0), f = max(a.fresh[r], 0);
  const int64_t have = blocks_of(c, a.log_page), want = blocks_of(c + f, a.log_page);
  if (first == 0) {
    a.starts[r] = (int32_t)start;
    a.lens[r] = (int32_t)min(c + f, (int64_t)0x7fffffff);
  }
  const int32_t* row = a.table + r * a.width;
  auto entry = [&](int64_t j) -> int32_t {
    if (j < have) return row[j];
    const int64_t p = take + j - have;
    return j < want && p < a.pool_n ? a.pool[p] : -1;
  };
  for (int64_t j = first; j < a.width; j += step) a.out_table[r * a.width + j] = entry(j);
  for (int64_t i = first; i < f && tok + i < a.tokens; i += step) {
    const int64_t p = c + i, j = p >> a.log_page;
    const int32_t e = j < a.width ? entry(j) : -1;
    const int64_t slot = ((int64_t)e << a.log_page) + (p & (page - 1));
    a.slots[tok + i] = e < 0 || slot > 0x7fffffff ? -1 : (int32_t)slot;
    a.positions[tok + i] = (int32_t)p;
  }
}

void launch_page_tables(const PageTablesArgs& a, hipStream_t stream) {
  // shares per request: about one table row or token run per thread, as long as
  // all workgroups run at once (each has the same sums to do first)
  const int64_t per = std::max(a.width, a.tokens / std::max<int64_t>(a.n, 1));
  const int64_t most = std::min<int64_t>(16, kResident / (a.n + 1));
  const unsigned y = (unsigned)std::max<int64_t>(1, std::min(most, per / kThreads));
  hipLaunchKernelGGL(page_tables_kernel, dim3((unsigned)(a.n + 1), y), dim3(kThreads), 0, stream,
                     a);
  REW_HIP(hipGetLastError());
}

// A thread per 16 bytes of a token's K and V rows: as fast as a copy (8191
// tokens of 8 heads x 128: 67 MB read and written in 11.7 us, 5.7 TB/s).
__global__ void __launch_bounds__(kThreads) page_write_kernel(PageWriteArgs a, int64_t total) {
  const int per_row = a.row_bytes / 16;
  const int64_t slots = a.pages << a.log_page;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per_row;  // (token, KV head)
    const int ch = (int)(i - row * per_row);
    const int64_t t = row / a.Hkv;
    const int h = (int)(row - t * a.Hkv);
    const int64_t s = a.slots[t];
    if (s < 0 || s >= slots) continue;
    const int64_t dst = (((s >> a.log_page) * a.Hkv + h) << a.log_page) +
                        (s & ((1ll << a.log_page) - 1));
    ((uint4*)a.k_pages)[dst * per_row + ch] = ((const uint4*)a.k)[i];
    ((uint4*)a.v_pages)[dst * per_row + ch] = ((const uint4*)a.v)[i];
  }
}

void launch_page_write(const PageWriteArgs& a, hipStream_t stream) {
  const int64_t total = a.T * a.Hkv * (a.row_bytes / 16);
  if (total == 0) return;
  const int64_t blocks = std::min<int64_t>((total + kThreads - 1) / kThreads, 256 * 16);
  hipLaunchKernelGGL(page_write_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, a,
                     total);
  REW_HIP(hipGetLastError());
}

}  // namespace rew
