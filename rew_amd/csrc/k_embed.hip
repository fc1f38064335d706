// Embedding rows and the gradient of their table (EmbedArgs and EmbedGradArgs
// in kernels.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "rows_device.h"

namespace rew {

namespace {

constexpr int kThreads = 256;

// f(type, run length): the element type and the longest run of at most 16
// bytes that divides a row of n values.
template <class F>
void by_run(int dt, int64_t n, F&& f) {
  auto runs = [&](auto t, auto most) {
    constexpr int M = decltype(most)::value;
    if (n % M == 0) f(t, std::integral_constant<int, M>());
    else if (M == 8 && n % 4 == 0) f(t, std::integral_constant<int, 4>());
    else if (n % 2 == 0) f(t, std::integral_constant<int, 2>());
    else f(t, std::integral_constant<int, 1>());
  };
  if (dt == kF32) runs(RowF32(), std::integral_constant<int, 4>());
  else if (dt == kBF16) runs(RowBf16(), std::integral_constant<int, 8>());
  else runs(RowF16(), std::integral_constant<int, 8>());
}

// Threads side by side on a row of `runs` runs: a power of two up to kThreads.
int row_threads(int64_t runs) {
  int x = 1;
  while (x < kThreads && x < runs) x *= 2;
  return x;
}

template <class T, int N>
__global__ void __launch_bounds__(kThreads) embed_kernel(EmbedArgs a) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= a.T) return;
  const int64_t id = a.ids[t];
  const bool there = id >= 0 && id < a.V;
  const int64_t src = there ? id * a.E : 0, dst = t * a.E;
  for (int64_t c = threadIdx.x * N; c < a.E; c += (int64_t)blockDim.x * N) {
    float f[N];
    if (there) {
      run_load<T, N>(a.w, src + c, f);
#pragma unroll
      for (int x = 0; x < N; ++x) f[x] *= a.scale;
    } else {
#pragma unroll
      for (int x = 0; x < N; ++x) f[x] = 0.0f;
    }
    run_store<T, N>(a.out, dst + c, f);
  }
}

// ---- gradient -----------------------------------------------------------------------
// The tokens are sorted by id (stable, so a row's tokens keep their order), then
// each row of the table sums its own: no atomics on values, one order of sums.

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortRows = 512, kSortBits = 9;  // rows of the table per workgroup

// Tokens per part of a row that is split; a row of more is "long".
int64_t part_tokens(int64_t T) {
  return std::max<int64_t>(64, ((T + 1023) / 1024 + 63) & ~(int64_t)63);
}

struct GradWork {
  int32_t *first, *order;  // [V + 1]: a row's first place in order; [T]: tokens by row
  float* part;             // [parts][2][E]
};
__host__ __device__ inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
GradWork grad_work(const EmbedGradArgs& a) {
  GradWork w;
  uint8_t* p = (uint8_t*)a.work;
  w.first = (int32_t*)p;
  p += up256((size_t)(a.V + 1) * 4);
  w.order = (int32_t*)p;
  p += up256((size_t)a.T * 4);
  w.part = (float*)p;
  return w;
}

// Workgroup b places the tokens of rows [512 b, 512 b + 512): every wave walks
// its own sixteenth of the ids, counts (LDS atomics on counts, whose order does
// not show), and, once all counts are summed, walks it again and puts each
// token behind those of the same row before it.  Reading all ids in each of
// V / 512 workgroups costs less than the several launches of a sort by digits.
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const int32_t* ids, int64_t T,
                                                                  int64_t V, GradWork w) {
  __shared__ int32_t cnt[kSortWaves][kSortRows];
  __shared__ int32_t tmp[kSortWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t lo = (int64_t)blockIdx.x * kSortRows;
  const int rows = (int)min((int64_t)kSortRows, V - lo);
  for (int i = tid; i < kSortWaves * kSortRows; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int64_t per = ((T + kSortWaves - 1) / kSortWaves + 63) & ~(int64_t)63;
  const int64_t t0 = min((int64_t)wave * per, T), t1 = min(t0 + per, T);
  int32_t below = 0;
  for (int64_t t = t0 + lane; t < t1; t += 64) {
    const int64_t r = ids[t] - lo;
    if (ids[t] >= 0 && r < 0) ++below;
    else if (r >= 0 && r < rows) atomicAdd(&cnt[wave][r], 1);
  }
  // the tokens of the rows before: this workgroup's first place
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) tmp[wave] = below;
  __syncthreads();
  int32_t base = 0;
#pragma unroll
  for (int i = 0; i < kSortWaves; ++i) base += tmp[i];
  __syncthreads();
  // row r of thread r: the waves' counts become offsets within the row
  int32_t total = 0;
  if (tid < kSortRows)
    for (int i = 0; i < kSortWaves; ++i) {
      const int32_t n = cnt[i][tid];
      cnt[i][tid] = total;
      total += n;
    }
  int32_t sum = total;  // inclusive over the rows
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 63) tmp[wave] = sum;
  __syncthreads();
  int32_t at = base + sum - total;
  for (int i = 0; i < wave; ++i) at += tmp[i];
  if (tid < kSortRows) {
    for (int i = 0; i < kSortWaves; ++i) cnt[i][tid] += at;
    if (tid < rows) w.first[lo + tid] = at;
    if (lo + tid == V - 1) w.first[V] = at + total;
  }
  __syncthreads();
  // (a wave's lanes agree on the number of turns, for the ballots)
  for (int64_t t = t0 + lane; t - lane < t1; t += 64) {
    const int64_t r = t < t1 ? (int64_t)ids[t] - lo : -1;
    const bool mine = r >= 0 && r < rows;
    uint64_t same = __ballot(mine);
    if (same == 0) continue;
#pragma unroll
    for (int b = 0; b < kSortBits; ++b) {
      const uint64_t set = __ballot(mine && (r >> b & 1));
      same &= r >> b & 1 ? set : ~set;
    }
    if (mine) {
      const int before = __popcll(same & ((1ull << lane) - 1));
      volatile int32_t* c = &cnt[wave][r];
      const int32_t p = *c;
      w.order[p + before] = (int32_t)t;
      if (before == 0) *c = p + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Rows of at most `part` tokens (none: zeros), summed in the tokens' order.
template <class T, int N>
__global__ void __launch_bounds__(kThreads) embed_rows_kernel(EmbedGradArgs a, GradWork w,
                                                              int64_t part) {
  const int64_t v = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (v >= a.V) return;
  const int32_t p0 = w.first[v], p1 = w.first[v + 1];
  if (p1 - p0 > part) return;
  for (int64_t c = threadIdx.x * N; c < a.E; c += (int64_t)blockDim.x * N) {
    float s[N];
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] = 0.0f;
    for (int32_t p = p0; p < p1; ++p) {
      float f[N];
      run_load<T, N>(a.grad, (int64_t)w.order[p] * a.E + c, f);
#pragma unroll
      for (int x = 0; x < N; ++x) s[x] += f[x];
    }
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] *= a.scale;
    run_store<T, N>(a.out, v * a.E + c, s);
  }
}

// The long rows that places [j part, j part + part) of the order touch: at most
// the row of the first place (side 0) and that of the last (side 1, where it is
// another one), since a row between them has fewer than `part` tokens.
struct LongRow {
  int64_t row = -1;
  int32_t p0, p1;  // its places
};
__device__ __forceinline__ LongRow long_row(const EmbedGradArgs& a, const GradWork& w, int32_t p,
                                            int64_t part) {
  LongRow l;
  const int64_t v = a.ids[w.order[p]];
  l.p0 = w.first[v];
  l.p1 = w.first[v + 1];
  if (l.p1 - l.p0 > part) l.row = v;
  return l;
}

template <class T, int N>
__global__ void __launch_bounds__(kThreads) embed_part_kernel(EmbedGradArgs a, GradWork w,
                                                              int64_t part) {
  const int32_t n = w.first[a.V];
  const int64_t j = blockIdx.x;
  if (j * part >= n) return;
  const int32_t q0 = (int32_t)(j * part), q1 = (int32_t)min(j * part + part, (int64_t)n);
  const int64_t c = ((int64_t)blockIdx.y * kThreads + threadIdx.x) * N;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const LongRow l = long_row(a, w, side ? q1 - 1 : q0, part);
    if (l.row < 0 || (side && l.p0 <= q0)) continue;
    if (c >= a.E) continue;
    float s[N];
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] = 0.0f;
    for (int32_t p = max(l.p0, q0); p < min(l.p1, q1); ++p) {
      float f[N];
      run_load<T, N>(a.grad, (int64_t)w.order[p] * a.E + c, f);
#pragma unroll
      for (int x = 0; x < N; ++x) s[x] += f[x];
    }
#pragma unroll
    for (int x = 0; x < N; ++x) w.part[(j * 2 + side) * a.E + c + x] = s[x];
  }
}

// The long row that begins in part j, from its parts in order.
template <class T, int N>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(EmbedGradArgs a, GradWork w,
                                                              int64_t part) {
  const int32_t n = w.first[a.V];
  const int64_t j = blockIdx.x;
  if (j * part >= n) return;
  const int32_t q0 = (int32_t)(j * part), q1 = (int32_t)min(j * part + part, (int64_t)n);
  const LongRow l = long_row(a, w, q1 - 1, part);
  const int64_t c = ((int64_t)blockIdx.y * kThreads + threadIdx.x) * N;
  if (l.row < 0 || l.p0 < q0 || c >= a.E) return;
  float s[N];
#pragma unroll
  for (int x = 0; x < N; ++x) s[x] = w.part[(j * 2 + (l.p0 > q0)) * a.E + c + x];
  for (int64_t i = j + 1; i * part < l.p1; ++i)
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] += w.part[i * 2 * a.E + c + x];
#pragma unroll
  for (int x = 0; x < N; ++x) s[x] *= a.scale;
  run_store<T, N>(a.out, l.row * a.E + c, s);
}

}  // namespace

void launch_embed(const EmbedArgs& a, hipStream_t stream) {
  if (a.T * a.E == 0) return;
  by_run(a.dt, a.E, [&](auto t, auto n) {
    constexpr int N = decltype(n)::value;
    const int x = row_threads(a.E / N), y = kThreads / x;
    hipLaunchKernelGGL((embed_kernel<decltype(t), N>), dim3((unsigned)((a.T + y - 1) / y)),
                       dim3(x, y), 0, stream, a);
  });
  REW_HIP(hipGetLastError());
}

size_t embed_grad_ws_bytes(int64_t T, int64_t V, int64_t E) {
  const int64_t part = part_tokens(T), parts = T > part ? (T + part - 1) / part : 0;
  return up256((size_t)(V + 1) * 4) + up256((size_t)T * 4) + (size_t)parts * 2 * E * 4;
}

int launch_embed_grad(const EmbedGradArgs& a, hipStream_t stream) {
  if (a.V * a.E == 0) return 0;
  const GradWork w = grad_work(a);
  const int64_t part = part_tokens(a.T);
  hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)((a.V + kSortRows - 1) / kSortRows)),
                     dim3(kSortThreads), 0, stream, a.ids, a.T, a.V, w);
  by_run(a.dt, a.E, [&](auto t, auto n) {
    typedef decltype(t) Ty;
    constexpr int N = decltype(n)::value;
    const int x = row_threads(a.E / N), y = kThreads / x;
    hipLaunchKernelGGL((embed_rows_kernel<Ty, N>), dim3((unsigned)((a.V + y - 1) / y)),
                       dim3(x, y), 0, stream, a, w, part);
    if (a.T <= part) return;
    const dim3 grid((unsigned)((a.T + part - 1) / part),
                    (unsigned)((a.E / N + kThreads - 1) / kThreads));
    hipLaunchKernelGGL((embed_part_kernel<Ty, N>), grid, dim3(kThreads), 0, stream, a, w, part);
    hipLaunchKernelGGL((embed_join_kernel<Ty, N>), grid, dim3(kThreads), 0, stream, a, w, part);
  });
  REW_HIP(hipGetLastError());
  return a.T > part ? 4 : 2;
}

}  // namespace rew
