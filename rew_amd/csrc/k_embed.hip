// Embedding rows and the gradient of their table (EmbedArgs and EmbedGradArgs
// in kernels.h).
//
// Bound: HBM.  16384 ids of text, 128256 x 4096 bfloat16: rows in 42.5 us (54 MB of the
// table and 134 MB written, 4.4 TB/s); gradient 155 us (sort and zeros, 1.05 GB at 6.8
// TB/s) + 75 (sums) + 6 (join).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "rows_device.h"

namespace rew {

namespace {

constexpr int kThreads = 256;

// f(element type, run length) for rows of n values.
template <class F>
void by_run(int dt, int64_t n, F&& f) {
  auto with = [&](auto t) {
    constexpr int N = kRun<decltype(t)>;
    if (n >= N) f(t, std::integral_constant<int, N>());
    else f(t, std::integral_constant<int, 1>());
  };
  if (dt == kF32) with(RowF32());
  else if (dt == kBF16) with(RowBf16());
  else with(RowF16());
}

// Threads side by side on a row of `runs` runs: a power of two up to `most`.
int row_threads(int64_t runs, int most) {
  int x = 1;
  while (x < most && x < runs) x *= 2;
  return x;
}

template <class T, int N>
__global__ void __launch_bounds__(kThreads) embed_kernel(EmbedArgs a) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= a.T) return;
  const int64_t id = a.ids[t];
  const bool there = id >= 0 && id < a.V;
  const int64_t src = there ? id * a.E : 0, dst = t * a.E;
  for (int64_t i = threadIdx.x * N; i < a.E; i += (int64_t)blockDim.x * N) {
    const int64_t c = run_start(i, a.E, N);
    float f[N];
    run_load<T, N>(a.w, src + c, f);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      f[x] *= a.scale;
      // (a product by itself: with the rounding to float16 the compiler makes it
      // v_fma_mixlo f scale + 0, which turns -0 into 0)
      asm("" : "+v"(f[x]));
      f[x] = there ? f[x] : 0.0f;
    }
    run_store<T, N>(a.out, dst + c, f);
  }
}

// ---- gradient -----------------------------------------------------------------------
// The tokens are sorted by id (stable, so a row's tokens keep their order), then
// each row of the table sums its own: no atomics on values, one order of sums.

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortRows = 512, kSortBits = 9;  // rows of the table per workgroup

// A row of more than kFew tokens is summed by the workgroups of the windows of
// kWindow places of the order that it touches.  (16384 tokens of text, 128256 x 4096:
// 64 instead of 8 takes 100 us more, 2 saves 5; 300 tokens, 1001 x 250 float32: 2 takes
// 17 us for 11, 4 takes 14.)
constexpr int kFew = 8, kWindow = 64;
int64_t windows_of(int64_t T) { return T > kFew ? (T + kWindow - 1) / kWindow : 0; }

// A large table of which most rows have no token is cleared as a whole beside the sort,
// in the order of its addresses (6.8 TB/s; zeros stored row by row between the sums
// come to 5.3), and the places of the order then write the rows that have tokens.
// 16384 tokens, 4096 wide: 128256 rows 264 -> 235 us, 65537 rows 173 -> 157; tables of
// 64 MB are the same either way, smaller ones 1 us slower.
bool clear_first(int64_t T, int64_t V, int64_t bytes) {
  return T <= V / 4 && bytes >= (int64_t)1 << 26;
}
constexpr int kPlaces = 8;  // of a workgroup (16: 5 us more)

struct GradWork {
  int32_t *first, *order;  // [V + 1]: a row's first place in order; [T]: tokens by row
  float* part;             // [windows][2][E]
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
// token behind those of the same row before it.  All ids are read by each of V / 512
// workgroups: one launch, whose time grows with T, and with V from 256 workgroups on.
// (us, rows 500 / 32000 / 128256 / 2^20: 300 ids 5 / 6 / 6 / 22, 16384 ids 22 / 18 / 15 /
// 54, 131072 ids 148 / 113 / 88 / 326, 2^20 ids 1175 / 771 / 628 / 2317.  With 2^20 ids the
// gradient of 128256 x 4096 bfloat16 moves 9.6 GB, 2 ms; a sort by digits was not built.)
// The workgroups behind them clear `bytes` of `out`, 16 by each thread.
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const int32_t* ids, int64_t T,
                                                                  int64_t V, GradWork w,
                                                                  uint8_t* out, int64_t bytes) {
  __shared__ int32_t cnt[kSortWaves][kSortRows];
  __shared__ int32_t tmp[kSortWaves];
  constexpr int kAhead = 8;       // loads under way
  constexpr int kOneByOne = 8;    // tokens of 64 (0, all rows at once always: 22 us for 15)
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t sorts = (uint32_t)((V + kSortRows - 1) / kSortRows);
  const int64_t block = block_of();
  if (block >= sorts) {
    const int64_t at = ((block - sorts) * kSortThreads + tid) * 16;
    if (at + 16 <= bytes) *(uint4*)(out + at) = make_uint4(0, 0, 0, 0);
    else
      for (int64_t i = at; i < bytes; i += 2) *(uint16_t*)(out + i) = 0;
    return;
  }
  const int64_t lo = block * kSortRows;
  const int rows = (int)min((int64_t)kSortRows, V - lo);
  const int64_t per = ((T + kSortWaves - 1) / kSortWaves + 63) & ~(int64_t)63;
  const int64_t t0 = min((int64_t)wave * per, T), t1 = min(t0 + per, T);
  // f(first token of 64, the lane's id) over this wave's share, -1 past its end
  auto walk = [&](auto&& f) {
    for (int64_t t = t0; t < t1; t += 64 * kAhead) {
      int32_t id[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t at = t + i * 64 + lane;
        id[i] = ids[min(at, T - 1)];
        if (at >= t1) id[i] = -1;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (t + i * 64 < t1) f(t + i * 64, id[i]);
    }
  };
  for (int i = tid; i < kSortWaves * kSortRows; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  int32_t below = 0;
  walk([&](int64_t, int32_t id) {
    const int64_t r = id - lo;
    if (id >= 0 && r < 0) ++below;
    else if (r >= 0 && r < rows) atomicAdd(&cnt[wave][r], 1);
  });
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
#pragma unroll
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
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) cnt[i][tid] += at;
    if (tid < rows) w.first[lo + tid] = at;
    if (lo + tid == V - 1) w.first[V] = at + total;
  }
  __syncthreads();
  walk([&](int64_t t, int32_t id) {
    const int64_t r64 = id - lo;
    const bool mine = id >= 0 && r64 >= 0 && r64 < rows;
    const int r = mine ? (int)r64 : -1;
    uint64_t todo = __ballot(mine);
    if (todo == 0) return;
    const uint64_t before = (1ull << lane) - 1;
    volatile int32_t* count = cnt[wave];
    if (__popcll(todo) <= kOneByOne) {
      // row by row
      while (todo) {
        const int key = __builtin_amdgcn_readlane(r, __ffsll((unsigned long long)todo) - 1);
        const uint64_t same = __ballot(r == key);
        const int32_t p = count[key];
        if (r == key) w.order[p + __popcll(same & before)] = (int32_t)(t + lane);
        if (lane == 0) count[key] = p + __popcll(same);
        todo &= ~same;
      }
    } else {
      // all rows at once: the lanes that agree with this one in every bit
      uint64_t same = todo;
#pragma unroll
      for (int b = 0; b < kSortBits; ++b) {
        const uint64_t set = __ballot(mine && (r >> b & 1));
        same &= r >> b & 1 ? set : ~set;
      }
      if (mine) {
        const int ahead = __popcll(same & before);
        const int32_t p = count[r];
        w.order[p + ahead] = (int32_t)(t + lane);
        if (ahead == 0) count[r] = p + __popcll(same);
      }
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// The sum of gradOut's columns c .. over places [p0, p1), one after another.
template <class T, int N>
__device__ __forceinline__ void sum_places(const EmbedGradArgs& a, const int32_t* order, int32_t p0,
                                           int32_t p1, int64_t c, float (&s)[N]) {
  constexpr int kAhead = 8;  // rows under way
#pragma unroll
  for (int x = 0; x < N; ++x) s[x] = 0.0f;
  for (int32_t p = p0; p < p1; p += kAhead) {
    RowRun<T, N> r[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      r[i] = run_at<T, N>(a.grad, (int64_t)order[min(p + i, p1 - 1)] * a.E + c);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int x = 0; x < N; ++x) s[x] += p + i < p1 ? T::get(r[i].v[x]) : 0.0f;
  }
}

// Workgroups before `window_blocks`: one slab of columns of the rows of more than
// kFew tokens in a window of the order; a row that lies in the window alone is
// finished, of another the sum goes to part[window][side], side 1 if it begins here.
// The others: `rows` rows of the table each, by groups of `lanes` threads; zeros for a
// row without tokens.  Both in one launch: the long sums hide behind the table's zeros.
// Or, rows 0 (a cleared table), the rows that begin in kPlaces places of the order each.
template <class T, int N, int S>
__global__ void __launch_bounds__(kThreads) embed_sum_kernel(EmbedGradArgs a, GradWork w,
                                                             uint32_t window_blocks, int lanes,
                                                             int rows) {
  __shared__ int32_t first[kThreads + 1];
  const int64_t block = block_of();
  const int lane = threadIdx.x % lanes, own = threadIdx.x / lanes, groups = kThreads / lanes;
  const int64_t slab = (int64_t)lanes * N;  // columns
  auto store = [&](int64_t v, int64_t c, float (&s)[N]) {
#pragma unroll
    for (int x = 0; x < N; ++x) s[x] *= a.scale;
    run_store<T, N>(a.out, v * a.E + c, s);
  };
  if (block < window_blocks) {
    __shared__ float tmp[kThreads][N];
    __shared__ int32_t row_of[kWindow];
    __shared__ int n_rows;
    const uint32_t slabs = (uint32_t)((a.E + slab - 1) / slab);
    const uint32_t j = (uint32_t)block / slabs, s0 = (uint32_t)block % slabs;
    const int64_t c = run_start(s0 * slab + lane * N, a.E, N);
    const int32_t n = w.first[a.V];
    const int64_t q = (int64_t)j * kWindow;
    if (q >= n) return;
    const int32_t q0 = (int32_t)q, q1 = (int32_t)min(q + kWindow, (int64_t)n);
    if (threadIdx.x < 64) {
      const int32_t p = min(q0 + (int32_t)threadIdx.x, q1 - 1);
      const int32_t v = a.ids[w.order[p]];
      const int32_t p0 = w.first[v], p1 = w.first[v + 1];
      const bool mine = q0 + (int32_t)threadIdx.x < q1 && p1 - p0 > kFew && p == max(p0, q0);
      const uint64_t all = __ballot(mine);
      if (mine) row_of[__popcll(all & ((1ull << threadIdx.x) - 1))] = v;
      if (threadIdx.x == 0) n_rows = __popcll(all);
    }
    __syncthreads();
    for (int i = 0; i < n_rows; ++i) {
      const int32_t v = row_of[i], p0 = w.first[v], p1 = w.first[v + 1];
      const int32_t b = max(p0, q0), e = min(p1, q1), per = (e - b + groups - 1) / groups;
      // the groups a share of the places each, joined in order
      float s[N];
      sum_places<T, N>(a, w.order, min(b + own * per, e), min(b + own * per + per, e), c, s);
#pragma unroll
      for (int x = 0; x < N; ++x) tmp[threadIdx.x][x] = s[x];
      __syncthreads();
      if (own == 0) {
        for (int g = 1; g < groups; ++g)
#pragma unroll
          for (int x = 0; x < N; ++x) s[x] += tmp[g * lanes + threadIdx.x][x];
        if (p0 >= q0 && p1 <= q1) {
          store(v, c, s);
        } else {
          float* out = w.part + ((int64_t)j * 2 + (p0 >= q0)) * a.E + c;
#pragma unroll
          for (int x = 0; x < N; ++x) out[x] = s[x];
        }
      }
      __syncthreads();
    }
    return;
  }
  auto sum_row = [&](int64_t v, int32_t p0, int32_t p1) {
    // S slabs at a time: a row of one token is S loads under way
    for (int64_t i = lane * N; i < a.E; i += S * slab) {
      int64_t c[S];
      float s[S][N];
#pragma unroll
      for (int k = 0; k < S; ++k) {
        c[k] = run_start(i + k * slab, a.E, N);
#pragma unroll
        for (int x = 0; x < N; ++x) s[k][x] = 0.0f;
      }
      for (int32_t p = p0; p < p1; ++p) {
        const int64_t row = (int64_t)w.order[p] * a.E;
        RowRun<T, N> g[S];
#pragma unroll
        for (int k = 0; k < S; ++k) g[k] = run_at<T, N>(a.grad, row + c[k]);
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
          for (int x = 0; x < N; ++x) s[k][x] += T::get(g[k].v[x]);
      }
#pragma unroll
      for (int k = 0; k < S; ++k)
        if (i + k * slab < a.E) store(v, c[k], s[k]);
    }
  };
  if (rows == 0) {
    __shared__ int32_t row_of[kPlaces], end[kPlaces];
    const int32_t n = w.first[a.V];
    const int64_t q = (block - window_blocks) * kPlaces;
    if (q >= n) return;
    if (threadIdx.x < kPlaces) {
      const int32_t p = (int32_t)min(q + threadIdx.x, (int64_t)n - 1);
      const int32_t v = a.ids[w.order[p]];
      const bool mine = q + threadIdx.x < n && w.first[v] == p;
      row_of[threadIdx.x] = mine ? v : -1;
      end[threadIdx.x] = w.first[v + 1];
    }
    __syncthreads();
    for (int i = own; i < kPlaces; i += groups) {
      const int32_t p0 = (int32_t)q + i;
      if (row_of[i] >= 0 && end[i] - p0 <= kFew) sum_row(row_of[i], p0, end[i]);
    }
    return;
  }
  const int64_t v0 = (block - window_blocks) * rows;
  const int here = (int)min((int64_t)rows, a.V - v0);
  for (int i = threadIdx.x; i <= here; i += kThreads) first[i] = w.first[v0 + i];
  __syncthreads();
  for (int r = own; r < here; r += groups)
    if (first[r + 1] - first[r] <= kFew) sum_row(v0 + r, first[r], first[r + 1]);
}

// The row that begins in window j and goes on behind it (its last place's, if any),
// from its parts in order.
template <class T>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(EmbedGradArgs a, GradWork w) {
  const int32_t n = w.first[a.V];
  const int64_t j = blockIdx.x, q0 = j * kWindow, q1 = q0 + kWindow;
  if (q1 >= n) return;
  const int64_t v = a.ids[w.order[q1 - 1]];
  const int32_t p0 = w.first[v], p1 = w.first[v + 1];
  const int64_t c = (int64_t)blockIdx.y * kThreads + threadIdx.x;
  if (p1 - p0 <= kFew || p0 < q0 || p1 <= q1 || c >= a.E) return;
  float s = w.part[(j * 2 + 1) * a.E + c];
#pragma unroll 8
  for (int64_t i = j + 1; i * kWindow < p1; ++i) s += w.part[i * 2 * a.E + c];
  ((typename T::elem*)a.out)[v * a.E + c] = T::put(s * a.scale);
}

}  // namespace

void launch_embed(const EmbedArgs& a, hipStream_t stream) {
  if (a.T * a.E == 0) return;
  by_run(a.dt, a.E, [&](auto t, auto n) {
    constexpr int N = decltype(n)::value;
    const int x = row_threads((a.E + N - 1) / N, kThreads), y = kThreads / x;
    hipLaunchKernelGGL((embed_kernel<decltype(t), N>), dim3((unsigned)((a.T + y - 1) / y)),
                       dim3(x, y), 0, stream, a);
  });
  REW_HIP(hipGetLastError());
}

size_t embed_grad_ws_bytes(int64_t T, int64_t V, int64_t E) {
  const int64_t windows = windows_of(T);
  return up256((size_t)(V + 1) * 4) + up256((size_t)T * 4) +
         (windows > 1 ? (size_t)windows * 2 * E * 4 : 0);
}

int launch_embed_grad(const EmbedGradArgs& a, hipStream_t stream) {
  if (a.V * a.E == 0) return 0;
  const GradWork w = grad_work(a);
  const int64_t windows = windows_of(a.T);
  const int64_t table = a.V * a.E * (a.dt == kF32 ? 4 : 2);
  const bool clear = clear_first(a.T, a.V, table);
  const int64_t bytes = clear ? table : 0;
  const int64_t sorts = (a.V + kSortRows - 1) / kSortRows;
  constexpr int64_t kCleared = 16 * kSortThreads;  // bytes of a workgroup
  hipLaunchKernelGGL(embed_sort_kernel, grid_of(sorts + (bytes + kCleared - 1) / kCleared),
                     dim3(kSortThreads), 0, stream, a.ids, a.T, a.V, w, (uint8_t*)a.out, bytes);
  if (a.T == 0 && clear) {
    REW_HIP(hipGetLastError());
    return 1;
  }
  by_run(a.dt, a.E, [&](auto t, auto n) {
    typedef decltype(t) Ty;
    constexpr int N = decltype(n)::value;
    const int64_t runs = (a.E + N - 1) / N;
    const int lanes = row_threads(runs, 64), groups = kThreads / lanes;
    // about 64 KiB of the table per workgroup, as long as that fills the card
    const int64_t bytes = a.E * (int64_t)sizeof(typename Ty::elem);
    int rows = (int)std::max<int64_t>(1, std::min<int64_t>(kThreads, 65536 / bytes));
    while (rows > groups && a.V < (int64_t)rows * 1024) rows /= 2;
    rows = std::max(groups, rows / groups * groups);
    const int64_t slabs = (runs + lanes - 1) / lanes;
    if (clear) rows = 0;
    const int64_t blocks =
        windows * slabs + (clear ? (a.T + kPlaces - 1) / kPlaces : (a.V + rows - 1) / rows);
    auto sum = [&](auto together) {
      hipLaunchKernelGGL((embed_sum_kernel<Ty, N, decltype(together)::value>),
                         grid_of(blocks), dim3(kThreads), 0, stream, a, w,
                         (uint32_t)(windows * slabs), lanes, rows);
    };
    if (slabs >= 4) sum(std::integral_constant<int, 4>());
    else if (slabs >= 2) sum(std::integral_constant<int, 2>());
    else sum(std::integral_constant<int, 1>());
    if (windows <= 1) return;
    hipLaunchKernelGGL((embed_join_kernel<Ty>),
                       dim3((unsigned)windows, (unsigned)((a.E + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, stream, a, w);
  });
  REW_HIP(hipGetLastError());
  return windows > 1 ? 3 : 2;
}

}  // namespace rew
