// Layer norm over rows of n values and its gradients (NormArgs and
// NormGradArgs in kernels.h).
//
// A row lies in the registers of a group of 64 to 1024 threads, kept from the
// first pass (mean) to the last: it is read once.  Thread i of the group holds
// the runs i, i + G, ... of 16 bytes (rows_device.h).
//
// Bound: HBM.  8192 x 4096 bfloat16 with float32 gamma: forward 30 us (4.4 TB/s),
// gradients 42 (4.8, their inputs partly in the caches) and 4 for the join.
// 300 x 20000 float16: 13.3, and 7.4 + 13.5 + 3.9, where a launch of a few rows on
// each CU is a chain of a row's load, two joined sums and its store.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "rows_device.h"

namespace rew {

namespace {

constexpr int kMaxGroup = 1024;
constexpr int64_t kMaxBlocks = 1 << 20;  // (a launch takes fewer than 2^32 threads)

// Sums of two values over the group of G threads, in all of them; `tmp` holds
// a pair per wave of the workgroup.  Every thread of the workgroup calls it.
template <int G>
__device__ __forceinline__ void group_sum2(float& x, float& y, float2* tmp) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    x += __shfl_xor(x, d);
    y += __shfl_xor(y, d);
  }
  if constexpr (G > 64) {
    const int wave = threadIdx.x >> 6, w0 = wave / (G / 64) * (G / 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[wave] = make_float2(x, y);
    __syncthreads();
    x = y = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) {
      x += tmp[w0 + w].x;
      y += tmp[w0 + w].y;
    }
  }
}

// The first pass leaves the mean as its roundings have it: (n / 1024 + some) steps off, which
// rstd multiplies (a row of 1001 values of 1000.1: results 0.04 off).  The second sums the
// deviations from it beside their squares: `rest`, their mean, is what it lacks.
// (A row of equal values, and eps far below what is left of its variance: not less than
// 2^-20 of the square taken away, some steps of it, so that rstd does not blow up `rest`'s
// own rounding.)
__device__ __forceinline__ float rstd_of(float square, float rest, float eps) {
  const float away = fminf(rest * rest, 3.402823466e38f);  // (an infinite square stays so)
  const float var = square - away, least = away * 0x1p-20f;
  return 1.0f / sqrtf((var < least ? least : var) + eps);
}

// The runs of thread g of a row's group: where they start, and from which value on
// they hold what no earlier run does (N: none).
template <int G, int C, int N>
struct Runs {
  int at[C], own[C];
  __device__ __forceinline__ Runs(int64_t n, int g) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t i = ((int64_t)c * G + g) * N;
      at[c] = (int)run_start(i, n, N);
      own[c] = (int)min(i - at[c], (int64_t)N);
    }
  }
};

// Workgroups of 256 threads, or of G where that is more: 256 / G rows each.
template <class T, class P, int N, int G, int C>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_kernel(NormArgs a) {
  constexpr int kRows = G > 256 ? 1 : 256 / G;
  __shared__ float2 tmp[(G > 256 ? G : 256) / 64];
  const int g = threadIdx.x % G;
  const int64_t n = a.n;
  const float inv = 1.0f / (float)n;
  const Runs<G, C, N> run(n, g);
  // Wide rows: one or two workgroups fit a CU, so each has its next row on the way, and
  // (up to 512 threads: the registers) keeps gamma and beta: read anew for every row
  // they are twice the bytes of x and y in 16 bits (3000 x 10000: 40 us).
  constexpr bool kAhead = G >= 256, kHold = G == 256 || G == 512;
  float w[C][N], b[C][N];
  if constexpr (kHold)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      run_load<P, N>(a.gamma, run.at[c], w[c]);
      run_load<P, N>(a.beta, run.at[c], b[c]);
    }
  RowRun<T, N> next[C];
  const int64_t step = (int64_t)gridDim.x * kRows;
  auto fetch = [&](int64_t r0) {
    const int64_t base = min(r0 + threadIdx.x / G, a.rows - 1) * n;
#pragma unroll
    for (int c = 0; c < C; ++c) next[c] = run_at<T, N>(a.x, base + run.at[c]);
  };
  if (kAhead) fetch((int64_t)blockIdx.x * kRows);
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + threadIdx.x / G;
    const bool there = row < a.rows;
    const int64_t base = (there ? row : a.rows - 1) * n;
    if (!kAhead) fetch(r0);
    float f[C][N];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) f[c][e] = T::get(next[c].v[e]);
    if (kAhead) fetch(r0 + step);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) s += e >= run.own[c] ? f[c][e] : 0.0f;
    group_sum2<G>(s, q, tmp);
    const float mean = s * inv;
    s = q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        f[c][e] -= mean;
        const float d = e >= run.own[c] ? f[c][e] : 0.0f;
        s += d;
        q = __builtin_fmaf(d, d, q);
      }
    group_sum2<G>(q, s, tmp);
    const float rest = s * inv, rstd = rstd_of(q * inv, rest, a.eps), shift = -rest * rstd;
    if (!there) continue;
    if (a.mean && g == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (run.own[c] == N) continue;
      if constexpr (!kHold) {
        run_load<P, N>(a.gamma, run.at[c], w[c]);
        run_load<P, N>(a.beta, run.at[c], b[c]);
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
        f[c][e] = __builtin_fmaf(__builtin_fmaf(f[c][e], rstd, shift), w[c][e], b[c][e]);
      run_store<T, N>(a.y, base + run.at[c], f[c]);
    }
  }
}

// Rows too long for the registers of 1024 threads: three walks over the row,
// the second and third from the caches.
template <class T, class P>
__global__ void __launch_bounds__(kMaxGroup) norm_long_kernel(NormArgs a) {
  constexpr int N = kRun<T>;
  __shared__ float2 tmp[kMaxGroup / 64];
  const int64_t row = blockIdx.x, n = a.n;
  const float inv = 1.0f / (float)n;
  auto walk = [&](auto&& f) {
    for (int64_t i = threadIdx.x * N; i < n; i += (int64_t)kMaxGroup * N) {
      const int64_t at = run_start(i, n, N);
      float v[N];
      run_load<T, N>(a.x, row * n + at, v);
      f(at, (int)(i - at), v);
    }
  };
  float s = 0.0f, q = 0.0f;
  walk([&](int64_t, int own, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) s += e >= own ? v[e] : 0.0f;
  });
  group_sum2<kMaxGroup>(s, q, tmp);
  const float mean = s * inv;
  s = q = 0.0f;
  walk([&](int64_t, int own, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = e >= own ? v[e] - mean : 0.0f;
      s += d;
      q = __builtin_fmaf(d, d, q);
    }
  });
  group_sum2<kMaxGroup>(q, s, tmp);
  const float rest = s * inv, rstd = rstd_of(q * inv, rest, a.eps), shift = -rest * rstd;
  if (a.mean && threadIdx.x == 0) {
    a.mean[row] = mean + rest;
    a.rstd[row] = rstd;
  }
  walk([&](int64_t at, int, float (&v)[N]) {
    float w[N], b[N];
    run_load<P, N>(a.gamma, at, w);
    run_load<P, N>(a.beta, at, b);
#pragma unroll
    for (int e = 0; e < N; ++e)
      v[e] = __builtin_fmaf(__builtin_fmaf(v[e] - mean, rstd, shift), w[e], b[e]);
    run_store<T, N>(a.y, row * n + at, v);
  });
}

// ---- gradients ----------------------------------------------------------------------

// Threads of a workgroup of norm_grad_kernel.
constexpr int grad_block(int G) { return G > 512 ? G : 512; }

// Workgroups that walk the rows, grad_block / G of them at a time (the next ones'
// values on their way while this one's sums are formed), and keep the columns' sums of
// dy xh and dy in registers; the row groups add theirs in LDS, in order, and leave one
// row of partial sums per workgroup: part[b][2][n].
template <class T, class P, int N, int G, int C>
__global__ void __launch_bounds__(grad_block(G)) norm_grad_kernel(NormGradArgs a, float* part) {
  constexpr int kRows = grad_block(G) / G;
  __shared__ float2 tmp[grad_block(G) / 64];
  __shared__ float sums[kRows > 1 ? G * N * C : 1];
  const int g = threadIdx.x % G, own = threadIdx.x / G;
  const int64_t n = a.n, step = (int64_t)gridDim.x * kRows;
  const float inv = 1.0f / (float)n;
  const Runs<G, C, N> run(n, g);
  float w[C][N], dg[C][N], db[C][N];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    run_load<P, N>(a.gamma, run.at[c], w[c]);
#pragma unroll
    for (int e = 0; e < N; ++e) dg[c][e] = db[c][e] = 0.0f;
  }
  RowRun<T, N> rx[C], ry[C];
  float mean = 0.0f, rstd = 0.0f;
  auto fetch = [&](int64_t r0) {
    const int64_t row = min(r0 + own, a.rows - 1);
#pragma unroll
    for (int c = 0; c < C; ++c) rx[c] = run_at<T, N>(a.x, row * n + run.at[c]);
#pragma unroll
    for (int c = 0; c < C; ++c) ry[c] = run_at<T, N>(a.dy, row * n + run.at[c]);
    mean = a.mean[row];
    rstd = a.rstd[row];
  };
  int64_t r0 = (int64_t)blockIdx.x * kRows;
  if (r0 < a.rows) fetch(r0);
  for (; r0 < a.rows; r0 += step) {
    const bool there = r0 + own < a.rows;
    float x[C][N], dy[C][N];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[c][e] = T::get(rx[c].v[e]);
        dy[c][e] = T::get(ry[c].v[e]);
      }
    const float m = mean, r = rstd;
    fetch(min(r0 + step, a.rows - 1));
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[c][e] = (x[c][e] - m) * r;
        dg[c][e] += there ? dy[c][e] * x[c][e] : 0.0f;
        db[c][e] += there ? dy[c][e] : 0.0f;
        dy[c][e] *= w[c][e];
        const float v = e >= run.own[c] ? dy[c][e] : 0.0f;
        s += v;
        q += e >= run.own[c] ? v * x[c][e] : 0.0f;
      }
    group_sum2<G>(s, q, tmp);
    s *= inv;
    q *= inv;
    if (!there) continue;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (run.own[c] == N) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) dy[c][e] = r * (dy[c][e] - s - x[c][e] * q);
      run_store<T, N>(a.dx, (r0 + own) * n + run.at[c], dy[c]);
    }
  }
  // the row groups' sums, one after another
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if constexpr (kRows > 1) {
      for (int o = kRows - 1; o > 0; --o) {
        __syncthreads();
        if (own == o)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < N; ++e)
              sums[(c * N + e) * G + g] = half ? db[c][e] : dg[c][e];
        __syncthreads();
        if (own == o - 1)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < N; ++e)
              (half ? db[c][e] : dg[c][e]) += sums[(c * N + e) * G + g];
      }
    }
    if (own == 0)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (run.own[c] == N) continue;
        float* p = part + ((int64_t)blockIdx.x * 2 + half) * n + run.at[c];
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = half ? db[c][e] : dg[c][e];
      }
  }
}

// Long rows: the two sums of each, mean w and mean w xh ...
template <class T, class P>
__global__ void __launch_bounds__(kMaxGroup) norm_grad_sums_kernel(NormGradArgs a, float2* out) {
  constexpr int N = kRun<T>;
  __shared__ float2 tmp[kMaxGroup / 64];
  const int64_t row = blockIdx.x, n = a.n;
  const float inv = 1.0f / (float)n, mean = a.mean[row], rstd = a.rstd[row];
  float s = 0.0f, q = 0.0f;
  for (int64_t i = threadIdx.x * N; i < n; i += (int64_t)kMaxGroup * N) {
    const int64_t at = run_start(i, n, N);
    float x[N], dy[N], w[N];
    run_load<T, N>(a.x, row * n + at, x);
    run_load<T, N>(a.dy, row * n + at, dy);
    run_load<P, N>(a.gamma, at, w);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool in = e >= i - at;
      const float v = dy[e] * w[e];
      s += in ? v : 0.0f;
      q += in ? v * ((x[e] - mean) * rstd) : 0.0f;
    }
  }
  group_sum2<kMaxGroup>(s, q, tmp);
  if (threadIdx.x == 0) out[row] = make_float2(s * inv, q * inv);
}

// .. and then dx and the columns' sums, 256 runs of columns over `per` rows in a
// workgroup: part[b][2][n].
template <class T, class P>
__global__ void __launch_bounds__(256) norm_grad_columns_kernel(NormGradArgs a, const float2* sums,
                                                                float* part, int64_t per) {
  constexpr int N = kRun<T>;
  const int64_t n = a.n, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= n) return;
  const int64_t at = run_start(i, n, N);
  float w[N], dg[N], db[N];
  run_load<P, N>(a.gamma, at, w);
#pragma unroll
  for (int e = 0; e < N; ++e) dg[e] = db[e] = 0.0f;
  const int64_t end = min(a.rows, ((int64_t)blockIdx.y + 1) * per);
#pragma unroll 4
  for (int64_t row = blockIdx.y * per; row < end; ++row) {
    float x[N], dy[N];
    run_load<T, N>(a.x, row * n + at, x);
    run_load<T, N>(a.dy, row * n + at, dy);
    const float mean = a.mean[row], rstd = a.rstd[row];
    const float2 m = sums[row];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xh = (x[e] - mean) * rstd;
      dg[e] += dy[e] * xh;
      db[e] += dy[e];
      dy[e] = rstd * (dy[e] * w[e] - m.x - xh * m.y);
    }
    run_store<T, N>(a.dx, row * n + at, dy);
  }
  float* p = part + (int64_t)blockIdx.y * 2 * n + at;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    p[e] = dg[e];
    p[n + e] = db[e];
  }
}

// dgamma and dbeta: the sum of the `parts` rows of partial sums, 16 waves a
// sixteenth of them each, joined in order.
template <class P>
__global__ void __launch_bounds__(1024) norm_join_kernel(NormGradArgs a, const float* part,
                                                         int parts) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = block_of() * 64 + lane;  // of the 2 n columns
  float s = 0.0f;
  if (i < 2 * a.n)
#pragma unroll 4
    for (int p = wave; p < parts; p += 16) s += part[(int64_t)p * 2 * a.n + i];
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || i >= 2 * a.n) return;
  for (int w = 1; w < 16; ++w) s += sums[w][lane];
  void* out = i < a.n ? a.dgamma : a.dbeta;
  ((typename P::elem*)out)[i < a.n ? i : i - a.n] = P::put(s);
}

// f(element type, parameter type, run length) for rows of n values.
template <class F>
void by_types(int dt, int p_dt, int64_t n, F&& f) {
  auto with = [&](auto t, auto p) {
    constexpr int N = kRun<decltype(t)>;
    if (n >= N) f(t, p, std::integral_constant<int, N>());
    else f(t, p, std::integral_constant<int, 1>());
  };
  if (dt == kF32) with(RowF32(), RowF32());
  else if (dt == kBF16 && p_dt == kF32) with(RowBf16(), RowF32());
  else if (dt == kBF16) with(RowBf16(), RowBf16());
  else if (p_dt == kF32) with(RowF16(), RowF32());
  else with(RowF16(), RowF16());
}

// f(group, runs of a thread) for a row of `runs` runs; false where it is too long: 4
// runs in each of 1024 threads, or (gradients, which hold six values for each of x) in
// each of 512.  Single: a row of fewer values than a run.  The smallest group that
// leaves registers for the next row and gamma: 3000 x 10000 bfloat16 on 512 threads 29.6
// us, on 1024 without 42; gradients 35 and, by the long rows' kernels, 65; 8000 x 4608 on
// 256 x 3 32 us, on 1024 44; 300 x 20000 on 1024 x 3 12.6, x 4 13.6.
template <bool Grad, bool Single, class F>
bool by_group(int64_t runs, F&& f) {
  if constexpr (Single) {
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    return true;
  } else {
    auto with = [&](auto g, auto c) { f(g, c); };
    std::integral_constant<int, 1> one;
    std::integral_constant<int, 2> two;
    if (runs <= 64) with(std::integral_constant<int, 64>(), one);
    else if (runs <= 128) with(std::integral_constant<int, 64>(), two);
    else if (runs <= 256) with(std::integral_constant<int, 256>(), one);
    else if (runs <= 512) with(std::integral_constant<int, 256>(), two);
    else if (runs <= 768)
      with(std::integral_constant<int, 256>(), std::integral_constant<int, 3>());
    else if (runs <= 1024) with(std::integral_constant<int, 512>(), two);
    else if (runs <= 1536)
      with(std::integral_constant<int, 512>(), std::integral_constant<int, 3>());
    else if (runs <= 2048)
      with(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
    else if (Grad || runs > 4 * kMaxGroup) return false;
    else if constexpr (!Grad) {
      if (runs <= 3 * kMaxGroup)
        with(std::integral_constant<int, 1024>(), std::integral_constant<int, 3>());
      else
        with(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    }
    return true;
  }
}

// Workgroups of norm_grad_kernel at most, one per CU, since each leaves a row of
// partial sums that is written and read once more; rows of a part of long rows.
// (300 and 1600 rows of 20000: 16 rows 12.9 and 37.5 us, 8 rows 12.9 and 42.5, 4 rows
// 14.9 and 43.8)
constexpr int64_t kParts = 256;
constexpr int64_t kPartRows = 16;

}  // namespace

void launch_norm(const NormArgs& a, hipStream_t stream) {
  if (a.rows * a.n == 0) return;
  by_types(a.x_dt, a.p_dt, a.n, [&](auto t, auto p, auto nn) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    constexpr int N = decltype(nn)::value;
    const bool fits = by_group<false, N == 1>((a.n + N - 1) / N, [&](auto g, auto c) {
      constexpr int G = decltype(g)::value, C = decltype(c)::value;
      constexpr int rows = G > 256 ? 1 : 256 / G;
      const int64_t most = G == 1024 ? 256 : G == 512 ? 512 : G == 256 ? 1024 : kMaxBlocks;
      const int64_t blocks = std::min((a.rows + rows - 1) / rows, most);
      hipLaunchKernelGGL((norm_kernel<T, P, N, G, C>), dim3((unsigned)blocks),
                         dim3(G > 256 ? G : 256), 0, stream, a);
    });
    if (!fits)
      hipLaunchKernelGGL((norm_long_kernel<T, P>), dim3((unsigned)a.rows), dim3(kMaxGroup), 0,
                         stream, a);
  });
  REW_HIP(hipGetLastError());
}

// (the sums of long rows, then the parts)
size_t norm_grad_ws_bytes(int64_t rows, int64_t n) {
  return (size_t)rows * sizeof(float2) + (size_t)std::min(std::max<int64_t>(rows, 1), kParts) * 2 *
                                             n * sizeof(float);
}

int launch_norm_grad(const NormGradArgs& a, hipStream_t stream) {
  if (a.n == 0) return 0;
  int launches = 2;
  float2* sums = (float2*)a.work;
  float* part = a.work + 2 * a.rows;
  by_types(a.x_dt, a.p_dt, a.n, [&](auto t, auto p, auto nn) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    constexpr int N = decltype(nn)::value;
    const int64_t runs = (a.n + N - 1) / N;
    int parts = 1;
    const bool fits = by_group<true, N == 1>(runs, [&](auto g, auto c) {
      constexpr int G = decltype(g)::value, C = decltype(c)::value;
      constexpr int rows = grad_block(G) / G;
      parts = (int)std::max<int64_t>(1, std::min((a.rows + rows - 1) / rows, kParts));
      hipLaunchKernelGGL((norm_grad_kernel<T, P, N, G, C>), dim3(parts), dim3(grad_block(G)), 0,
                         stream, a, part);
    });
    if (!fits) {
      launches = 3;
      const int64_t per = std::max(kPartRows, (a.rows + kParts - 1) / kParts);
      parts = (int)std::max<int64_t>(1, (a.rows + per - 1) / per);
      if (a.rows)
        hipLaunchKernelGGL((norm_grad_sums_kernel<T, P>), dim3((unsigned)a.rows), dim3(kMaxGroup),
                           0, stream, a, sums);
      hipLaunchKernelGGL((norm_grad_columns_kernel<T, P>),
                         dim3((unsigned)((runs + 255) / 256), parts), dim3(256), 0, stream, a, sums,
                         part, per);
    }
    hipLaunchKernelGGL((norm_join_kernel<P>), grid_of((2 * a.n + 63) / 64), dim3(1024), 0, stream,
                       a, part, parts);
  });
  REW_HIP(hipGetLastError());
  return launches;
}

}  // namespace rew
