// Layer norm over rows of n values and its gradients (NormArgs and
// NormGradArgs in kernels.h).
//
// A row lies in the registers of a group of 64 to 1024 threads, kept from the
// first pass (mean) to the last: it is read once.  Thread i of the group holds
// runs i, i + G, ... of at most 16 bytes.
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

// A row of n values in registers: C runs of N.
template <class T, int N, int G, int C>
__device__ __forceinline__ void row_load(const void* x, int64_t row, int64_t n, int g,
                                         float (&f)[C][N]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int64_t i = ((int64_t)c * G + g) * N;
    if (i < n) run_load<T, N>(x, row * n + i, f[c]);
    else
#pragma unroll
      for (int e = 0; e < N; ++e) f[c][e] = 0.0f;
  }
}

// Workgroups of 256 threads, or of G where that is more: 256 / G rows each.
template <class T, class P, int N, int G, int C>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_kernel(NormArgs a) {
  constexpr int kRows = G > 256 ? 1 : 256 / G;
  __shared__ float2 tmp[(G > 256 ? G : 256) / 64];
  const int g = threadIdx.x % G;
  const int64_t n = a.n;
  const float inv = 1.0f / (float)n;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t row = r0 + threadIdx.x / G;
    const bool there = row < a.rows;
    float f[C][N];
    row_load<T, N, G, C>(a.x, there ? row : a.rows - 1, n, g, f);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) s += f[c][e];
    group_sum2<G>(s, q, tmp);
    const float mean = s * inv;
    q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = ((int64_t)c * G + g) * N < n;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        f[c][e] -= mean;
        q += in ? f[c][e] * f[c][e] : 0.0f;
      }
    }
    group_sum2<G>(q, s, tmp);
    const float rstd = 1.0f / sqrtf(q * inv + a.eps);
    if (!there) continue;
    if (a.mean && g == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t i = ((int64_t)c * G + g) * N;
      if (i >= n) continue;
      float w[N], b[N];
      run_load<P, N>(a.gamma, i, w);
      run_load<P, N>(a.beta, i, b);
#pragma unroll
      for (int e = 0; e < N; ++e) f[c][e] = f[c][e] * rstd * w[e] + b[e];
      run_store<T, N>(a.y, row * n + i, f[c]);
    }
  }
}

// Rows too long for the registers of 1024 threads: three walks over the row,
// the second and third from the caches.
template <class T, class P, int N>
__global__ void __launch_bounds__(kMaxGroup) norm_long_kernel(NormArgs a) {
  __shared__ float2 tmp[kMaxGroup / 64];
  const int64_t row = blockIdx.x, n = a.n;
  constexpr int64_t kStep = (int64_t)kMaxGroup * N;
  const int64_t i0 = threadIdx.x * N;
  const float inv = 1.0f / (float)n;
  float s = 0.0f, q = 0.0f;
  for (int64_t i = i0; i < n; i += kStep) {
    float f[N];
    run_load<T, N>(a.x, row * n + i, f);
#pragma unroll
    for (int e = 0; e < N; ++e) s += f[e];
  }
  group_sum2<kMaxGroup>(s, q, tmp);
  const float mean = s * inv;
  q = 0.0f;
  for (int64_t i = i0; i < n; i += kStep) {
    float f[N];
    run_load<T, N>(a.x, row * n + i, f);
#pragma unroll
    for (int e = 0; e < N; ++e) q += (f[e] - mean) * (f[e] - mean);
  }
  group_sum2<kMaxGroup>(q, s, tmp);
  const float rstd = 1.0f / sqrtf(q * inv + a.eps);
  if (a.mean && threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  for (int64_t i = i0; i < n; i += kStep) {
    float f[N], w[N], b[N];
    run_load<T, N>(a.x, row * n + i, f);
    run_load<P, N>(a.gamma, i, w);
    run_load<P, N>(a.beta, i, b);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (f[e] - mean) * rstd * w[e] + b[e];
    run_store<T, N>(a.y, row * n + i, f);
  }
}

// ---- gradients ----------------------------------------------------------------------

// Workgroups of 1024 threads, 1024 / G rows at a time, that walk the rows
// blockIdx.x * (1024 / G), + gridDim.x * (1024 / G), ... and keep the columns'
// sums of dy xh and dy in registers; the row groups add theirs in LDS, in order,
// and leave one row of partial sums per workgroup: part[b][2][n].
template <class T, class P, int N, int G, int C>
__global__ void __launch_bounds__(kMaxGroup) norm_grad_kernel(NormGradArgs a) {
  constexpr int kRows = kMaxGroup / G;
  __shared__ float2 tmp[kMaxGroup / 64];
  __shared__ float sums[kRows > 1 ? G * N * C : 1];
  const int g = threadIdx.x % G, own = threadIdx.x / G;
  const int64_t n = a.n;
  const float inv = 1.0f / (float)n;
  float w[C][N], dg[C][N], db[C][N];
  row_load<P, N, G, C>(a.gamma, 0, n, g, w);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < N; ++e) dg[c][e] = db[c][e] = 0.0f;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (int64_t)gridDim.x * kRows) {
    const bool there = r0 + own < a.rows;
    const int64_t row = there ? r0 + own : a.rows - 1;
    float x[C][N], dy[C][N];
    row_load<T, N, G, C>(a.x, row, n, g, x);
    row_load<T, N, G, C>(a.dy, row, n, g, dy);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = ((int64_t)c * G + g) * N < n;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[c][e] = in ? (x[c][e] - mean) * rstd : 0.0f;
        if (there) {
          dg[c][e] += dy[c][e] * x[c][e];
          db[c][e] += dy[c][e];
        }
        dy[c][e] *= w[c][e];
        s += dy[c][e];
        q += dy[c][e] * x[c][e];
      }
    }
    group_sum2<G>(s, q, tmp);
    s *= inv;
    q *= inv;
    if (!there) continue;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t i = ((int64_t)c * G + g) * N;
      if (i >= n) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) dy[c][e] = rstd * (dy[c][e] - s - x[c][e] * q);
      run_store<T, N>(a.dx, row * n + i, dy[c]);
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
        const int64_t i = ((int64_t)c * G + g) * N;
        if (i >= n) continue;
#pragma unroll
        for (int e = 0; e < N; ++e)
          a.work[((int64_t)blockIdx.x * 2 + half) * n + i + e] = half ? db[c][e] : dg[c][e];
      }
  }
}

// Long rows: dx alone, the row walked twice.
template <class T, class P, int N>
__global__ void __launch_bounds__(kMaxGroup) norm_grad_long_kernel(NormGradArgs a) {
  __shared__ float2 tmp[kMaxGroup / 64];
  const int64_t row = blockIdx.x, n = a.n;
  constexpr int64_t kStep = (int64_t)kMaxGroup * N;
  const int64_t i0 = threadIdx.x * N;
  const float inv = 1.0f / (float)n, mean = a.mean[row], rstd = a.rstd[row];
  float s = 0.0f, q = 0.0f;
  for (int64_t i = i0; i < n; i += kStep) {
    float x[N], dy[N], w[N];
    run_load<T, N>(a.x, row * n + i, x);
    run_load<T, N>(a.dy, row * n + i, dy);
    run_load<P, N>(a.gamma, i, w);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      s += dy[e] * w[e];
      q += dy[e] * w[e] * ((x[e] - mean) * rstd);
    }
  }
  group_sum2<kMaxGroup>(s, q, tmp);
  s *= inv;
  q *= inv;
  for (int64_t i = i0; i < n; i += kStep) {
    float x[N], dy[N], w[N];
    run_load<T, N>(a.x, row * n + i, x);
    run_load<T, N>(a.dy, row * n + i, dy);
    run_load<P, N>(a.gamma, i, w);
#pragma unroll
    for (int e = 0; e < N; ++e)
      dy[e] = rstd * (dy[e] * w[e] - s - (x[e] - mean) * rstd * q);
    run_store<T, N>(a.dx, row * n + i, dy);
  }
}

// .. and the columns' sums over the rows b, b + parts, ...: part[b][2][n].
template <class T, int N>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormGradArgs a, int parts) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N, n = a.n;
  if (i >= n) return;
  float dg[N], db[N];
#pragma unroll
  for (int e = 0; e < N; ++e) dg[e] = db[e] = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += parts) {
    float x[N], dy[N];
    run_load<T, N>(a.x, row * n + i, x);
    run_load<T, N>(a.dy, row * n + i, dy);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      dg[e] += dy[e] * ((x[e] - mean) * rstd);
      db[e] += dy[e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    a.work[(int64_t)blockIdx.y * 2 * n + i + e] = dg[e];
    a.work[((int64_t)blockIdx.y * 2 + 1) * n + i + e] = db[e];
  }
}

// dgamma and dbeta: the sum of the `parts` rows of partial sums, 16 waves a
// sixteenth of them each, joined in order.
template <class P>
__global__ void __launch_bounds__(1024) norm_join_kernel(NormGradArgs a, int parts) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;  // of the 2 n columns
  float s = 0.0f;
  if (i < 2 * a.n)
    for (int p = wave; p < parts; p += 16) s += a.work[(int64_t)p * 2 * a.n + i];
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || i >= 2 * a.n) return;
  for (int w = 1; w < 16; ++w) s += sums[w][lane];
  void* out = i < a.n ? a.dgamma : a.dbeta;
  ((typename P::elem*)out)[i < a.n ? i : i - a.n] = P::put(s);
}

// f(element type, parameter type, run length): the longest run of at most 16
// bytes of x's values that divides a row.  (A run of parameters in float32 is
// then up to 32 bytes: two loads.)
template <class F>
void by_types(int dt, int p_dt, int64_t n, F&& f) {
  auto runs = [&](auto t, auto p, auto most) {
    constexpr int M = decltype(most)::value;
    if (n % M == 0) f(t, p, std::integral_constant<int, M>());
    else f(t, p, std::integral_constant<int, 1>());
  };
  std::integral_constant<int, 8> eight;
  if (dt == kF32) runs(RowF32(), RowF32(), std::integral_constant<int, 4>());
  else if (dt == kBF16 && p_dt == kF32) runs(RowBf16(), RowF32(), eight);
  else if (dt == kBF16) runs(RowBf16(), RowBf16(), eight);
  else if (p_dt == kF32) runs(RowF16(), RowF32(), eight);
  else runs(RowF16(), RowF16(), eight);
}

// f(group, runs per thread) for a row of `runs` runs of N values, false where it
// is too long: at most 16 values a thread.
template <int N, class F>
bool by_group(int64_t runs, F&& f) {
  constexpr int C = 16 / N;  // most runs of a thread
  auto with = [&](auto g) {
    constexpr int G = decltype(g)::value;
    if constexpr (C <= 4) {
      if (runs <= G) f(g, std::integral_constant<int, 1>());
      else if (runs <= 2 * G) f(g, std::integral_constant<int, 2>());
      else f(g, std::integral_constant<int, C>());
    } else {
      if (runs <= 4 * G) f(g, std::integral_constant<int, 4>());
      else f(g, std::integral_constant<int, C>());
    }
  };
  if (runs > (int64_t)C * kMaxGroup) return false;
  if (runs <= 64 * C) with(std::integral_constant<int, 64>());
  else if (runs <= 256 * C) with(std::integral_constant<int, 256>());
  else with(std::integral_constant<int, kMaxGroup>());
  return true;
}

// Workgroups of norm_grad_kernel (or shares of norm_columns_kernel's rows): one
// per CU, since each leaves a row of partial sums that is written and read once
// more.
int64_t grad_parts(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(rows, 256)); }

}  // namespace

void launch_norm(const NormArgs& a, hipStream_t stream) {
  if (a.rows * a.n == 0) return;
  by_types(a.x_dt, a.p_dt, a.n, [&](auto t, auto p, auto nn) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    constexpr int N = decltype(nn)::value;
    const bool fits = by_group<N>(a.n / N, [&](auto g, auto c) {
      constexpr int G = decltype(g)::value, C = decltype(c)::value;
      constexpr int rows = G > 256 ? 1 : 256 / G;
      const int64_t blocks = std::min<int64_t>((a.rows + rows - 1) / rows, kMaxBlocks);
      hipLaunchKernelGGL((norm_kernel<T, P, N, G, C>), dim3((unsigned)blocks),
                         dim3(G > 256 ? G : 256), 0, stream, a);
    });
    if (!fits)
      hipLaunchKernelGGL((norm_long_kernel<T, P, N>), dim3((unsigned)a.rows), dim3(kMaxGroup), 0,
                         stream, a);
  });
  REW_HIP(hipGetLastError());
}

size_t norm_grad_ws_bytes(int64_t rows, int64_t n) {
  return (size_t)grad_parts(rows) * 2 * n * sizeof(float);
}

int launch_norm_grad(const NormGradArgs& a, hipStream_t stream) {
  if (a.n == 0) return 0;
  int parts = (int)grad_parts(a.rows), launches = 2;
  by_types(a.x_dt, a.p_dt, a.n, [&](auto t, auto p, auto nn) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    constexpr int N = decltype(nn)::value;
    const bool fits = by_group<N>(a.n / N, [&](auto g, auto c) {
      constexpr int G = decltype(g)::value, C = decltype(c)::value;
      constexpr int rows = kMaxGroup / G;
      parts = (int)std::min<int64_t>(parts, std::max<int64_t>(1, (a.rows + rows - 1) / rows));
      hipLaunchKernelGGL((norm_grad_kernel<T, P, N, G, C>), dim3(parts), dim3(kMaxGroup), 0,
                         stream, a);
    });
    if (!fits) {
      launches = 3;
      if (a.rows)
        hipLaunchKernelGGL((norm_grad_long_kernel<T, P, N>), dim3((unsigned)a.rows),
                           dim3(kMaxGroup), 0, stream, a);
      hipLaunchKernelGGL((norm_columns_kernel<T, N>),
                         dim3((unsigned)((a.n / N + 255) / 256), parts), dim3(256), 0, stream, a,
                         parts);
    }
    hipLaunchKernelGGL((norm_join_kernel<P>), dim3((unsigned)((2 * a.n + 63) / 64)), dim3(1024), 0,
                       stream, a, parts);
  });
  REW_HIP(hipGetLastError());
  return launches;
}

}  // namespace rew
