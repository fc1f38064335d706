// The gradients of packed attention (PackedGradArgs in kernels.h), without
// anything of size rows x keys in memory.
//
// Three launches.  The first writes delta = dout . out per row.  The second
// gives each workgroup 128 keys of one KV head and walks the rows that see
// them, dK and dV staying in registers; the third gives each workgroup 128
// rows and walks their keys, dQ staying in registers.  Both recompute
// P = exp(S - lse), so the scores are formed twice: 7 products of rows x keys
// x D where 5 would do, for sums whose order never changes (a single pass
// would add dQ across workgroups with atomics).  The rows of the H / Hkv heads
// of a KV head are walked together, so the sum over the group is part of the
// accumulation.
//
// In each product one operand stays in registers and the other is read from
// LDS; S and dP come out with the operand in registers along the lanes, so P
// and dS go from the accumulators straight into the next product, as in the
// forward kernel, and the LDS operand of that product is read transposed.
#include <algorithm>

#include "attn_device.h"
#include "kernels.h"

namespace rew {

namespace pg {
constexpr int BR = 128;  // rows (dQ) or keys (dK, dV) of a workgroup
constexpr int BT = 64;   // rows or keys of a tile that it walks
constexpr int64_t kDeltaBlocks = 2048;
constexpr float kLog2e = 1.4426950408889634f;
}  // namespace pg

// Chunk pc (16 bytes) of row r of an LDS tile of D / 8 = CPR chunks a row
// holds logical chunk pc ^ grad_swizzle(r): reading one chunk column of 16
// consecutive rows touches every bank once, and so does the transposed read of
// 4 rows x 32 bytes by each of four 16-lane groups.
template <int CPR>
__device__ __forceinline__ int grad_swizzle(int r) {
  if constexpr (CPR == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}

// ---- delta --------------------------------------------------------------------------
// D / 8 lanes per row of T H rows.  float16 has no room for dS at any scale:
// it is stored as F dS, F the power of two that takes the bound
// |dS| <= 2 D max|dout| max|V| to 2^15, so this kernel also leaves the maxima
// of its workgroups (a maximum does not depend on their order).
template <class M, int D>
__global__ void __launch_bounds__(256) grad_delta_kernel(PackedGradArgs a) {
  constexpr int L = D / 8;
  const int64_t rows = a.T * a.H, step = gridDim.x * (256ll / L);
  const int ch = threadIdx.x % L;
  float* delta = (float*)a.work;
  float most = 0.0f, most_v = 0.0f;
  for (int64_t i = blockIdx.x * (256ll / L) + threadIdx.x / L; i < rows; i += step) {
    const uint4 x = ((const uint4*)a.out)[i * L + ch], y = ((const uint4*)a.dout)[i * L + ch];
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y0 = M::lo(ys[k]), y1 = M::hi(ys[k]);
      s = fmaf(M::lo(xs[k]), y0, s);
      s = fmaf(M::hi(xs[k]), y1, s);
      if constexpr (M::kScaled) most = fmaxf(most, fmaxf(fabsf(y0), fabsf(y1)));
    }
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if (ch == 0) delta[i] = s;
  }
  if constexpr (M::kScaled) {
    const int64_t n = a.T * a.Hkv * L;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
      const uint4 x = ((const uint4*)a.v)[i];
      for (uint32_t w : {x.x, x.y, x.z, x.w})
        most_v = fmaxf(most_v, fmaxf(fabsf(M::lo(w)), fabsf(M::hi(w))));
    }
    __shared__ float part[8];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      most = fmaxf(most, __shfl_xor(most, d));
      most_v = fmaxf(most_v, __shfl_xor(most_v, d));
    }
    if ((threadIdx.x & 63) == 0) {
      part[threadIdx.x >> 6] = most;
      part[4 + (threadIdx.x >> 6)] = most_v;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      const float* q = part + 4 * threadIdx.x;
      delta[rows + blockIdx.x * 2 + threadIdx.x] = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
    }
  }
}
// F, from the maxima of the delta kernel's workgroups (a power of two; 1 for
// bfloat16).  Every thread of a workgroup of 256 calls it.
template <class M, int D>
__device__ __forceinline__ float grad_factor(const PackedGradArgs& a) {
  if constexpr (!M::kScaled) return 1.0f;
  __shared__ float part[8];
  const float* m = (const float*)a.work + a.T * a.H;
  float d = 0.0f, v = 0.0f;
  for (int i = threadIdx.x; i < a.delta_blocks; i += 256) {
    d = fmaxf(d, m[2 * i]);
    v = fmaxf(v, m[2 * i + 1]);
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) {
    d = fmaxf(d, __shfl_xor(d, x));
    v = fmaxf(v, __shfl_xor(v, x));
  }
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = d;
    part[4 + (threadIdx.x >> 6)] = v;
  }
  __syncthreads();
  d = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  v = fmaxf(fmaxf(part[4], part[5]), fmaxf(part[6], part[7]));
  const float bound = 2.0f * D * d * v;
  if (!(bound > 0.0f && bound < INFINITY)) return 1.0f;
  int e;
  (void)frexpf(bound, &e);  // bound <= 2^e
  return ldexpf(1.0f, min(max(15 - e, -60), 60));
}

// Fragment offsets in an LDS tile of D columns: `rows` for the operand whose
// rows lie along the lanes (row c, chunk 2t + g), `cols` for the transposed
// read (ds_read_b64_tr_b16) of 8 rows' columns dt 32 + 16 (G & 1) ..; the
// second half of it, 8 rows on, is at (cols ^ 16) + 8 D.
template <int D>
struct GradFrags {
  int rows[D / 16], cols[D / 32];
  __device__ __forceinline__ GradFrags() {
    constexpr int CPR = D / 8;
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
    const int g16 = lane >> 4, s16 = lane & 15;
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
      rows[t] = c * D + (((2 * t + g) ^ grad_swizzle<CPR>(c)) * 8);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const int r = 4 * (g16 >> 1) + (s16 >> 2), col = dt * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
      cols[dt] = r * D + (((col >> 3) ^ grad_swizzle<CPR>(r)) * 8) + (col & 7);
    }
  }
};
template <class M, int D>
__device__ __forceinline__ typename M::frag grad_cols(const uint16_t* tile, int off) {
  union {
    v4s h[2];
    typename M::frag v;
  } f;
  f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(tile + off));
  f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(tile + ((off ^ 16) + 8 * D)));
  return f.v;
}
// acc[dt] += (columns of 16 rows of `tile`)^T x the packed values of those rows
template <class M, int D>
__device__ __forceinline__ void grad_accumulate(f32x16_t (&acc)[D / 32], const uint16_t* tile,
                                                const GradFrags<D>& fr, const uint32_t (&pk)[8]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    union {
      uint32_t w[4];
      typename M::frag v;
    } p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p.w[i] = pk[u * 4 + i];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
      acc[dt] = M::mma(grad_cols<M, D>(tile + u * 16 * D, fr.cols[dt]), p.v, acc[dt]);
  }
}

// ---- dK, dV -----------------------------------------------------------------------------
template <class M, int D>
__global__ void __launch_bounds__(256, 1) grad_kv_kernel(PackedGradArgs a) {
  using namespace pg;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BT * D, RPD = 64 / CPR;
  constexpr int NDMA = TILE / 512 / 4;
  __shared__ __attribute__((aligned(1024))) uint16_t Qs[TILE], Ds[TILE];
  __shared__ __attribute__((aligned(16))) float lse_s[BT], delta_s[BT];
  __shared__ __attribute__((aligned(16))) int seen_s[BT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, hk = blockIdx.x % a.Hkv;
  const SeqTile st = find_tile(a.starts, a.n_seq, (int)a.T, 1, BR, blockIdx.x / a.Hkv);
  if (st.seq == -2) return;
  const int rows = st.real(a.n_seq) ? st.n * G : 0;
  const int k0 = st.tile * BR, key = k0 + wave * 32 + c;  // this lane's key
  const int64_t kstride = (int64_t)a.Hkv * D;
  frag kf[NT], vf[NT];
  {
    const int64_t at = (st.first + min(key, st.n - 1)) * kstride + hk * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      kf[t] = *(const frag*)((const uint16_t*)a.k + at + t * 16 + g * 8);
      vf[t] = *(const frag*)((const uint16_t*)a.v + at + t * 16 + g * 8);
    }
  }
  const GradFrags<D> fr;
  const int row_in = lane / CPR, pc = lane % CPR;
  f32x16_t dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.0f;
  const float sl2 = a.scale * kLog2e;
  const float* delta = (const float*)a.work;
  const float F = grad_factor<M, D>(a), fs = F * exp2f(-M::kGradShift);
  // causal: rows of tokens before the workgroup's first key do not see it
  const int first_row = a.causal ? k0 * G / BT * BT : 0;
  for (int r0 = first_row; r0 < rows; r0 += BT) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NDMA; ++q) {
      const int blk = wave * NDMA + q, lr = blk * RPD + row_in;
      const int r = min(r0 + lr, rows - 1), t = r / G, hg = r - t * G;
      const int64_t at = ((int64_t)(st.first + t) * a.H + hk * G + hg) * D +
                         (pc ^ grad_swizzle<CPR>(lr)) * 8;
      dma16((const uint16_t*)a.q + at, Qs + blk * 512);
      dma16((const uint16_t*)a.dout + at, Ds + blk * 512);
    }
    if (threadIdx.x < BT) {
      const int r = r0 + threadIdx.x, rr = min(r, rows - 1), t = rr / G;
      const int64_t at = (int64_t)(st.first + t) * a.H + hk * G + rr - t * G;
      lse_s[threadIdx.x] = a.lse[at] * kLog2e - M::kGradShift;
      delta_s[threadIdx.x] = delta[at];
      // keys below it are seen by this row; a row past the last one sees none
      seen_s[threadIdx.x] = r >= rows ? 0 : a.causal ? t + 1 : st.n;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool all = r0 + BT <= rows && (!a.causal || r0 / G >= k0 + BR - 1);
#pragma unroll
    for (int h = 0; h < BT / 32; ++h) {
      const uint16_t *Qt = Qs + h * 32 * D, *Dt = Ds + h * 32 * D;
      f32x16_t s, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s = M::mma(*(const frag*)(Qt + fr.rows[t]), kf[t], s);
        dp = M::mma(*(const frag*)(Dt + fr.rows[t]), vf[t], dp);
      }
      uint32_t pp[8], pd[8];
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int lr = h * 32 + e4 * 8 + g * 4;
        const float4 l4 = *(const float4*)(lse_s + lr), d4 = *(const float4*)(delta_s + lr);
        const int4 t4 = *(const int4*)(seen_s + lr);
        const float l[4] = {l4.x, l4.y, l4.z, l4.w}, dl[4] = {d4.x, d4.y, d4.z, d4.w};
        const int seen[4] = {t4.x, t4.y, t4.z, t4.w};
        float p[4], ds[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e4 * 4 + i;
          const bool see = all || key < seen[i];
          const float x = fa_exp2(fmaf(s[e], sl2, -l[i]));
          float y = x * (dp[e] - dl[i]);
          if constexpr (M::kScaled) y *= fs;
          p[i] = see ? x : 0.0f;
          ds[i] = see ? y : 0.0f;
        }
        pp[e4 * 2] = M::pack(p[0], p[1]);
        pp[e4 * 2 + 1] = M::pack(p[2], p[3]);
        pd[e4 * 2] = M::pack(ds[0], ds[1]);
        pd[e4 * 2 + 1] = M::pack(ds[2], ds[3]);
      }
      grad_accumulate<M, D>(dv, Dt, fr, pp);
      grad_accumulate<M, D>(dk, Qt, fr, pd);
    }
  }
  if (key >= st.n) return;
  const int64_t at = (st.first + key) * kstride + hk * D;
  uint16_t *DK = (uint16_t*)a.dk + at, *DV = (uint16_t*)a.dv + at;
  const float sv = exp2f(-M::kGradShift), sk = a.scale / F;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = dt * 32 + r * 8 + g * 4;
      *(uint2*)(DK + d) = make_uint2(M::pack(dk[dt][r * 4] * sk, dk[dt][r * 4 + 1] * sk),
                                     M::pack(dk[dt][r * 4 + 2] * sk, dk[dt][r * 4 + 3] * sk));
      *(uint2*)(DV + d) = make_uint2(M::pack(dv[dt][r * 4] * sv, dv[dt][r * 4 + 1] * sv),
                                     M::pack(dv[dt][r * 4 + 2] * sv, dv[dt][r * 4 + 3] * sv));
    }
}

// ---- dQ -----------------------------------------------------------------------------------
template <class M, int D>
__global__ void __launch_bounds__(256, 2) grad_q_kernel(PackedGradArgs a) {
  using namespace pg;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BT * D, RPD = 64 / CPR;
  constexpr int NDMA = TILE / 512 / 4;
  __shared__ __attribute__((aligned(1024))) uint16_t Ks[TILE], Vs[TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, hk = blockIdx.x % a.Hkv;
  const SeqTile st = find_tile(a.starts, a.n_seq, (int)a.T, G, BR, blockIdx.x / a.Hkv);
  if (st.seq == -2) return;
  const int rows = st.n * G, keys = st.real(a.n_seq) ? st.n : 0;
  const int r0 = st.tile * BR + wave * 32, row = r0 + c;
  const int tok = min(row, rows - 1) / G, hg = min(row, rows - 1) - tok * G;
  const int64_t at = (int64_t)(st.first + tok) * a.H + hk * G + hg;
  auto limit = [&](int r) { return a.causal ? min(min(r, rows - 1) / G + 1, keys) : keys; };
  const int my_limit = limit(row), least = limit(r0);
  const int nkt = (limit(st.tile * BR + BR - 1) + BT - 1) / BT;
  frag qf[NT], df[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    qf[t] = *(const frag*)((const uint16_t*)a.q + at * D + t * 16 + g * 8);
    df[t] = *(const frag*)((const uint16_t*)a.dout + at * D + t * 16 + g * 8);
  }
  const float sl2 = a.scale * kLog2e;
  const float F = grad_factor<M, D>(a), fs = F * exp2f(-M::kGradShift);
  const float l = a.lse[at] * kLog2e - M::kGradShift, dl = ((const float*)a.work)[at];
  const GradFrags<D> fr;
  const int row_in = lane / CPR, pc = lane % CPR;
  const int64_t kstride = (int64_t)a.Hkv * D, kbase = (st.first * (int64_t)a.Hkv + hk) * D;
  RowTiles kr((const uint16_t*)a.k + kbase, 0, keys, kstride, D, BT);
  RowTiles vr((const uint16_t*)a.v + kbase, 0, keys, kstride, D, BT);
  uint32_t src[NDMA];
#pragma unroll
  for (int q = 0; q < NDMA; ++q) {
    const int lr = (wave * NDMA + q) * RPD + row_in;
    src[q] = (uint32_t)((lr * kstride + (pc ^ grad_swizzle<CPR>(lr)) * 8) * 2);
  }
  f32x16_t dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[dt][e] = 0.0f;
  for (int kt = 0; kt < nkt; ++kt) {
    __syncthreads();
    const __amdgpu_buffer_rsrc_t rk = kr.next(), rv = vr.next();
#pragma unroll
    for (int q = 0; q < NDMA; ++q) {
      const int blk = wave * NDMA + q;
      dma16_buf(rk, src[q], 0, Ks + blk * 512);
      dma16_buf(rv, src[q], 0, Vs + blk * 512);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool all = kt * BT + BT <= least;
#pragma unroll
    for (int h = 0; h < BT / 32; ++h) {
      const uint16_t *Kt = Ks + h * 32 * D, *Vt = Vs + h * 32 * D;
      const int seen = my_limit - kt * BT - h * 32 - g * 4;
      f32x16_t s, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s = M::mma(*(const frag*)(Kt + fr.rows[t]), qf[t], s);
        dp = M::mma(*(const frag*)(Vt + fr.rows[t]), df[t], dp);
      }
      uint32_t pd[8];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const int off = (e >> 2) * 8 + (e & 3);
        float y0 = fa_exp2(fmaf(s[e], sl2, -l)) * (dp[e] - dl);
        float y1 = fa_exp2(fmaf(s[e + 1], sl2, -l)) * (dp[e + 1] - dl);
        if constexpr (M::kScaled) {
          y0 *= fs;
          y1 *= fs;
        }
        pd[e >> 1] = M::pack(all || off < seen ? y0 : 0.0f, all || off + 1 < seen ? y1 : 0.0f);
      }
      grad_accumulate<M, D>(dq, Kt, fr, pd);
    }
  }
  if (row >= rows) return;
  uint16_t* DQ = (uint16_t*)a.dq + at * D;
  const float sq = a.scale / F;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(uint2*)(DQ + dt * 32 + r * 8 + g * 4) =
          make_uint2(M::pack(dq[dt][r * 4] * sq, dq[dt][r * 4 + 1] * sq),
                     M::pack(dq[dt][r * 4 + 2] * sq, dq[dt][r * 4 + 3] * sq));
}

// delta, then two maxima for each workgroup of the delta kernel
size_t packed_grad_ws_bytes(int64_t T, int H) {
  return (size_t)(T * H + 2 * pg::kDeltaBlocks) * 4;
}

template <class M, int D>
static void launch_grad(PackedGradArgs a, hipStream_t stream) {
  a.delta_blocks = (int)std::min(pg::kDeltaBlocks, (a.T * a.H * (D / 8) + 255) / 256);
  const int64_t kv = max_seq_tiles(a.T, a.n_seq, 1, pg::BR) * a.Hkv;
  const int64_t q = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pg::BR) * a.Hkv;
  if (kv >= (1ll << 31) || q >= (1ll << 31))
    fail(REW_MI355X_ERR_UNSUPPORTED, "packed attention gradient: too many tiles");
  hipLaunchKernelGGL((grad_delta_kernel<M, D>), dim3((unsigned)a.delta_blocks), dim3(256), 0,
                     stream, a);
  hipLaunchKernelGGL((grad_kv_kernel<M, D>), dim3((unsigned)kv), dim3(256), 0, stream, a);
  hipLaunchKernelGGL((grad_q_kernel<M, D>), dim3((unsigned)q), dim3(256), 0, stream, a);
}
template <class M>
static void launch_grad_t(const PackedGradArgs& a, hipStream_t stream) {
  if (a.D == 32) launch_grad<M, 32>(a, stream);
  else if (a.D == 64) launch_grad<M, 64>(a, stream);
  else launch_grad<M, 128>(a, stream);
}

void launch_packed_grad(const PackedGradArgs& a, hipStream_t stream) {
  if (a.T == 0) return;
  if (a.f16) launch_grad_t<MmaF16>(a, stream);
  else launch_grad_t<MmaBf16>(a, stream);
  REW_HIP(hipGetLastError());
}

}  // namespace rew
