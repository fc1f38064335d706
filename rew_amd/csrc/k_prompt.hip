// Attention over packed sequences and paged caches (PackedArgs in kernels.h).
//
// The H / Hkv query heads of a KV head read the same keys, so the rows of a
// tile are (token, head of the group) pairs in token order: 128 of them per
// workgroup share each K and V tile, whatever the group's size, and a causal
// tile ends with the last of its few tokens.  Four waves of 32 rows; key
// tiles of 64 keys move by DMA into two LDS stages.  S^T = K Q^T leaves the
// scores of one row in a lane and its neighbour lane ^ 32, so the softmax's
// running max and sum need one exchange; O^T = V^T P^T takes the
// probabilities from the accumulators, with V read transposed from LDS.
//
// Rounding: scores, max, sum and O in float32; the probabilities are rounded
// to the operands' 16 bits for the second product (not in the sum, which the
// gradients need), the output once.
#include <algorithm>

#include "attn_device.h"
#include "kernels.h"

namespace rew {

namespace pa {
constexpr int BR = 128;  // rows per workgroup
}  // namespace pa

template <class M, int D, bool PAGED>
__global__ void __launch_bounds__(256, 2) prompt_attn_kernel(PackedArgs a) {
  using namespace pa;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BK * D;
  constexpr int RPD = 64 / CPR;        // key rows per DMA instruction
  constexpr int NDMA = TILE / 512 / 4;  // instructions per wave and K (or V) tile
  __shared__ __attribute__((aligned(1024))) uint16_t Ks0[TILE], Ks1[TILE], Vs0[TILE], Vs1[TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv;
  const int hk = blockIdx.x % a.Hkv;
  const SeqTile st = find_tile(a.starts, a.n_seq, (int)a.T, G, BR, blockIdx.x / a.Hkv,
                               PAGED ? kDecodeRows : 0);
  if (st.seq == -2) return;
  const bool real = st.real(a.n_seq);
  const int rows = st.n * G;
  const int len = !real ? 0 : PAGED ? max(a.lens[st.seq], 0) : st.n;
  const int cap = !real ? 0 : PAGED ? (int)min((int64_t)len, (int64_t)a.width << a.log_page) : len;
  // keys that row r sees: [0, limit(r)), growing with r
  auto limit = [&](int r) -> int {
    const int t = min(r, rows - 1) / G;
    return min(max(a.causal ? len - st.n + t + 1 : len, 0), cap);
  };
  const int r0 = st.tile * BR + wave * 32;
  const int row = r0 + c;
  const int tok = min(row, rows - 1) / G, hg = min(row, rows - 1) - tok * G;
  const int my_limit = limit(row), least = limit(r0);
  const int nkt = (limit(st.tile * BR + BR - 1) + BK - 1) / BK;

  frag qf[NT];
  {
    const uint16_t* qp = (const uint16_t*)a.q +
                         ((int64_t)(st.first + tok) * a.H + hk * G + hg) * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) qf[t] = *(const frag*)(qp + t * 16 + g * 8);
  }

  // chunk pc of key row r holds logical chunk pc ^ (r % CPR) of K and
  // pc ^ (4 (r & 3)) of V: both reads then spread over the LDS banks
  const int row_in = lane / CPR, pc = lane % CPR;
  const int64_t kstride = (int64_t)a.Hkv * D;
  const uint16_t* K = (const uint16_t*)a.k + (PAGED ? 0 : (st.first * (int64_t)a.Hkv + hk) * D);
  const uint16_t* V = (const uint16_t*)a.v + (PAGED ? 0 : (st.first * (int64_t)a.Hkv + hk) * D);
  RowTiles kr(K, 0, cap, kstride, D, BK), vr(V, 0, cap, kstride, D, BK);
  uint32_t k_src[NDMA], v_src[NDMA];
  int key_row[NDMA];
#pragma unroll
  for (int q = 0; q < NDMA; ++q) {
    const int r = (wave * NDMA + q) * RPD + row_in;
    key_row[q] = r;
    const int ck = (pc ^ (r % CPR)) * 8, cv = (pc ^ ((4 * (r & 3)) % CPR)) * 8;
    k_src[q] = PAGED ? (uint32_t)ck : (uint32_t)((r * kstride + ck) * 2);
    v_src[q] = PAGED ? (uint32_t)cv : (uint32_t)((r * kstride + cv) * 2);
  }
  PageWindow win(PAGED && real ? a.table + (int64_t)st.seq * a.width : nullptr,
                 PAGED && real ? a.width : 0, a.log_page, a.pages);
  auto dma_tile = [&](uint16_t* ks, uint16_t* vs, int kt) {  // (kt: one after another)
    if constexpr (PAGED) {
      if (kt >= nkt) return;
      win.reach(kt * BK);
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int j = kt * BK + key_row[q];
        const int pg = win.page(j);
        const bool there = pg >= 0 && j < cap;
        const int64_t at = ((((int64_t)(there ? pg : 0) * a.Hkv + hk) << a.log_page) +
                            (j & ((1 << a.log_page) - 1))) * D;
        const int blk = wave * NDMA + q;
        dma16(there ? K + at + k_src[q] : g_zero_row, ks + blk * 512);
        dma16(there ? V + at + v_src[q] : g_zero_row, vs + blk * 512);
      }
    } else {
      const __amdgpu_buffer_rsrc_t rk = kr.next(), rv = vr.next();
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int blk = wave * NDMA + q;
        dma16_buf(rk, k_src[q], 0, ks + blk * 512);
        dma16_buf(rv, v_src[q], 0, vs + blk * 512);
      }
    }
  };

  int k_off[NT], v_off[DT];
#pragma unroll
  for (int t = 0; t < NT; ++t) k_off[t] = c * D + (((2 * t + g) ^ (c % CPR)) * 8);
  const int g16 = lane >> 4, s16 = lane & 15;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int r = 4 * (g16 >> 1) + (s16 >> 2), col = dt * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
    v_off[dt] = r * D + (((col >> 3) ^ ((4 * (r & 3)) % CPR)) * 8) + (col & 7);
  }

  f32x16_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const float sl2 = a.scale * kLog2e;

  // missing: whether a key of this tile has no page, and the window that knows
  auto k_tile = [&](const uint16_t* ks, const uint16_t* vs, uint16_t* ks_n, uint16_t* vs_n,
                    int kt) {
    const bool holes = PAGED && win.any_missing(kt * BK, cap);
    const PageWindow w = win;
    if (kt + 1 < nkt) dma_tile(ks_n, vs_n, kt + 1);
    f32x16_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[0] = M::mma(*(const frag*)(ks + k_off[t]), qf[t], s[0]);
      s[1] = M::mma(*(const frag*)(ks + k_off[t] + 32 * D), qf[t], s[1]);
    }
    uint32_t pk[2][8];
    float alpha;
    const int k0 = kt * BK;
    if (k0 + BK <= least && !holes)
      alpha = soft_step<M, true>(s, 0, g, sl2, pk, m_run, l_run, [](int) { return false; });
    else if (!holes)
      alpha = soft_step<M, false>(s, my_limit - k0, g, sl2, pk, m_run, l_run,
                                  [](int) { return false; });
    else
      alpha = soft_step<M, false>(s, my_limit - k0, g, sl2, pk, m_run, l_run,
                                  [&](int off) { return w.missing(k0 + off); });
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      union {
        uint32_t w[4];
        frag v;
      } pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf.w[i] = pk[u >> 1][(u & 1) * 4 + i];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint16_t* p = vs + v_off[dt] + u * 16 * D;
        union {
          v4s h[2];
          frag v;
        } vf;
        vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p);
        vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 8 * D));
        o[dt] = M::mma(vf.v, pf.v, o[dt]);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if (nkt > 0) {
    dma_tile(Ks0, Vs0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kt = 0; kt < nkt; kt += 2) {
      k_tile(Ks0, Vs0, Ks1, Vs1, kt);
      if (kt + 1 < nkt) k_tile(Ks1, Vs1, Ks0, Vs0, kt + 1);
    }
  }

  const float l = fa_sum_halves(l_run);
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays NaN)
  if (row >= rows) return;
  const int64_t at = (int64_t)(st.first + tok) * a.H + hk * G + hg;
  if (a.lse && g == 0) a.lse[at] = (m_run - M::kShift + __log2f(l)) * kLn2;
  uint16_t* O = (uint16_t*)a.out + at * D;
  float most = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float* x = (float*)&o[dt] + r * 4;
      const uint2 w = make_uint2(M::pack(x[0] * inv, x[1] * inv), M::pack(x[2] * inv, x[3] * inv));
      *(uint2*)(O + dt * 32 + r * 8 + g * 4) = w;
      if (a.rest) {  // (uniform)
        const float y[4] = {M::lo(w.x), M::hi(w.x), M::lo(w.y), M::hi(w.y)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          most = fmaxf(most, fabsf(y[i]));
          x[i] = fmaf(x[i], inv, -y[i]);
        }
      }
    }
  if (!a.rest) return;
  // (lanes of a row, l and l ^ 32, are both here)
  most = fa_max_halves(most);
  const float per_step = most > 0.0f ? 1.0f / (most * M::kRestStep) : 0.0f;
  int8_t* rest = a.rest + at * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float q = rintf(fminf(fmaxf(o[dt][r * 4 + i] * per_step, -127.0f), 127.0f));
        w |= ((uint32_t)(int)q & 255u) << (8 * i);
      }
      *(uint32_t*)(rest + dt * 32 + r * 8 + g * 4) = w;
    }
}

template <class M, int D>
static void launch_prompt(const PackedArgs& a, unsigned grid, hipStream_t stream) {
  if (a.table)
    hipLaunchKernelGGL((prompt_attn_kernel<M, D, true>), dim3(grid), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((prompt_attn_kernel<M, D, false>), dim3(grid), dim3(256), 0, stream, a);
}
template <class M>
static void launch_prompt_t(const PackedArgs& a, unsigned grid, hipStream_t stream) {
  if (a.D == 32) launch_prompt<M, 32>(a, grid, stream);
  else if (a.D == 64) launch_prompt<M, 64>(a, grid, stream);
  else launch_prompt<M, 128>(a, grid, stream);
}

const char* packed_attn_variant(const PackedArgs& a) {
  return a.table ? "paged_attn" : "packed_attn";
}

// Paged: requests of few rows go to the decode kernels; so do all where the
// caller expects no other (they are right for any number of rows).
int launch_packed_attn(const PackedArgs& a, hipStream_t stream) {
  if (a.T == 0) return 0;
  const int64_t G = a.H / a.Hkv;
  if (a.table) {
    const int64_t most = a.max_new > 0 ? std::min(a.max_new, a.T) : a.T;
    const bool all = most * G <= kDecodeRows;
    launch_paged_decode(a, all, stream);
    if (all) {
      REW_HIP(hipGetLastError());
      return 2;
    }
  }
  const int64_t tiles = max_seq_tiles(a.T, a.n_seq, G, pa::BR) * a.Hkv;
  if (tiles >= (1ll << 31)) fail(REW_MI355X_ERR_UNSUPPORTED, "packed attention: too many tiles");
  if (a.f16) launch_prompt_t<MmaF16>(a, (unsigned)tiles, stream);
  else launch_prompt_t<MmaBf16>(a, (unsigned)tiles, stream);
  REW_HIP(hipGetLastError());
  return a.table ? 3 : 1;
}

}  // namespace rew
