// The gradients of packed attention (PackedGradArgs in kernels.h), without
// anything of size rows x keys in memory.
//
// delta = dout . out per row is taken from out and what its rounding left (out
// alone would put out's rounding into every dS, next to dS's own): by a first
// launch for float16, by the dQ kernel for bfloat16 (2 % of the case below,
// forward pass included).  The dQ kernel gives each workgroup 128 rows and
// walks their keys, dQ staying in registers; the last launch gives each
// workgroup 128 keys of one KV head and walks the rows that see them, dK and dV
// staying in registers.  Both recompute P = exp(S - lse), so the scores are
// formed twice: 7 products of rows x keys x D where 5 would do, for sums whose
// order never changes (a single pass would add dQ across workgroups with
// atomics).  The rows of the H / Hkv heads of a KV head are walked together, so
// the sum over the group is part of the accumulation.  6 documents of up to 4000
// tokens, 32 / 8 heads x 128, bf16: 272 us (267 GFLOP, 0.98 PFLOP/s) and 401 us
// (357 GFLOP, 0.89 PFLOP/s), passes back to back.
//
// In each product one operand stays in registers and the other is read from
// LDS; S and dP come out with the operand in registers along the lanes, so P
// and dS go from the accumulators straight into the next product, as in the
// forward kernel, and the LDS operand of that product is read transposed.
#include <algorithm>
#include <type_traits>

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
// Per row (D / 8 lanes each of T H rows) what the scores and dP are added to:
// kGradShift - log2(e) lse, and -delta.  float16 has no room for dS at any scale:
// it is stored as F dS, F a power of two that takes a bound on |dS| to 2^15.  Of the
// rows and keys that share a sum nothing else may set it, or another document's (or
// head's, or an unseen row's) large gradient would take this one's bits: dQ has
// an F per row i, from
//   |dS_ij| <= D max|dout_i| max|V seen by i| + |delta_i|,
// dK one per key j, from
//   |dS_ij| <= D max|dout of rows that see j| max|V_j| + max|delta of these rows|,
// maxima over finite values.  So this kernel also leaves each row's max|dout| and
// |delta|, and each key's max|V|, in the order in which a KV head's rows and keys are
// read.  (bfloat16 needs none: its dQ kernel forms -lse and -delta from its own rows.)
struct GradMaxima {
  const float2* rows;  // [Hkv][T H / Hkv]: (max|dout|, |delta|)
  const float* values; // [Hkv][T]: max|V|
  __device__ __forceinline__ explicit GradMaxima(const PackedGradArgs& a)
      : rows((const float2*)((const float*)a.work + 2 * a.T * a.H)),
        values((const float*)a.work + 4 * a.T * a.H) {}
};
__device__ __forceinline__ float finite_abs(float x) {
  return fabsf(x) < INFINITY ? fabsf(x) : 0.0f;
}
// F for a bound (1 without one)
__device__ __forceinline__ float grad_factor(float bound) {
  if (!(bound > 0.0f && bound < INFINITY)) return 1.0f;
  int e;
  (void)frexpf(bound, &e);  // bound < 2^e
  return ldexpf(1.0f, min(max(15 - e, -60), 60));
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// Adds to s, rest and most what eight values x of a row of out, y of dout and z of
// what rounding took from out give: dout . out, dout . rest, max |out|.
template <class M>
__device__ __forceinline__ void delta_terms(uint4 x, uint4 y, uint2 z, float& s, float& rest,
                                            float& most) {
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[2] = {z.x, z.y};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float y0 = M::lo(ys[k]), y1 = M::hi(ys[k]), x0 = M::lo(xs[k]), x1 = M::hi(xs[k]);
    s = fmaf(x0, y0, s);
    s = fmaf(x1, y1, s);
    const int sh = (k & 1) * 16;
    rest = fmaf((float)(int8_t)(zs[k >> 1] >> sh), y0, rest);
    rest = fmaf((float)(int8_t)(zs[k >> 1] >> (sh + 8)), y1, rest);
    most = fmaxf(most, fmaxf(fabsf(x0), fabsf(x1)));
  }
}
template <class M, int D>
__global__ void __launch_bounds__(256) grad_delta_kernel(PackedGradArgs a) {
  constexpr int L = D / 8;
  const int64_t rows = a.T * a.H, keys = a.T * a.Hkv, step = gridDim.x * (256ll / L);
  const int ch = threadIdx.x % L, G = a.H / a.Hkv;
  const int64_t first = blockIdx.x * (256ll / L) + threadIdx.x / L;
  float *neg_lse = (float*)a.work, *neg_delta = neg_lse + rows;
  const GradMaxima maxima(a);
  for (int64_t i = first; i < rows; i += step) {
    const uint4 x = ((const uint4*)a.out)[i * L + ch], y = ((const uint4*)a.dout)[i * L + ch];
    float s = 0.0f, rest = 0.0f, row = 0.0f, most = 0.0f;
    delta_terms<M>(x, y, ((const uint2*)a.rest)[i * L + ch], s, rest, row);
    for (uint32_t w : {y.x, y.y, y.z, y.w})
      most = fmaxf(most, fmaxf(finite_abs(M::lo(w)), finite_abs(M::hi(w))));
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) {
      s += __shfl_xor(s, d);
      rest += __shfl_xor(rest, d);
      row = fmaxf(row, __shfl_xor(row, d));
      most = fmaxf(most, __shfl_xor(most, d));
    }
    s = fmaf(rest, fmaxf(row, M::kRestLeast) * M::kRestStep, s);
    if (ch == 0) {
      neg_lse[i] = M::kGradShift - a.lse[i] * pg::kLog2e;
      neg_delta[i] = -s;
      const int64_t t = i / a.H;
      const int h = (int)(i - t * a.H), hk = h / G;
      ((float2*)maxima.rows)[(hk * a.T + t) * G + h - hk * G] = make_float2(most, finite_abs(s));
    }
  }
  for (int64_t i = first; i < keys; i += step) {
    const uint4 x = ((const uint4*)a.v)[i * L + ch];
    float most = 0.0f;
    for (uint32_t w : {x.x, x.y, x.z, x.w})
      most = fmaxf(most, fmaxf(finite_abs(M::lo(w)), finite_abs(M::hi(w))));
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    const int64_t t = i / a.Hkv;
    if (ch == 0) ((float*)maxima.values)[(i - t * a.Hkv) * a.T + t] = most;
  }
}
// F of the lane's key in a dK, dV workgroup (keys k0 .. of KV head hk, 32 kw + c the
// lane's).  Its eight waves call it.
template <int D>
__device__ __forceinline__ float key_factor(const PackedGradArgs& a, const SeqTile& st, int rows,
                                            int hk, int k0, int kw) {
  __shared__ float2 part[8 + 4];
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5, G = a.H / a.Hkv;
  const int key = k0 + kw * 32 + c;
  const GradMaxima maxima(a);
  const float2* of = maxima.rows + (hk * a.T + st.first) * G;  // of row r of the sequence
  float2 x = make_float2(0.0f, 0.0f);
  auto add = [](float2& m, float2 y) { m.x = fmaxf(m.x, y.x), m.y = fmaxf(m.y, y.y); };
  // the rows that see all keys of the workgroup
  const int from = a.causal ? (k0 + pg::BR) * G : 0;
  for (int r = from + (int)threadIdx.x; r < rows; r += 512) add(x, of[r]);
  part[threadIdx.x >> 6] = make_float2(wave_max(x.x), wave_max(x.y));
  x = make_float2(0.0f, 0.0f);
  if (a.causal) {  // those of the wave's own tokens, from each key's token on
    const int last = min((key + 1) * G, rows);
    for (int r = key * G + g; r < last; r += 2) add(x, of[r]);
    x = make_float2(fa_max_halves(x.x), fa_max_halves(x.y));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float2 y = make_float2(__shfl_down(x.x, d, 32), __shfl_down(x.y, d, 32));
      add(x, y);  // (the last d lanes have their own again)
    }
    if (lane == 0) part[8 + kw] = x;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) add(x, part[w]);
  if (a.causal)
    for (int w = kw + 1; w < 4; ++w) add(x, part[8 + w]);
  const float v = key < st.n ? maxima.values[hk * a.T + st.first + key] : 0.0f;
  return grad_factor(fmaf(D * x.x, v, x.y));
}
// F of the lane's row in a dQ workgroup: it sees the keys below my_limit (my_limit -
// least < 32), every row of its wave those below `least`, of the workgroup those
// below block_least.  Its four waves call it.
template <int D>
__device__ __forceinline__ float row_factor(const PackedGradArgs& a, const SeqTile& st, int hk,
                                            int my_limit, int least, int block_least, float dout,
                                            float delta) {
  __shared__ float part[4];
  const int lane = threadIdx.x & 63;
  const float* of = GradMaxima(a).values + hk * a.T + st.first;
  float v = 0.0f;
  for (int j = threadIdx.x; j < block_least; j += 256) v = fmaxf(v, of[j]);
  part[threadIdx.x >> 6] = wave_max(v);
  __syncthreads();
  v = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  float w = 0.0f;
  for (int j = block_least + lane; j < least; j += 64) w = fmaxf(w, of[j]);
  v = fmaxf(v, wave_max(w));
  // the wave's own tokens' keys, up to each row's
  const int j = least + (lane & 31);
  float x = j < st.n && least < st.n ? of[j] : 0.0f;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) x = fmaxf(x, __shfl_up(x, d, 32));
  const float own = __shfl(x, max(my_limit - least - 1, 0), 32);
  if (my_limit > least) v = fmaxf(v, own);
  return grad_factor(fmaf(D * dout, v, finite_abs(delta)));
}

// Where a lane reads its fragments in an LDS tile of D columns, in bytes.
// `rows`, for the operand whose rows lie along the lanes: row c, chunk g; chunk
// 2t + g is at rows ^ 32 t.  `cols`, for the transposed read
// (ds_read_b64_tr_b16) of 8 rows' columns 16 (G & 1) ..: columns 32 dt on are
// at cols ^ 64 dt, the next 8 rows at (cols ^ 32) + 16 D.  A tile starts at a
// multiple of 256 bytes, so its address can be added first and one XOR per
// fragment remains; kept as registers, the offsets would be 16 for each array.
template <int D>
struct GradFrags {
  uint32_t rows, cols;
  __device__ __forceinline__ GradFrags() {
    constexpr int CPR = D / 8;
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
    const int g16 = lane >> 4, s16 = lane & 15;
    rows = (c * D + ((g ^ grad_swizzle<CPR>(c)) * 8)) * 2;
    const int r = 4 * (g16 >> 1) + (s16 >> 2), col = 16 * (g16 & 1) + 4 * (s16 & 3);
    cols = (r * D + (((col >> 3) ^ grad_swizzle<CPR>(r)) * 8) + (col & 7)) * 2;
  }
};
typedef __attribute__((address_space(3))) const char lds_char;
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
// Makes x a value that the compiler cannot compute ahead (the XORs of a
// loop-invariant address would be hoisted, into registers that are not there).
__device__ __forceinline__ void opaque(uint32_t& x) { asm volatile("" : "+v"(x)); }
// Reads at an offset: in an array (while a DMA into another array is in
// flight, which the compiler then need not wait for) or at a whole address.
struct InTile {
  lds_char* p;
  __device__ __forceinline__ lds_char* operator()(uint32_t off) const { return p + off; }
};
struct Whole {
  __device__ __forceinline__ lds_char* operator()(uint32_t at) const {
    return (lds_char*)(uintptr_t)at;
  }
};
template <class F, class At>
__device__ __forceinline__ F grad_read(At at, uint32_t off) {
  return *(__attribute__((address_space(3))) const F*)at(off);
}
template <class M, int D, class At>
__device__ __forceinline__ typename M::frag grad_cols(At at, uint32_t off, uint32_t up, int plus) {
  union {
    v4s h[2];
    typename M::frag v;
  } f;
  f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at(off) + plus));
  f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at(up) + (plus + 16 * D)));
  return f.v;
}
// acc[dt] += (columns of 32 rows of a tile)^T x the packed values of those
// rows, for N tiles (addresses cols[i], values pk[i]) in turn; the fragments
// are read four products ahead.
template <class M, int D, int N, class At>
__device__ __forceinline__ void grad_accumulate(f32x16_t (*const (&acc)[N])[D / 32],
                                                At at, const uint32_t (&cols)[N],
                                                const uint32_t (*const (&pk)[N])[8]) {
  typedef typename M::frag frag;
  constexpr int PER = 2 * (D / 32), ALL = N * PER, AHEAD = ALL < 4 ? ALL : 4;
  frag p[N][2], f[AHEAD];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      union {
        uint32_t w[4];
        frag v;
      } x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] = (*pk[n])[u * 4 + i];
      p[n][u] = x.v;
    }
  auto read = [&](int i) {  // product i: tile i / PER, columns 32 dt, rows 16 u
    const int n = i / PER, dt = i % PER / 2, u = i & 1;
    f[i % AHEAD] =
        grad_cols<M, D>(at, cols[n] ^ (64 * dt), cols[n] ^ (64 * dt + 32), u * 32 * D);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
  for (int i = 0; i < ALL; ++i) {
    const int n = i / PER, dt = i % PER / 2, u = i & 1;
    (*acc[n])[dt] = M::mma(f[i % AHEAD], p[n][u], (*acc[n])[dt]);
    if (i + AHEAD < ALL) read(i + AHEAD);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
  for (int i = 0; i < ALL; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i + AHEAD < ALL) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
}

// ---- dK, dV -----------------------------------------------------------------------------
//
// Eight waves over 128 keys in two groups of four; wave w of a group owns keys
// 32 w .. + 31, and the groups take turns at the blocks of 32 rows.  Halving
// the rows of each wave halves the longest workgroup, which is what a causal
// batch waits for (the first keys of a long sequence are seen by all its
// rows); the halves meet in LDS at the end.  dK and dV take half of the
// registers, so K and V are read from LDS like the rows.
//
// Waves w of both groups share a SIMD and alternate between a phase of products
// (dV and dK of their last block, S and dP of the next) and one of
// exponentials, a barrier apart, so that each phase runs beside the other
// group's other one; left to themselves both waves of a SIMD did the same at
// the same time (39 % of the matrix core's cycles in use).  A group requests
// its next block by DMA when a phase of exponentials begins, into the buffer
// that its products have just finished with, and waits for it at that
// phase's end.
template <class M, int D>
__global__ void __launch_bounds__(512, 1) grad_kv_kernel(PackedGradArgs a) {
  using namespace pg;
  typedef typename M::frag frag;
  typedef __attribute__((address_space(3))) uint16_t lds_u16;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, RPD = 64 / CPR;
  constexpr int BLK = 32 * D;               // elements of 32 rows of Q (or dout)
  constexpr int NDMA = 2 * BLK / 512 / 4;   // DMA instructions per wave and block
  __shared__ __attribute__((aligned(1024))) uint16_t S[4 * 2 * BLK];  // [group][slot] Q, dout
  __shared__ __attribute__((aligned(1024))) uint16_t Ks[BR * D];
  // V, then the meeting of the row halves (32 KiB)
  __shared__ __attribute__((aligned(1024))) uint16_t Vs[BR * D < 16384 ? 16384 : BR * D];
  __shared__ __attribute__((aligned(256))) float R[4 * 64];  // [group][slot] -lse, -delta
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5, kw = wave & 3, grp = wave >> 2;
  const int G = a.H / a.Hkv, hk = blockIdx.x % a.Hkv, rank = blockIdx.x / a.Hkv;
  SeqTile st = a.n_seq <= kLevelSeqs ? rising_tile(a.starts, a.n_seq, (int)a.T, 1, BR, rank)
                                     : find_tile(a.starts, a.n_seq, (int)a.T, 1, BR, rank);
  if (st.seq == -2) return;
  // causal work falls with the key: the order of rising work runs backwards
  if (a.n_seq <= kLevelSeqs) st.tile = (st.n - 1) / BR - st.tile;
  const int rows = st.real(a.n_seq) ? st.n * G : 0;
  const int k0 = st.tile * BR, wk = k0 + kw * 32, key = wk + c;  // this lane's key
  const int64_t kstride = (int64_t)a.Hkv * D;
  const DivBy by_g(G);
  const GradFrags<D> fr;
  const int row_in = lane / CPR, pc = lane % CPR;
#pragma unroll
  for (int i = 0; i < BR * D / 512 / 8; ++i) {
    const int blk = wave + i * 8, lr = blk * RPD + row_in;
    const int64_t at = (st.first + min(k0 + lr, st.n - 1)) * kstride + hk * D;
    const int ch = (pc ^ grad_swizzle<CPR>(lr)) * 8;
    dma16((const uint16_t*)a.k + at + ch, Ks + blk * 512);
    dma16((const uint16_t*)a.v + at + ch, Vs + blk * 512);
  }
  f32x16_t dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.0f;
  const float sl2 = a.scale * kLog2e;
  // (P has the factor 2^kGradShift already)
  const float fs = M::kScaled ? key_factor<D>(a, st, rows, hk, k0, kw) * exp2f(-M::kGradShift) : 1.0f;
  const int64_t base = (int64_t)st.first * a.H + hk * G;  // row (tok, hg): base + tok H + hg
  const float* stats = (const float*)a.work;
  // causal: rows of tokens before the workgroup's first key do not see it
  const int r0 = a.causal ? k0 * G / 64 * 64 : 0;
  const int n = (rows - r0 + 63) / 64;  // blocks of each group (the last may be empty)
  auto row_of = [&](int m) { return r0 + (2 * m + grp) * 32; };
  auto slot = [&](int m) { return grp * 2 + (m & 1); };

  // groups that divide a block: its rows are whole tokens' heads, at the same
  // offsets in each block, and only the scalar unit has addresses to compute
  // (tokens behind the last read as zeros): 8 % fewer cycles than by rows
  const bool whole = NDMA >= 2 && 32 % G == 0;
  const int log_g = __builtin_ctz(G);
  uint32_t row_at[NDMA < 2 ? 1 : NDMA / 2];
#pragma unroll
  for (int i = 0; i < NDMA / 2; ++i) {
    const int lr = (kw + i * 4) * RPD + row_in;
    row_at[i] = (uint32_t)(((lr / G * a.H + lr % G) * D + (pc ^ grad_swizzle<CPR>(lr)) * 8) * 2);
  }

  auto request = [&](int m) {
    const int w0 = row_of(m);
    uint16_t* s = S + slot(m) * 2 * BLK;
    if (whole) {
      const int tok = w0 >> log_g;
      const int64_t at = (base + (int64_t)tok * a.H) * D;
      const int64_t left = w0 < rows ? ((int64_t)(st.n - 1 - tok) * a.H + G) * D * 2 : 0;
      const uint32_t bytes = (uint32_t)min(left, (int64_t)0x7fffffff);
      const __amdgpu_buffer_rsrc_t rq = fa_rsrc((const uint16_t*)a.q + at, bytes);
      const __amdgpu_buffer_rsrc_t rd = fa_rsrc((const uint16_t*)a.dout + at, bytes);
#pragma unroll
      for (int i = 0; i < NDMA / 2; ++i) {
        dma16_buf(rq, row_at[i], 0, s + (kw + i * 4) * 512);
        dma16_buf(rd, row_at[i], 0, s + BLK + (kw + i * 4) * 512);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NDMA; ++i) {
        const int x = kw + i * 4, blk = x % (BLK / 512), lr = blk * RPD + row_in;
        const bool q = x < BLK / 512;
        int hg;
        const int tok = by_g.div(min(w0 + lr, rows - 1), hg);
        const int64_t at =
            (base + (int64_t)tok * a.H + hg) * D + (pc ^ grad_swizzle<CPR>(lr)) * 8;
        dma16((const uint16_t*)(q ? a.q : a.dout) + at, s + x * 512);
      }
    }
    if (kw == 0) {  // lanes 0..31: -lse, 32..63: -delta
      int hg;
      const int tok = by_g.div(min(w0 + c, rows - 1), hg);
      const float* src = stats + (g ? a.T * a.H : 0) + base + (int64_t)tok * a.H + hg;
      __builtin_amdgcn_global_load_lds(src, (lds_void*)(R + slot(m) * 64), 4, 0, 0);
    }
  };
  // whether any row of block m sees any of this wave's keys (row r sees key j
  // from r = j G on, if causal)
  auto live = [&](int m) {
    const int w0 = row_of(m);
    return w0 < rows && (!a.causal || w0 + 31 >= wk * G);
  };
  f32x16_t x, dp;
  float4 l4[4];
  uint32_t pp[8], pd[8];
  // An infinity or NaN of a row's Q makes its lse, one of its dout its delta such
  // a value, and 0 times it would reach dK and dV of keys that do not see the row.
  // So a block with such an lse or delta (`odd`, the same in all waves of the
  // group) goes another way.  Beside its scores the infinities and NaN of dout are
  // added to dV of the keys that see them, by column: P = 0 there only by underflow.
  // (dK needs nothing: the row's dS is NaN.)
  bool odd = false;
  auto is_odd = [&](float stat) {  // (lane's of the block's 64 values)
    odd = __builtin_amdgcn_ballot_w64(!(fabsf(stat) < INFINITY)) != 0;
  };
  auto add_odd = [&](int m) __attribute__((always_inline)) {
    if (!odd || !live(m)) return;
    uint32_t l = lane;
    opaque(l);
    lds_u16* Dt = (lds_u16*)(S + slot(m) * 2 * BLK + BLK);
    if (!any_special<M, 32, D>(Dt, l)) return;
    const int w0 = row_of(m);
    add_special<M, 32, D>(dv, Dt, a.causal ? key * G - w0 : 0, rows - w0, (int)l >> 5,
                          grad_swizzle<CPR>);
  };
  // Before its second products they are zeros, each wave's own part of the block.
  auto clean = [&](int m) {
    if (!odd) return;
    uint32_t l = lane;
    opaque(l);
#pragma unroll 1
    for (int i = 0; i < NDMA; ++i) {
      u32x4_t* p = (u32x4_t*)(S + slot(m) * 2 * BLK + (kw + i * 4) * 512 + l * 8);
      u32x4_t w = *p;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] ^= special<M>(w[j]);
      *p = w;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  auto scores = [&](int m) {
    if (!live(m)) return;
    const uint16_t* Qt = S + slot(m) * 2 * BLK;
    const float* rt = R + slot(m) * 64 + g * 4;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const float4 d4 = *(const float4*)(rt + 32 + e4 * 8);
      const float d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[e4 * 4 + i] = 0.0f;
        dp[e4 * 4 + i] = d[i];
      }
    }
    // Q, dout, K and V fragments are read three k-steps ahead (two: 2 % more cycles;
    // four: spills, whose reloads wait for every DMA)
    constexpr int AHEAD = NT < 3 ? NT : 3;
    uint32_t qa = lds_at(Qt) + fr.rows, ka = lds_at(Ks) + kw * BLK * 2 + fr.rows,
             va = lds_at(Vs) + kw * BLK * 2 + fr.rows;
    opaque(ka);
    opaque(va);
    frag f[AHEAD][4];
    auto read = [&](int t) {
      f[t % AHEAD][0] = grad_read<frag>(Whole(), qa ^ (32 * t));
      f[t % AHEAD][1] = grad_read<frag>(Whole(), ka ^ (32 * t));
      f[t % AHEAD][2] = grad_read<frag>(Whole(), (qa ^ (32 * t)) + BLK * 2);
      f[t % AHEAD][3] = grad_read<frag>(Whole(), va ^ (32 * t));
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) read(t);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      x = M::mma(f[t % AHEAD][0], f[t % AHEAD][1], x);
      dp = M::mma(f[t % AHEAD][2], f[t % AHEAD][3], dp);
      if (t + AHEAD < NT) read(t + AHEAD);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4 + 4 * AHEAD, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      if (t + AHEAD < NT) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
    }
  };
  // (before the next request: the compiler makes a read of R wait for a DMA into it)
  auto read_lse = [&](int m) {
    const float* rt = R + slot(m) * 64 + g * 4;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) l4[e4] = *(const float4*)(rt + e4 * 8);
  };
  auto values = [&](int m) {
    if (!live(m)) return;
    const int w0 = row_of(m);
    // rows of the block that see this lane's key: span of them from lo
    const int lo = a.causal ? key * G - w0 - g * 4 : -64;
    const uint32_t span = (uint32_t)max(rows - w0 - g * 4 - lo, 0);
    auto go = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const float l[4] = {l4[e4].x, l4[e4].y, l4[e4].z, l4[e4].w};
        float p[4], ds[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e4 * 4 + i;
          if constexpr (masked) {  // (selects, no branches)
            const bool see = (uint32_t)(e4 * 8 + i - lo) < span;
            dp[e] = see ? dp[e] : 0.0f;
            p[i] = fa_exp2(fmaf(x[e], sl2, l[i]));
            p[i] = see ? p[i] : 0.0f;
          } else {
            p[i] = fa_exp2(fmaf(x[e], sl2, l[i]));
          }
          ds[i] = p[i] * dp[e];
          if constexpr (M::kScaled) ds[i] *= fs;
        }
        pp[e4 * 2] = M::pack(p[0], p[1]);
        pp[e4 * 2 + 1] = M::pack(p[2], p[3]);
        pd[e4 * 2] = M::pack(ds[0], ds[1]);
        pd[e4 * 2 + 1] = M::pack(ds[2], ds[3]);
      }
    };
    if (w0 + 32 <= rows && (!a.causal || w0 >= (wk + 31) * G)) go(std::false_type());
    else go(std::true_type());
  };
  auto accumulate = [&](int m) {
    if (!live(m)) return;
    const uint32_t at = lds_at(S + slot(m) * 2 * BLK) + fr.cols;
    grad_accumulate<M, D, 2>({&dv, &dk}, Whole(), {at + BLK * 2, at}, {&pp, &pd});
  };
  auto vm_wait = []() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };

  // half-step   0     1     2           3           ...  2n - 1    2n
  // group 0     S 0   exp 0 dKV 0, S 1  exp 1            exp n-1   dKV n-1
  // group 1     -     S 0   exp 0       dKV 0, S 1       ..        exp n-1, dKV n-1
  if (n > 0) {
    request(0);
    vm_wait();
    block_barrier_fa();
    if (grp == 1) block_barrier_fa();
    __builtin_amdgcn_s_setprio(1);
    is_odd(R[slot(0) * 64 + lane]);
    add_odd(0);
    scores(0);
    block_barrier_fa();
    for (int m = 1; m < n; ++m) {
      __builtin_amdgcn_s_setprio(0);
      read_lse(m - 1);
      request(m);
      values(m - 1);
      vm_wait();
      clean(m - 1);
      block_barrier_fa();
      __builtin_amdgcn_s_setprio(1);
      const float stat = R[slot(m) * 64 + lane];
      accumulate(m - 1);
      is_odd(stat);
      add_odd(m);
      scores(m);
      block_barrier_fa();
    }
    __builtin_amdgcn_s_setprio(0);
    read_lse(n - 1);
    values(n - 1);
    clean(n - 1);
    block_barrier_fa();
    accumulate(n - 1);
    if (grp == 0) block_barrier_fa();
  }
  // the two row halves meet: wave w keeps dK and takes the other's, wave w + 4
  // likewise dV
  typedef float f32x4_t __attribute__((ext_vector_type(4)));
  f32x4_t* X = (f32x4_t*)Vs;  // [8 waves][4][64 lanes]
  vm_wait();  // (V's own DMA, where there were no rows)
  auto meet = [&](f32x16_t(&mine)[DT], f32x16_t(&other)[DT], void* to, float m) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        X[(wave * 4 + i) * 64 + lane] = (f32x4_t){other[dt][i * 4], other[dt][i * 4 + 1],
                                                  other[dt][i * 4 + 2], other[dt][i * 4 + 3]};
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4_t v = X[((wave ^ 4) * 4 + i) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[dt][i * 4 + j] += v[j];
      }
    }
    if (key >= st.n) return;
    uint16_t* out = (uint16_t*)to + (st.first + key) * kstride + hk * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(uint2*)(out + dt * 32 + r * 8 + g * 4) =
            make_uint2(M::pack(mine[dt][r * 4] * m, mine[dt][r * 4 + 1] * m),
                       M::pack(mine[dt][r * 4 + 2] * m, mine[dt][r * 4 + 3] * m));
  };
  // (both branches pass the same barriers)
  if (grp == 0) meet(dk, dv, a.dk, a.scale * exp2f(-M::kGradShift) / fs);
  else meet(dv, dk, a.dv, exp2f(-M::kGradShift));
}

// ---- dQ -----------------------------------------------------------------------------------
//
// Four waves of 32 rows, as in the forward kernel: Q and dout of a row in
// registers, K and V tiles of 64 keys by DMA, one ahead, lse and delta of the
// row one value per lane.
template <class M, int D>
__global__ void __launch_bounds__(256, 2) grad_q_kernel(PackedGradArgs a) {
  using namespace pg;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BT * D, RPD = 64 / CPR;
  constexpr int NDMA = TILE / 512 / 4;
  __shared__ __attribute__((aligned(1024))) uint16_t K0[TILE], K1[TILE], V0[TILE], V1[TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, hk = blockIdx.x % a.Hkv, rank = blockIdx.x / a.Hkv;
  const SeqTile st = a.n_seq <= kLevelSeqs
                         ? rising_tile(a.starts, a.n_seq, (int)a.T, G, BR, rank)
                         : find_tile(a.starts, a.n_seq, (int)a.T, G, BR, rank);
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
  float l, dl, fs = 1.0f;  // (fs: with P's factor 2^kGradShift, F)
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
  auto dma_tile = [&](uint16_t* ks, uint16_t* vs) {
    const __amdgpu_buffer_rsrc_t rk = kr.next(), rv = vr.next();
#pragma unroll
    for (int q = 0; q < NDMA; ++q) {
      const int blk = wave * NDMA + q;
      dma16_buf(rk, src[q], 0, ks + blk * 512);
      dma16_buf(rv, src[q], 0, vs + blk * 512);
    }
  };
  f32x16_t dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[dt][e] = 0.0f;
  typedef __attribute__((address_space(3))) uint16_t lds_u16;
  const int block_least = limit(st.tile * BR);
  auto tile = [&](uint16_t* ks, const uint16_t* vs, uint16_t* ks_n, uint16_t* vs_n, int kt) {
    // (as in the forward kernel's V: the same answer in all waves)
    const bool special = block_least < min(kt * BT + BT, keys) &&
                         any_special<M, BT, D>((lds_u16*)ks);
    if (kt + 1 < nkt) dma_tile(ks_n, vs_n);
#pragma unroll
    for (int h = 0; h < BT / 32; ++h) {
      const InTile Kt{(lds_char*)(ks + h * 32 * D)}, Vt{(lds_char*)(vs + h * 32 * D)};
      uint32_t rows_at = fr.rows, cols_at = fr.cols;
      opaque(rows_at);
      opaque(cols_at);
      f32x16_t s, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = 0.0f;
        dp[e] = dl;
      }
      constexpr int AHEAD = NT < 3 ? NT : 3;
      frag f[AHEAD][2];
      auto read = [&](int t) {
        f[t % AHEAD][0] = grad_read<frag>(Kt, rows_at ^ (32 * t));
        f[t % AHEAD][1] = grad_read<frag>(Vt, rows_at ^ (32 * t));
      };
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) read(t);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s = M::mma(f[t % AHEAD][0], qf[t], s);
        dp = M::mma(f[t % AHEAD][1], df[t], dp);
        if (t + AHEAD < NT) read(t + AHEAD);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        if (t + AHEAD < NT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      uint32_t pd[8];
      auto values = [&](auto masked) __attribute__((always_inline)) {
        const int seen = my_limit - kt * BT - h * 32 - g * 4;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const int off = (e >> 2) * 8 + (e & 3);
          float y[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            y[i] = fa_exp2(fmaf(s[e + i], sl2, l)) * dp[e + i];
            if constexpr (M::kScaled) y[i] *= fs;
            if constexpr (masked) y[i] = off + i < seen ? y[i] : 0.0f;
          }
          pd[e >> 1] = M::pack(y[0], y[1]);
        }
      };
      if (kt * BT + BT <= least) values(std::false_type());
      else values(std::true_type());
      if (special) {
        lds_u16* half = (lds_u16*)(ks + h * 32 * D);
        add_special<M, 32, D>(dq, half, 0, my_limit - kt * BT - h * 32, g, grad_swizzle<CPR>);
        __syncthreads();
        clear_special<M, 32, D, 256>(half, threadIdx.x);
        __syncthreads();
      }
      grad_accumulate<M, D, 1>({&dq}, Kt, {cols_at}, {&pd});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if (nkt > 0) dma_tile(K0, V0);  // (on its way while delta is formed)
  if constexpr (M::kScaled) {
    l = ((const float*)a.work)[at];
    dl = ((const float*)a.work)[a.T * a.H + at];
    float dout = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint4 y;
      __builtin_memcpy(&y, &df[t], 16);
      for (uint32_t w : {y.x, y.y, y.z, y.w})
        dout = fmaxf(dout, fmaxf(finite_abs(M::lo(w)), finite_abs(M::hi(w))));
    }
    fs = row_factor<D>(a, st, hk, my_limit, uniform(least), block_least, fa_max_halves(dout), dl) *
         exp2f(-M::kGradShift);
  } else {
    float s = 0.0f, rest = 0.0f, most = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t i = at * D + t * 16 + g * 8;
      uint4 y;
      __builtin_memcpy(&y, &df[t], 16);
      delta_terms<M>(*(const uint4*)((const uint16_t*)a.out + i), y, *(const uint2*)(a.rest + i),
                     s, rest, most);
    }
    most = fmaxf(fa_max_halves(most), M::kRestLeast);
    s = fa_sum_halves(fmaf(rest, most * M::kRestStep, s));
    l = M::kGradShift - a.lse[at] * kLog2e;
    dl = -s;
    if (g == 0 && row < rows) {  // (for the dK, dV kernel)
      ((float*)a.work)[at] = l;
      ((float*)a.work)[a.T * a.H + at] = dl;
    }
  }
  if (nkt > 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kt = 0; kt < nkt; kt += 2) {
      tile(K0, V0, K1, V1, kt);
      if (kt + 1 < nkt) tile(K1, V1, K0, V0, kt + 1);
    }
  }
  if (row >= rows) return;
  uint16_t* DQ = (uint16_t*)a.dq + at * D;
  const float sq = a.scale * exp2f(-M::kGradShift) / fs;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *(uint2*)(DQ + dt * 32 + r * 8 + g * 4) =
          make_uint2(M::pack(dq[dt][r * 4] * sq, dq[dt][r * 4 + 1] * sq),
                     M::pack(dq[dt][r * 4 + 2] * sq, dq[dt][r * 4 + 3] * sq));
}

// two values per row, and for float16 two maxima per row and one per key
size_t packed_grad_ws_bytes(int64_t T, int H, int Hkv, bool f16) {
  return (size_t)(f16 ? 4 * T * H + T * Hkv : 2 * T * H) * 4;
}

template <class M, int D>
static void launch_grad(const PackedGradArgs& a, hipStream_t stream) {
  const int64_t kv = max_seq_tiles(a.T, a.n_seq, 1, pg::BR) * a.Hkv;
  const int64_t q = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pg::BR) * a.Hkv;
  if constexpr (M::kScaled) {
    const int64_t blocks = std::min(pg::kDeltaBlocks, (a.T * a.H * (D / 8) + 255) / 256);
    hipLaunchKernelGGL((grad_delta_kernel<M, D>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  }
  hipLaunchKernelGGL((grad_q_kernel<M, D>), dim3((unsigned)q), dim3(256), 0, stream, a);
  hipLaunchKernelGGL((grad_kv_kernel<M, D>), dim3((unsigned)kv), dim3(512), 0, stream, a);
}
template <class M>
static void launch_grad_t(const PackedGradArgs& a, hipStream_t stream) {
  if (a.D == 32) launch_grad<M, 32>(a, stream);
  else if (a.D == 64) launch_grad<M, 64>(a, stream);
  else launch_grad<M, 128>(a, stream);
}

int launch_packed_grad(const PackedGradArgs& a, hipStream_t stream) {
  if (a.T == 0) return 0;
  if (a.f16) launch_grad_t<MmaF16>(a, stream);
  else launch_grad_t<MmaBf16>(a, stream);
  REW_HIP(hipGetLastError());
  return a.f16 ? 3 : 2;
}

}  // namespace rew
