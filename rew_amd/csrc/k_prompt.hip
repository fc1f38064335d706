// Attention of many rows over packed sequences and paged caches (PackedArgs in
// kernels.h).
//
// The H / Hkv query heads of a KV head read the same keys, so the rows of a
// block are (token, head of the group) pairs in token order: 128 of them per
// workgroup share each K and V tile, whatever the group's size, and a causal
// block ends with the last of its few tokens.  Four waves of 32 rows; key
// tiles of 64 keys move by DMA into two LDS stages.  S^T = K Q^T leaves the
// scores of one row in a lane and its neighbour lane ^ 32, so the softmax's
// running max and sum need one exchange; O^T = V^T P^T takes the
// probabilities from the accumulators, with V read transposed from LDS.  Two
// workgroups fit a CU, so that one's products can run beside the other's
// exponentials; nothing but chance puts them there.
//
// 8 ragged prompts of up to 4001 tokens, 32 / 8 heads x 128, bf16 (173 GFLOP):
// 198 us, 0.87 PFLOP/s, at the 1.8 GHz that the card holds under this load (a
// large product reaches 1.36 PFLOP/s).  The matrix cores are busy for 47 % of the
// cycles and the vector ALUs for 50 %; 39 % of the former have one of the latter
// beside them, and for a fifth of the time neither works.  Wave priorities
// changed nothing; the scores of tile i + 1 formed beside the exponentials of tile i
// in one wave need more registers than there are and were no faster.
//
// Rounding: scores, max, sum and O in float32; the probabilities are rounded
// to the operands' 16 bits for the second product (not in the sum, which the
// gradients need), the output once.
#include <algorithm>

#include "attn_line.h"

namespace rew {

namespace pa {
constexpr int BR = 128;           // rows per block
constexpr int kChunkSlots = 512;  // workgroups that run at once: two on each of 256 CUs
constexpr int kPieceTiles = 16;   // key tiles that are worth a piece of a block
}  // namespace pa

// Tokens of a sequence or request whose rows one block holds, as a lane sees
// them.
struct BlockRows {
  int row, tok, hg;  // this lane's row of the sequence; its token, its head of the group
  __device__ __forceinline__ BlockRows(int block, int rows, int G) {
    const int wave = threadIdx.x >> 6, c = threadIdx.x & 31;
    row = block * pa::BR + wave * 32 + c;
    const int r = min(row, rows - 1);
    tok = r / G;
    hg = r - tok * G;
  }
};

// O (unnormalised), running max and this lane's part of the running sum of a
// block's rows over key tiles [kt0, kt1) of a sequence that starts at token
// `first` (or, PAGED, of the request with block table `table`): `cap` keys,
// this lane's row sees those below my_limit, every row of the wave those below
// `least`, every row of the block those below block_least.  Four waves; ends
// with a barrier behind the last read of LDS.
template <class M, int D, bool PAGED>
__device__ __forceinline__ void attend_block(const PackedArgs& a, const BlockRows& br, int first,
                                             const int32_t* table, int hk, int cap, int my_limit,
                                             int least, int block_least, int kt0, int kt1,
                                             f32x16_t (&o)[D / 32],
                                             float& m_run, float& l_run) {
  using namespace pa;
  typedef typename M::frag frag;
  typedef __attribute__((address_space(3))) uint16_t lds_u16;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BK * D;
  constexpr int RPD = 64 / CPR;         // key rows per DMA instruction
  constexpr int NDMA = TILE / 512 / 4;  // instructions per wave and K (or V) tile
  __shared__ __attribute__((aligned(1024))) uint16_t Ks0[TILE], Ks1[TILE], Vs0[TILE], Vs1[TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, tok = br.tok, hg = br.hg;
  frag qf[NT];
  {
    const uint16_t* qp = (const uint16_t*)a.q +
                         ((int64_t)(first + tok) * a.H + hk * G + hg) * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) qf[t] = *(const frag*)(qp + t * 16 + g * 8);
  }

  // chunk pc of key row r holds logical chunk pc ^ (r % CPR) of K and
  // pc ^ (4 (r & 3)) of V: both reads then spread over the LDS banks
  const int row_in = lane / CPR, pc = lane % CPR;
  const int64_t kstride = (int64_t)a.Hkv * D;
  const uint16_t* K = (const uint16_t*)a.k + (PAGED ? 0 : (first * (int64_t)a.Hkv + hk) * D);
  const uint16_t* V = (const uint16_t*)a.v + (PAGED ? 0 : (first * (int64_t)a.Hkv + hk) * D);
  RowTiles kr(K, kt0 * BK, cap, kstride, D, BK), vr(V, kt0 * BK, cap, kstride, D, BK);
  uint32_t k_src[NDMA], v_src[NDMA];
#pragma unroll
  for (int q = 0; q < NDMA; ++q) {
    const int r = (wave * NDMA + q) * RPD + row_in;
    const int ck = (pc ^ (r % CPR)) * 8, cv = (pc ^ ((4 * (r & 3)) % CPR)) * 8;
    k_src[q] = PAGED ? (uint32_t)(row_in * D + ck) : (uint32_t)((r * kstride + ck) * 2);
    v_src[q] = PAGED ? (uint32_t)(row_in * D + cv) : (uint32_t)((r * kstride + cv) * 2);
  }
  PageWindow win(table, table ? a.width : 0, a.log_page, a.pages);
  uint64_t none_next = 0;  // of the tile last requested: bit i for a key i without a page
  auto dma_tile = [&](uint16_t* ks, uint16_t* vs, int kt) {  // (kt: one after another)
    if constexpr (PAGED) {
      win.reach(kt * BK);
      none_next = win.any_missing(kt * BK, BK, cap)
                      ? __builtin_amdgcn_ballot_w64(win.missing(kt * BK + lane))
                      : 0;
      // whole tiles of whole pages: an instruction's rows lie in one page, whose
      // address the scalar unit computes beside the vector unit's work
      if ((1 << a.log_page) >= RPD && none_next == 0 && kt * BK + BK <= cap) {
#pragma unroll
        for (int q = 0; q < NDMA; ++q) {
          const int blk = wave * NDMA + q, j = kt * BK + blk * RPD;
          const int64_t at = ((((int64_t)win.page_uniform(j) * a.Hkv + hk) << a.log_page) +
                              (j & ((1 << a.log_page) - 1))) * D;
          dma16(K + at + k_src[q], ks + blk * 512);
          dma16(V + at + v_src[q], vs + blk * 512);
        }
        return;
      }
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int j = kt * BK + (wave * NDMA + q) * RPD + row_in;
        const int pg = win.page(j);
        const bool there = pg >= 0 && j < cap;
        const int64_t at = ((((int64_t)(there ? pg : 0) * a.Hkv + hk) << a.log_page) +
                            (j & ((1 << a.log_page) - 1)) - row_in) * D;
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

#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
  m_run = -INFINITY;
  l_run = 0.0f;
  const float sl2 = a.scale * kLog2e;

  auto k_tile = [&](const uint16_t* ks, uint16_t* vs, uint16_t* ks_n, uint16_t* vs_n,
                    int kt) {
    const uint64_t none = none_next;
    if (kt + 1 < kt1) dma_tile(ks_n, vs_n, kt + 1);
    f32x16_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
    // the K fragments of k-step t + AHEAD are read while step t multiplies
    constexpr int AHEAD = NT < 3 ? NT : 3;
    frag kf[AHEAD][2];
    auto ld_k = [&](int t) {
      kf[t % AHEAD][0] = *(const frag*)(ks + k_off[t]);
      kf[t % AHEAD][1] = *(const frag*)(ks + k_off[t] + 32 * D);
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) ld_k(t);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[0] = M::mma(kf[t % AHEAD][0], qf[t], s[0]);
      s[1] = M::mma(kf[t % AHEAD][1], qf[t], s[1]);
      if (t + AHEAD < NT) ld_k(t + AHEAD);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      if (t + AHEAD < NT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    uint32_t pk[2][8];
    float alpha;
    const int k0 = kt * BK;
    const Seen<2> vis(my_limit - k0, none, g);
    alpha = k0 + BK <= least && none == 0 ? soft_max<M, true, 2>(s, vis, sl2, m_run)
                                          : soft_max<M, false, 2>(s, vis, sl2, m_run);
    soft_rescale<DT>(o, l_run, alpha);
    soft_exp<M, 2>(s, sl2, m_run, pk, l_run);
    // (the same answer in all waves)
    if (block_least < min(k0 + BK, cap) && any_special<M, BK, D>((lds_u16*)vs)) {
      add_special<M, BK, D>(o, (lds_u16*)vs, 0, my_limit - k0, g, value_swizzle<D>);
      __syncthreads();
      clear_special<M, BK, D, 256>((lds_u16*)vs, threadIdx.x);
      __syncthreads();
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
  if (kt0 < kt1) {
    dma_tile(Ks0, Vs0, kt0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kt = kt0; kt < kt1; kt += 2) {
      k_tile(Ks0, Vs0, Ks1, Vs1, kt);
      if (kt + 1 < kt1) k_tile(Ks1, Vs1, Ks0, Vs0, kt + 1);
    }
  }
}

template <class M, int D>
__global__ void __launch_bounds__(256, 2) prompt_attn_kernel(PackedArgs a) {
  using namespace pa;
  constexpr int DT = D / 32;
  const int G = a.H / a.Hkv, g = (threadIdx.x & 63) >> 5;
  const int hk = blockIdx.x % a.Hkv;
  // Under causality a block's work grows with its place in its sequence: the
  // heaviest start first (8 ragged prompts, 8 times the blocks that run at once:
  // 219 us in sequence order, 200 us so; the search costs 0.3 us).
  const int rank = blockIdx.x / a.Hkv;
  const SeqTile st = a.causal && a.n_seq <= kLevelSeqs
                         ? rising_tile(a.starts, a.n_seq, (int)a.T, G, BR, rank)
                         : find_tile(a.starts, a.n_seq, (int)a.T, G, BR, rank);
  if (st.seq == -2) return;
  const int rows = st.n * G, len = st.real(a.n_seq) ? st.n : 0;
  // keys that row r sees: [0, limit(r)), growing with r
  auto limit = [&](int r) { return a.causal ? min(min(r, rows - 1) / G + 1, len) : len; };
  const BlockRows br(st.tile, rows, G);
  f32x16_t o[DT];
  float m_run, l_run;
  attend_block<M, D, false>(a, br, st.first, nullptr, hk, len, limit(br.row),
                            uniform(limit(st.tile * BR + (threadIdx.x >> 6) * 32)),
                            limit(st.tile * BR), 0, (limit(st.tile * BR + BR - 1) + BK - 1) / BK, o,
                            m_run, l_run);
  const float l = fa_sum_halves(l_run);
  if (br.row >= rows) return;
  const int64_t at = (int64_t)(st.first + br.tok) * a.H + hk * G + br.hg;
  if (!a.rest) {
    store_whole<M, D>((uint16_t*)a.out + at * D, o, l, g);
    return;
  }
  if (g == 0) a.lse[at] = (m_run - M::kShift + __log2f(l)) * kLn2;
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays NaN)
  uint16_t* O = (uint16_t*)a.out + at * D;
  float most = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float* x = (float*)&o[dt] + r * 4;
      const uint2 w = make_uint2(M::pack(x[0] * inv, x[1] * inv), M::pack(x[2] * inv, x[3] * inv));
      *(uint2*)(O + dt * 32 + r * 8 + g * 4) = w;
      const float y[4] = {M::lo(w.x), M::hi(w.x), M::lo(w.y), M::hi(w.y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        most = fmaxf(most, fabsf(y[i]));
        x[i] = fmaf(x[i], inv, -y[i]);
      }
    }
  // (lanes of a row, l and l ^ 32, are both here)
  most = fa_max_halves(most);
  const float per_step = 1.0f / (fmaxf(most, M::kRestLeast) * M::kRestStep);
  int8_t* rest = a.rest + at * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // 1.5 2^23 + x holds x, rounded, in its low bits (|x| <= 127 by the step)
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        b[i] = __float_as_uint(fmaf(o[dt][r * 4 + i], per_step, 0x1.8p23f));
      *(uint32_t*)(rest + dt * 32 + r * 8 + g * 4) =
          __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400) |
          __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    }
}

// ---- chunks over a paged cache -----------------------------------------------------
//
// A chunk of a few hundred tokens over a long cache is few blocks of many key
// tiles, so a request's blocks may each be split over P workgroups, which leave
// partial results for a second launch to join.  A piece costs about six tiles'
// time (its 64 KiB are written and read), so P is the number of times that the
// request's middle block holds C tiles, rounded, C being a CU's share of all
// tiles or at least kPieceTiles: no block is split where the blocks fill the
// CUs by themselves (2048 tokens over 30001 keys: 1.07 ms, 0.97 PFLOP/s; cut
// into 512 equal runs, 1.30 ms and 140 us of joining).  Single tokens of other
// requests in the same step are blocks of few rows here: 13 requests of 1 to
// 539 new tokens over up to 4400 keys take 44 us and 8 us of joining, with
// pieces of 8 or 12 tiles the same, of 20 more.
struct ChunkPlan {
  const PackedArgs& a;
  int G, C;
  // what this lane's request has: row blocks, workgroups per block and KV head
  struct Share {
    Request r;
    int blocks, P;
  };
  static __device__ __forceinline__ int tiles_of(const PackedArgs& a, int G, const Request& r,
                                                 int qt) {
    return (r.limit(a, G, qt * pa::BR + pa::BR - 1) + pa::BK - 1) / pa::BK;
  }
  __device__ __forceinline__ Share share(int base, int& floor) const {  // (floor: SeqRows)
    Share x;
    x.r = lane_request(a, G, base, floor);
    x.blocks = (x.r.rows + pa::BR - 1) / pa::BR;
    x.P = x.blocks ? max((tiles_of(a, G, x.r, x.blocks / 2) + C / 2) / C, 1) : 0;
    return x;
  }
  __device__ __forceinline__ explicit ChunkPlan(const PackedArgs& a_)
      : a(a_), G(a_.H / a_.Hkv), C(0x7fffffff / 2) {
    int n = 0, floor = 0;
    for (int base = -1; base <= a.n_seq; base += 64) {
      const Share x = share(base, floor);
      n += wave_sum(x.blocks ? x.blocks * tiles_of(a, G, x.r, x.blocks / 2) * a.Hkv : 0);
    }
    C = max((n + pa::kChunkSlots - 1) / pa::kChunkSlots, pa::kPieceTiles);
  }
  // The 64 requests from `base`, one per lane, those of the longest pieces first,
  // so that these start first.
  struct Sorted {
    Share x;          // of request base + lane
    int s, blocks, P; // of the request that has this lane's place in the order
    __device__ __forceinline__ Sorted(const ChunkPlan& plan, int base, int& floor)
        : x(plan.share(base, floor)) {
      const int lane = threadIdx.x & 63;
      const int piece =
          x.blocks ? tiles_of(plan.a, plan.G, x.r, x.blocks / 2) / x.P : -1;
      const int n = uniform(min(plan.a.n_seq + 1 - base, 64));
      int rank = lane;
      if (n > 1) {
        rank = 0;
        for (int j = 0; j < n; ++j) {
          const int other = __builtin_amdgcn_readlane(piece, j);
          rank += other > piece || (other == piece && j < lane);
        }
        if (lane >= n) rank = lane;
      }
      const int from = __builtin_amdgcn_ds_permute(rank * 4, lane) * 4;
      s = base + from / 4;
      blocks = __builtin_amdgcn_ds_bpermute(from, x.blocks);
      P = __builtin_amdgcn_ds_bpermute(from, x.P);
    }
  };
};
// Workgroup `idx` of the plan's (or, SPLIT, of the split blocks' joins, one per
// block and KV head).
template <bool SPLIT>
struct ChunkPlace {
  bool found;
  int s, hk, qt, part, P, slot;  // slot: of this block's first partial result, if P > 1
  Request r;
  __device__ __forceinline__ ChunkPlace(const ChunkPlan& plan, int idx) : found(false) {
    int slots = 0, floor = 0;
    const int Hkv = plan.a.Hkv;
    for (int base = -1; base <= plan.a.n_seq; base += 64) {
      const ChunkPlan::Sorted x(plan, base, floor);
      const int pieces = x.P > 1 ? x.blocks * x.P * Hkv : 0;
      const int mine = !SPLIT ? x.blocks * x.P * Hkv : x.P > 1 ? x.blocks * Hkv : 0;
      const int sum = wave_scan(mine), psum = wave_scan(pieces);
      const int total = __builtin_amdgcn_readlane(sum, 63);
      if (idx >= total) {
        idx -= total;
        slots += __builtin_amdgcn_readlane(psum, 63);
        continue;
      }
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > idx));
      found = true;
      s = __builtin_amdgcn_readlane(x.s, at);
      r = request_from(x.x.r, s - base);
      P = __builtin_amdgcn_readlane(x.P, at);
      const int blocks = __builtin_amdgcn_readlane(x.blocks, at);
      int u = idx - __builtin_amdgcn_readlane(sum - mine, at);
      // KV heads first: with eight of them a head's workgroups share an XCD (those
      // whose indices agree mod 8 do) and its L2; the blocks of most keys first
      hk = u % Hkv;
      u /= Hkv;
      part = SPLIT ? 0 : u % P;
      qt = blocks - 1 - (SPLIT ? u : u / P);
      slot = slots + __builtin_amdgcn_readlane(psum - pieces, at) + (qt * Hkv + hk) * P;
      return;
    }
  }
};

template <class M, int D>
__global__ void __launch_bounds__(256, 2) chunk_attn_kernel(PackedArgs a) {
  using namespace pa;
  constexpr int DT = D / 32;
  const int G = a.H / a.Hkv, g = (threadIdx.x & 63) >> 5;
  const ChunkPlace<false> at(ChunkPlan(a), blockIdx.x);
  if (!at.found) return;
  const Request& r = at.r;
  const int tiles = ChunkPlan::tiles_of(a, G, r, at.qt);
  const bool real = at.s >= 0 && at.s < a.n_seq;
  const BlockRows br(at.qt, r.rows, G);
  f32x16_t o[DT];
  float m_run, l_run;
  attend_block<M, D, true>(a, br, r.first, real ? a.table + (int64_t)at.s * a.width : nullptr,
                           at.hk, r.cap, r.limit(a, G, br.row),
                           uniform(r.limit(a, G, at.qt * BR + (threadIdx.x >> 6) * 32)),
                           r.limit(a, G, at.qt * BR),
                           (int)((int64_t)tiles * at.part / at.P),
                           (int)((int64_t)tiles * (at.part + 1) / at.P), o, m_run, l_run);
  const float l = fa_sum_halves(l_run);
  if (br.row >= r.rows) return;
  if (at.P == 1)
    store_whole<M, D>(
        (uint16_t*)a.out + ((int64_t)(r.first + br.tok) * a.H + at.hk * G + br.hg) * D, o, l, g);
  else
    store_part<D>(a.work + (int64_t)(at.slot + at.part) * part_floats(BR, D), BR,
                  br.row - at.qt * BR, o, m_run, l, g);
}

template <class M, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(PackedArgs a) {
  using namespace pa;
  const ChunkPlace<true> at(ChunkPlan(a), blockIdx.x);
  if (!at.found) return;
  const int G = a.H / a.Hkv;
  join_rows<M, D, BR>(
      min(at.r.rows - at.qt * BR, BR), at.P,
      [&](int k) { return a.work + (int64_t)(at.slot + k) * part_floats(BR, D); },
      [&](int i) {
        const int row = at.qt * BR + i, tok = row / G, hg = row - tok * G;
        return (uint16_t*)a.out + ((int64_t)(at.r.first + tok) * a.H + at.hk * G + hg) * D;
      });
}

// ---- launches ---------------------------------------------------------------------------

// Whether the caller expects a request whose rows fill more than one block of the
// decode kernels; both they and the chunk kernels are right for any rows.
static bool expects_chunks(const PackedArgs& a) {
  const int64_t most = a.max_new > 0 ? std::min(a.max_new, a.T) : a.T;
  return most * (a.H / a.Hkv) > kDecodeRows;
}
// Split blocks have P >= 2 and P <= 4/3 of their tiles / C, all tiles together at
// most kChunkSlots C.
constexpr int kChunkPieces = pa::kChunkSlots * 4 / 3;
size_t paged_ws_bytes(const PackedArgs& a) {
  // (the finest cut, the decode kernels' blocks and tiles)
  const int64_t keys = ((int64_t)a.width << a.log_page) / 32 + 1;
  if (max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, kDecodeRows) * keys >= (1ll << 31) / a.Hkv)
    fail(REW_MI355X_ERR_UNSUPPORTED, "paged attention: 2^31 key tiles or more");
  return (expects_chunks(a) ? (size_t)kChunkPieces * part_floats(pa::BR, a.D)
                            : decode_ws_floats(a)) * 4;
}

int64_t packed_threads(int64_t T, int64_t n_seq, int H, int Hkv, bool grad) {
  const int64_t rows = (max_seq_tiles(T, n_seq, H / Hkv, pa::BR) * Hkv + kChunkPieces) * 256;
  // (dK, dV: workgroups of 512 threads, 128 keys each)
  return grad ? std::max(rows, max_seq_tiles(T, n_seq, 1, 128) * Hkv * 512) : rows;
}

template <class M, int D>
static int launch_prompt(const PackedArgs& a, hipStream_t stream) {
  if (a.table && !expects_chunks(a)) return launch_paged_decode(a, stream);
  const int64_t tiles = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pa::BR) * a.Hkv;
  if (!a.table) {
    hipLaunchKernelGGL((prompt_attn_kernel<M, D>), dim3((unsigned)tiles), dim3(256), 0, stream, a);
    return 1;
  }
  hipLaunchKernelGGL((chunk_attn_kernel<M, D>), dim3((unsigned)tiles + kChunkPieces), dim3(256), 0,
                     stream, a);
  // 32 rows of a block per workgroup
  hipLaunchKernelGGL((chunk_join_kernel<M, D>), dim3(kChunkPieces / 2, 4), dim3(256), 0, stream, a);
  return 2;
}
template <class M>
static int launch_prompt_t(const PackedArgs& a, hipStream_t stream) {
  if (a.D == 32) return launch_prompt<M, 32>(a, stream);
  if (a.D == 64) return launch_prompt<M, 64>(a, stream);
  return launch_prompt<M, 128>(a, stream);
}

const char* packed_attn_variant(const PackedArgs& a) {
  return !a.table ? "packed_attn" : expects_chunks(a) ? "paged_attn_chunks" : "paged_attn_decode";
}

int launch_packed_attn(const PackedArgs& a, hipStream_t stream) {
  if (a.T == 0) return 0;
  const int n = a.f16 ? launch_prompt_t<MmaF16>(a, stream) : launch_prompt_t<MmaBf16>(a, stream);
  REW_HIP(hipGetLastError());
  return n;
}

}  // namespace rew
