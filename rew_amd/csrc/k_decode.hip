// Paged attention of few rows: decode steps (PackedArgs in kernels.h).
//
// A request's rows (its new tokens times the H / Hkv heads of a KV head) are
// columns of one 32-column MFMA block, so each key and value is read once per
// KV head and 32 rows; what bounds the kernel is that stream.  A worker of the
// tile line (attn_line.h) is a workgroup of one wave, which walks its run with
// two LDS stages of 32 keys of its own, no barrier anywhere.  A tile is a long
// chain of dependent steps (about 2 us), so it takes four workers on a CU, one
// per SIMD, to ask for the memory's rate (D = 128: 64 KiB in flight per CU).
// 64 requests of 400 to 16000 keys, 32 / 8 heads x 128: 194 us, 5.7 TB/s of keys
// and values, and 8 us of joining (two workers with tiles of 64 keys took 27 us
// more, with four stages of 32 keys 48).  The partial results lie behind the output
// in its own block: two captured launches never share them.
#include <algorithm>
#include <type_traits>

#include "attn_line.h"

namespace rew {

namespace pd {
constexpr int kRows = kDecodeRows;
constexpr int BK = 32;     // keys per tile
constexpr int kLeast = 2;  // key tiles that are worth a worker
constexpr int kWaves = 8;  // of a workgroup of short tables
// The most keys that a short table has room for, and the most workgroups of a
// launch over them.  Requests of up to 1000 keys (32 / 8 heads x 128; one launch
// against runs and their join): 4 requests 11 and 15 us, 32 requests 18 and 24,
// 200 requests 82 and 79; of up to 2000 keys 4 requests 16 and 18, of up to
// 4000 keys 26 and 20.
constexpr int64_t kShortKeys = 2048, kShortGroups = 1024;
// workers on 256 CUs: one wave per SIMD (4 tiles of 32 x 128 values each fill the
// LDS), two for the smaller heads
constexpr int workers(int D) { return 256 * (D == 128 ? 4 : 8); }
}  // namespace pd

typedef TileLine<pd::kRows, pd::BK> DecodeLine;
static __device__ __forceinline__ DecodeLine decode_line(const PackedArgs& a) {
  return DecodeLine{a, a.H / a.Hkv};
}

// What a wave needs to walk key tiles of 32 rows of one request and KV head.
// lds_u16: LDS tiles of 32 keys x D.
typedef __attribute__((address_space(3))) uint16_t lds_u16;
template <class M, int D>
struct DecodeRows {
  static constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = pd::BK * D;
  static constexpr int RPD = 64 / CPR;     // key rows per DMA instruction
  static constexpr int NDMA = TILE / 512;  // instructions per K (or V) tile
  typedef typename M::frag frag;
  // where this lane reads its fragments: chunk pc of key row r holds logical chunk
  // pc ^ (r % CPR) of K and pc ^ (4 (r & 3)) of V
  int k_off[NT], v_off[DT];
  frag qf[NT];
  int row, tok, hg;     // this lane's row of the request; its token and head of the group
  int my_limit, least;  // keys that it sees, and that every row sees
  f32x16_t o[DT];
  float m_run, l_run;
  __device__ __forceinline__ DecodeRows() {
    const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
#pragma unroll
    for (int t = 0; t < NT; ++t) k_off[t] = c * D + (((2 * t + g) ^ (c % CPR)) * 8);
    const int g16 = lane >> 4, s16 = lane & 15;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int r = 4 * (g16 >> 1) + (s16 >> 2), col = dt * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
      v_off[dt] = r * D + (((col >> 3) ^ ((4 * (r & 3)) % CPR)) * 8) + (col & 7);
    }
  }
  // to row block qt of KV head hk of request r
  __device__ __forceinline__ void begin(const PackedArgs& a, const Request& r, int G, int hk,
                                        int qt) {
    const int c = threadIdx.x & 31, g = (threadIdx.x & 63) >> 5;
    row = qt * pd::kRows + c;
    tok = min(row, r.rows - 1) / G;
    hg = min(row, r.rows - 1) - tok * G;
    my_limit = r.limit(a, G, row);
    least = r.limit(a, G, qt * pd::kRows);
    const uint16_t* qp = (const uint16_t*)a.q + ((int64_t)(r.first + tok) * a.H + hk * G + hg) * D;
#pragma unroll
    for (int t = 0; t < NT; ++t) qf[t] = *(const frag*)(qp + t * 16 + g * 8);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    m_run = -INFINITY;
    l_run = 0.0f;
  }
  // Requests key tile kt: K to ks, V to vs (KEYS or VALUES alone).  The keys of a
  // tile without a page, as bits.
  template <bool KEYS, bool VALUES>
  __device__ __forceinline__ uint32_t request(const PackedArgs& a, PageWindow& win, int cap,
                                              int hk, int kt, lds_u16* ks, lds_u16* vs) const {
    const int lane = threadIdx.x & 63, row_in = lane / CPR, pc = lane % CPR;
    win.reach(kt * pd::BK);
    const uint32_t none =
        win.any_missing(kt * pd::BK, pd::BK, cap)
            ? (uint32_t)__builtin_amdgcn_ballot_w64(win.missing(kt * pd::BK + (lane & 31)))
            : 0;
    // whole tiles of whole pages: an instruction's rows lie in one page, whose
    // address the scalar unit computes
    if ((1 << a.log_page) >= RPD && none == 0 && kt * pd::BK + pd::BK <= cap) {
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int lr = q * RPD + row_in, j = kt * pd::BK + q * RPD;
        const int64_t x = ((((int64_t)win.page_uniform(j) * a.Hkv + hk) << a.log_page) +
                           (j & ((1 << a.log_page) - 1))) * D;
        const uint32_t k = row_in * D + (pc ^ (lr % CPR)) * 8;
        const uint32_t v = row_in * D + (pc ^ ((4 * (lr & 3)) % CPR)) * 8;
        if constexpr (KEYS)
          __builtin_amdgcn_global_load_lds((const uint16_t*)a.k + x + k,
                                           (lds_void*)(ks + q * 512), 16, 0, 0);
        if constexpr (VALUES)
          __builtin_amdgcn_global_load_lds((const uint16_t*)a.v + x + v,
                                           (lds_void*)(vs + q * 512), 16, 0, 0);
      }
      return none;
    }
#pragma unroll
    for (int q = 0; q < NDMA; ++q) {
      const int lr = q * RPD + row_in, j = kt * pd::BK + lr;
      const int pg = win.page(j);
      const bool there = pg >= 0 && j < cap;
      const int64_t x = ((((int64_t)(there ? pg : 0) * a.Hkv + hk) << a.log_page) +
                         (j & ((1 << a.log_page) - 1))) * D;
      const uint16_t* k = (const uint16_t*)a.k + x + (pc ^ (lr % CPR)) * 8;
      const uint16_t* v = (const uint16_t*)a.v + x + (pc ^ ((4 * (lr & 3)) % CPR)) * 8;
      if constexpr (KEYS)
        __builtin_amdgcn_global_load_lds(there ? k : g_zero_row, (lds_void*)(ks + q * 512), 16, 0,
                                         0);
      if constexpr (VALUES)
        __builtin_amdgcn_global_load_lds(there ? v : g_zero_row, (lds_void*)(vs + q * 512), 16, 0,
                                         0);
    }
    return none;
  }
  __device__ __forceinline__ f32x16_t scores(lds_u16* ks) const {
    f32x16_t s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      s = M::mma(*(__attribute__((address_space(3))) const frag*)(ks + k_off[t]), qf[t], s);
    return s;
  }
  // the softmax step of the tile's scores
  __device__ __forceinline__ void values(f32x16_t sc, int kt, uint32_t none, float sl2,
                                         uint32_t (&pk)[1][8]) {
    f32x16_t s[1] = {sc};
    const int k0 = kt * pd::BK;
    const Seen<1> vis(my_limit - k0, none, (threadIdx.x & 63) >> 5);
    const float alpha = k0 + pd::BK <= least && none == 0
                            ? soft_max<M, true, 1>(s, vis, sl2, m_run)
                            : soft_max<M, false, 1>(s, vis, sl2, m_run);
    soft_rescale<DT>(o, l_run, alpha);
    soft_exp<M, 1>(s, sl2, m_run, pk, l_run);
  }
  __device__ __forceinline__ void accumulate(lds_u16* vs, int kt, int cap,
                                             const uint32_t (&pk)[1][8]) {
    const int k0 = kt * pd::BK, lane = threadIdx.x & 63;
    if (least < min(k0 + pd::BK, cap) && any_special<M, pd::BK, D>(vs)) {
      add_special<M, pd::BK, D>(o, vs, 0, my_limit - k0, lane >> 5, value_swizzle<D>);
      clear_special<M, pd::BK, D, 64>(vs, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      union {
        uint32_t x[4];
        frag v;
      } pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf.x[i] = pk[0][u * 4 + i];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        union {
          v4s h[2];
          frag v;
        } vf;
        vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vs + v_off[dt] + u * 16 * D));
        vf.h[1] =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vs + v_off[dt] + (u * 16 + 8) * D));
        o[dt] = M::mma(vf.v, pf.v, o[dt]);
      }
    }
  }
};

template <class M, int D>
__global__ void __launch_bounds__(64, D == 128 ? 1 : 2) decode_kernel(PackedArgs a) {
  typedef DecodeRows<M, D> Rows;
  constexpr int TILE = Rows::TILE;
  __shared__ __attribute__((aligned(1024))) uint16_t S0[2 * TILE], S1[2 * TILE];
  auto at_stage = [&](auto i) -> lds_u16* {
    return (lds_u16*)(i == 0 ? S0 : S1);
  };
  const int g = threadIdx.x >> 5, c = threadIdx.x & 31;
  const int G = a.H / a.Hkv, w = blockIdx.x;
  const DecodeLine line = decode_line(a);
  const Runs runs(line, gridDim.x, pd::kLeast);
  const int from = runs.start(w), to = runs.start(w + 1);
  if (from >= to) return;
  TilePlace<DecodeLine> at;
  at.find(line, from, runs.step, runs.floor);
  const float sl2 = a.scale * pa::kLog2e;
  Rows x;

  for (int pos = from; pos < to; at.next(line)) {
    const Request r = at.r;
    const int tiles = line.item_tiles(r, at.qt), kt0 = at.kt;
    const int kt1 = min(tiles, kt0 + (to - pos));  // this run's tiles
    pos += kt1 - kt0;
    const bool real = at.s >= 0 && at.s < a.n_seq;
    x.begin(a, r, G, at.hk, at.qt);
    PageWindow win(real ? a.table + (int64_t)at.s * a.width : nullptr, real ? a.width : 0,
                   a.log_page, a.pages);
    uint32_t holes[2];  // per stage: the keys of its tile without a page
    auto request = [&](auto stage, int kt) __attribute__((always_inline)) {
      holes[stage] = x.template request<true, true>(a, win, r.cap, at.hk, kt, at_stage(stage),
                                                    at_stage(stage) + TILE);
    };
    // tile kt from its stage, once it is there, while the next one moves into
    // the other, whose reads are done
    auto step = [&](auto stage, int kt) __attribute__((always_inline)) {
      constexpr std::integral_constant<int, 1 - stage> next;
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (kt + 1 < kt1) {
        request(next, kt + 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Rows::NDMA) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_sched_barrier(0);
      uint32_t pk[1][8];
      x.values(x.scores(at_stage(stage)), kt, holes[stage], sl2, pk);
      x.accumulate(at_stage(stage) + TILE, kt, r.cap, pk);
    };
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the last item's reads of the stages)
    constexpr std::integral_constant<int, 0> s0;
    constexpr std::integral_constant<int, 1> s1;
    request(s0, kt0);
    for (int kt = kt0; kt < kt1; kt += 2) {
      step(s0, kt);
      if (kt + 1 < kt1) step(s1, kt + 1);
    }

    const float l = fa_sum_halves(x.l_run);
    if (x.row >= r.rows) continue;
    if (kt0 == 0 && kt1 == tiles)
      store_whole<M, D>(
          (uint16_t*)a.out + ((int64_t)(r.first + x.tok) * a.H + at.hk * G + x.hg) * D, x.o, l,
          g);
    else
      store_part<D>(a.work + ((int64_t)w * 2 + (kt0 == 0)) * part_floats(pd::kRows, D), pd::kRows,
                    c, x.o, x.m_run, l, g);
  }
}

// Workgroup w joins the item that run w + 1 is the first to continue: the piece
// that run w left in its second slot, then those of runs w + 1, w + 2, .. in
// their first.
template <class M, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(PackedArgs a, int workers) {
  const DecodeLine line = decode_line(a);
  const int w = blockIdx.x + 1;
  const Runs runs(line, workers, pd::kLeast);
  const int from = runs.start(w);
  if (from >= runs.total) return;
  TilePlace<DecodeLine> at;
  at.find(line, from, runs.step, runs.floor);
  const int first = from - at.kt;  // the item's first tile
  if (at.kt == 0 || first < runs.start(w - 1)) return;
  const int end = first + line.item_tiles(at.r, at.qt);
  int n = 2;
  while (runs.start(w - 1 + n) < end) ++n;
  join_rows<M, D, pd::kRows>(
      min(at.r.rows - at.qt * pd::kRows, pd::kRows), n,
      [&](int k) {
        return a.work + ((int64_t)(w - 1 + k) * 2 + (k == 0)) * part_floats(pd::kRows, D);
      },
      [&](int i) {
        const int row = at.qt * pd::kRows + i, tok = row / line.G, hg = row - tok * line.G;
        return (uint16_t*)a.out + ((int64_t)(at.r.first + tok) * a.H + at.hk * line.G + hg) * D;
      });
}

// Short tables: one workgroup of eight waves per 32 rows of a request and KV head,
// the waves taking its key tiles in turn and joining their results in LDS, so that
// one launch does it all.  K's and V's tile of a wave move apart: the next K is
// requested when this one's scores are formed, the next V behind its product.
template <class M, int D>
__global__ void __launch_bounds__(64 * pd::kWaves) decode_block_kernel(PackedArgs a) {
  using pd::kWaves;
  typedef DecodeRows<M, D> Rows;
  constexpr int TILE = Rows::TILE, NDMA = Rows::NDMA;
  // K tiles of all waves, then their results' O; V tiles
  __shared__ __attribute__((aligned(1024))) uint16_t Ks[kWaves * TILE], Vs[kWaves * TILE];
  __shared__ float2 ML[kWaves * pd::kRows];
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.H / a.Hkv, hk = blockIdx.x % a.Hkv;
  const SeqTile st = find_tile(a.starts, a.n_seq, (int)a.T, G, pd::kRows, blockIdx.x / a.Hkv);
  if (st.seq == -2) return;
  const bool real = st.real(a.n_seq);
  Request r;
  r.first = st.first;
  r.n = st.n;
  r.rows = st.n * G;
  r.len = real ? max(a.lens[st.seq], 0) : 0;
  r.cap = (int)min((int64_t)r.len, (int64_t)a.width << a.log_page);
  const int qt = st.tile, rows = min(r.rows - qt * pd::kRows, pd::kRows);
  const int tiles = (r.limit(a, G, qt * pd::kRows + pd::kRows - 1) + pd::BK - 1) / pd::BK;
  const float sl2 = a.scale * pa::kLog2e;
  Rows x;
  x.begin(a, r, G, hk, qt);
  PageWindow win(real ? a.table + (int64_t)st.seq * a.width : nullptr, real ? a.width : 0,
                 a.log_page, a.pages);
  lds_u16 *ks = (lds_u16*)Ks + wave * TILE, *vs = (lds_u16*)Vs + wave * TILE;
  uint32_t none = 0;
  if (wave < tiles) {
    none = x.template request<true, false>(a, win, r.cap, hk, wave, ks, vs);
    x.template request<false, true>(a, win, r.cap, hk, wave, ks, vs);
  }
  for (int kt = wave; kt < tiles; kt += kWaves) {
    const bool more = kt + kWaves < tiles;
    uint32_t pk[1][8], none_next = 0;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NDMA) : "memory");  // (V's behind it)
    __builtin_amdgcn_sched_barrier(0);
    const f32x16_t s = x.scores(ks);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) none_next = x.template request<true, false>(a, win, r.cap, hk, kt + kWaves, ks, vs);
    x.values(s, kt, none, sl2, pk);
    __builtin_amdgcn_sched_barrier(0);
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NDMA) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    x.accumulate(vs, kt, r.cap, pk);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) x.template request<false, true>(a, win, r.cap, hk, kt + kWaves, ks, vs);
    none = none_next;
  }
  const float l = fa_sum_halves(x.l_run);
  if (tiles <= 1) {
    if (wave == 0 && x.row < r.rows)
      store_whole<M, D>(
          (uint16_t*)a.out + ((int64_t)(r.first + x.tok) * a.H + hk * G + x.hg) * D, x.o, l, g);
    return;
  }
  // the waves' tiles are read: their O takes the same memory, half of the waves
  // at a time (32 rows of D floats are two tiles)
  const int n = min(tiles, kWaves);
  float* part = (float*)(wave < kWaves / 2 ? Ks : Vs) + (wave % (kWaves / 2)) * TILE;
  __syncthreads();
  if (c < rows) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4*)(part + c * D + dt * 32 + i * 8 + g * 4) =
            make_float4(x.o[dt][i * 4], x.o[dt][i * 4 + 1], x.o[dt][i * 4 + 2],
                        x.o[dt][i * 4 + 3]);
    if (g == 0) ML[wave * pd::kRows + c] = make_float2(x.m_run, l);
  }
  __syncthreads();
  constexpr int L = D / 4;
  for (int u = threadIdx.x; u < rows * L; u += 64 * kWaves) {
    const int i = u / L, d = u % L * 4;
    float m = -INFINITY, sum = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < n; ++k) m = __builtin_elementwise_maximum(m, ML[k * pd::kRows + i].x);
    const float mu = m == -INFINITY ? 0.0f : m;
    for (int k = 0; k < n; ++k) {
      const float2 ml = ML[k * pd::kRows + i];
      const float4 p = *(const float4*)((float*)(k < kWaves / 2 ? Ks : Vs) +
                                        (k % (kWaves / 2)) * TILE + i * D + d);
      const float f = fa_exp2(ml.x - mu);
      sum = fmaf(ml.y, f, sum);
      y[0] = fmaf(p.x, f, y[0]);
      y[1] = fmaf(p.y, f, y[1]);
      y[2] = fmaf(p.z, f, y[2]);
      y[3] = fmaf(p.w, f, y[3]);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    const int row = qt * pd::kRows + i, tok = row / G, hg = row - tok * G;
    *(uint2*)((uint16_t*)a.out + ((int64_t)(r.first + tok) * a.H + hk * G + hg) * D + d) =
        make_uint2(M::pack(y[0] * inv, y[1] * inv), M::pack(y[2] * inv, y[3] * inv));
  }
}

// Workers of a launch: no more than the tiles that the table's width allows.
static int64_t decode_workers(const PackedArgs& a) {
  const int64_t keys = ((int64_t)a.width << a.log_page) / pd::BK + 1;
  const int64_t items = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pd::kRows) * a.Hkv;
  return std::min<int64_t>(pd::workers(a.D), (items * keys + pd::kLeast - 1) / pd::kLeast);
}
// Workgroups of the one launch over short tables; 0 where the runs are better.
static int64_t short_groups(const PackedArgs& a) {
  const int64_t n = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pd::kRows) * a.Hkv;
  return (int64_t)a.width << a.log_page <= pd::kShortKeys && n <= pd::kShortGroups ? n : 0;
}
size_t decode_ws_floats(const PackedArgs& a) {
  if (short_groups(a)) return 0;
  return (size_t)decode_workers(a) * 2 * part_floats(pd::kRows, a.D);
}

template <class M, int D>
static int launch_decode(const PackedArgs& a, hipStream_t stream) {
  if (const int64_t n = short_groups(a)) {
    hipLaunchKernelGGL((decode_block_kernel<M, D>), dim3((unsigned)n), dim3(64 * pd::kWaves), 0,
                       stream, a);
    return 1;
  }
  const unsigned W = (unsigned)decode_workers(a);
  hipLaunchKernelGGL((decode_kernel<M, D>), dim3(W), dim3(64), 0, stream, a);
  if (W == 1) return 1;
  // the rows that a block is expected to hold, 1024 / D of them per workgroup
  const int64_t most = (a.max_new > 0 ? std::min(a.max_new, a.T) : a.T) * (a.H / a.Hkv);
  const unsigned y = (unsigned)((std::min<int64_t>(pd::kRows, most) * D + 1023) / 1024);
  hipLaunchKernelGGL((decode_join_kernel<M, D>), dim3(W - 1, y), dim3(256), 0, stream, a,
                     (int)W);
  return 2;
}
template <class M>
static int launch_decode_t(const PackedArgs& a, hipStream_t stream) {
  if (a.D == 32) return launch_decode<M, 32>(a, stream);
  if (a.D == 64) return launch_decode<M, 64>(a, stream);
  return launch_decode<M, 128>(a, stream);
}

int launch_paged_decode(const PackedArgs& a, hipStream_t stream) {
  return a.f16 ? launch_decode_t<MmaF16>(a, stream) : launch_decode_t<MmaBf16>(a, stream);
}

}  // namespace rew
