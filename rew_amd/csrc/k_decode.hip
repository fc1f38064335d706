// Paged attention of few rows: decode steps (PackedArgs in kernels.h).
//
// A request's rows (its new tokens times the H / Hkv heads of a KV head) are
// columns of one 32-column MFMA block, so each key and value is read once per
// KV head and 32 rows; what bounds the kernel is that stream.  A worker of the
// tile line (attn_line.h) is a workgroup of one wave, which walks its run with
// two LDS stages of 32 keys of its own, no barrier anywhere.  A tile is a long
// chain of dependent steps (about 2 us), so it takes four workers on a CU, one
// per SIMD, to ask for the memory's rate (D = 128: 64 KiB in flight per CU).
// 64 requests of 400 to 16000 keys, 32 / 8 heads x 128: 198 us, 5.5 TB/s of keys
// and values; two workers with tiles of 64 keys 225 us, with four stages of 32
// keys 246 us.  The partial results lie behind the output in its own block:
// two captured launches never share them.
#include <algorithm>
#include <type_traits>

#include "attn_line.h"

namespace rew {

namespace pd {
constexpr int kRows = kDecodeRows;
constexpr int BK = 32;     // keys per tile
constexpr int kLeast = 2;  // key tiles that are worth a worker
// workers on 256 CUs: one wave per SIMD (4 tiles of 32 x 128 values each fill the
// LDS), two for the smaller heads
constexpr int workers(int D) { return 256 * (D == 128 ? 4 : 8); }
}  // namespace pd

typedef TileLine<pd::kRows, pd::BK> DecodeLine;
static __device__ __forceinline__ DecodeLine decode_line(const PackedArgs& a) {
  return DecodeLine{a, a.H / a.Hkv};
}

template <class M, int D>
__global__ void __launch_bounds__(64, D == 128 ? 1 : 2) decode_kernel(PackedArgs a) {
  using pd::BK;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BK * D;
  constexpr int RPD = 64 / CPR;     // key rows per DMA instruction
  constexpr int NDMA = TILE / 512;  // instructions per K (or V) tile
  __shared__ __attribute__((aligned(1024))) uint16_t S0[2 * TILE], S1[2 * TILE];
  typedef __attribute__((address_space(3))) uint16_t lds_u16;
  auto at_stage = [&](auto i) -> lds_u16* {
    return (lds_u16*)(i == 0 ? S0 : S1);
  };
  const int lane = threadIdx.x, c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, w = blockIdx.x;
  const DecodeLine line = decode_line(a);
  const Runs runs(line, gridDim.x, pd::kLeast);
  const int from = runs.start(w), to = runs.start(w + 1);
  if (from >= to) return;
  TilePlace<DecodeLine> at;
  at.find(line, from, runs.x, runs.sum);

  const int row_in = lane / CPR, pc = lane % CPR;
  int k_off[NT], v_off[DT];
#pragma unroll
  for (int t = 0; t < NT; ++t) k_off[t] = c * D + (((2 * t + g) ^ (c % CPR)) * 8);
  const int g16 = lane >> 4, s16 = lane & 15;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int r = 4 * (g16 >> 1) + (s16 >> 2), col = dt * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
    v_off[dt] = r * D + (((col >> 3) ^ ((4 * (r & 3)) % CPR)) * 8) + (col & 7);
  }
  const float sl2 = a.scale * pa::kLog2e;

  for (int pos = from; pos < to; at.next(line)) {
    const Request r = at.r;
    const int tiles = line.item_tiles(r, at.qt), kt0 = at.kt;
    const int kt1 = min(tiles, kt0 + (to - pos));  // this run's tiles
    pos += kt1 - kt0;
    const int row = at.qt * pd::kRows + c;
    const int tok = min(row, r.rows - 1) / G, hg = min(row, r.rows - 1) - tok * G;
    const int my_limit = r.limit(a, G, row), least = r.limit(a, G, at.qt * pd::kRows);
    const bool real = at.s >= 0 && at.s < a.n_seq;
    frag qf[NT];
    {
      const uint16_t* qp = (const uint16_t*)a.q +
                           ((int64_t)(r.first + tok) * a.H + at.hk * G + hg) * D;
#pragma unroll
      for (int t = 0; t < NT; ++t) qf[t] = *(const frag*)(qp + t * 16 + g * 8);
    }
    PageWindow win(real ? a.table + (int64_t)at.s * a.width : nullptr, real ? a.width : 0,
                   a.log_page, a.pages);
    uint32_t holes[2];  // per stage: bit i for a key i of its tile without a page
    auto dma_tile = [&](auto stage, int kt) __attribute__((always_inline)) {
      lds_u16* st = at_stage(stage);
      win.reach(kt * BK);
      holes[stage] = win.any_missing(kt * BK, BK, r.cap)
                          ? (uint32_t)__builtin_amdgcn_ballot_w64(win.missing(kt * BK + c))
                          : 0;
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int lr = q * RPD + row_in, j = kt * BK + lr;
        const int pg = win.page(j);
        const bool there = pg >= 0 && j < r.cap;
        const int64_t x = ((((int64_t)(there ? pg : 0) * a.Hkv + at.hk) << a.log_page) +
                           (j & ((1 << a.log_page) - 1))) * D;
        const uint16_t* ks = (const uint16_t*)a.k + x + (pc ^ (lr % CPR)) * 8;
        const uint16_t* vs = (const uint16_t*)a.v + x + (pc ^ ((4 * (lr & 3)) % CPR)) * 8;
        __builtin_amdgcn_global_load_lds(there ? ks : g_zero_row, (lds_void*)(st + q * 512), 16, 0,
                                         0);
        __builtin_amdgcn_global_load_lds(there ? vs : g_zero_row,
                                         (lds_void*)(st + TILE + q * 512), 16, 0, 0);
      }
    };
    f32x16_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    // tile kt from its stage, once it is there, while the next one moves into
    // the other, whose reads are done
    auto step = [&](auto stage, int kt) __attribute__((always_inline)) {
      lds_u16* st = at_stage(stage);
      constexpr std::integral_constant<int, 1 - stage> next;
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (kt + 1 < kt1) {
        dma_tile(next, kt + 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NDMA) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16_t s[1];
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        s[0] = M::mma(*(__attribute__((address_space(3))) const frag*)(st + k_off[t]), qf[t], s[0]);
      uint32_t pk[1][8];
      float alpha;
      const int k0 = kt * BK;
      const uint32_t none = holes[stage];
      const Seen<1> vis(my_limit - k0, none, g);
      alpha = k0 + BK <= least && none == 0 ? soft_max<M, true, 1>(s, vis, sl2, m_run)
                                            : soft_max<M, false, 1>(s, vis, sl2, m_run);
      soft_rescale<DT>(o, l_run, alpha);
      soft_exp<M, 1>(s, sl2, m_run, pk, l_run);
      if (least < min(k0 + BK, r.cap) && any_special<M, BK, D>(st + TILE)) {
        add_special<M, BK, D>(o, st + TILE, my_limit - k0, g);
        clear_special<M, BK, D, 64>(st + TILE, lane);
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
          vf.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_v4s*)(st + (TILE + v_off[dt] + u * 16 * D)));
          vf.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_v4s*)(st + (TILE + v_off[dt] + (u * 16 + 8) * D)));
          o[dt] = M::mma(vf.v, pf.v, o[dt]);
        }
      }
    };
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the last item's reads of the stages)
    constexpr std::integral_constant<int, 0> s0;
    constexpr std::integral_constant<int, 1> s1;
    dma_tile(s0, kt0);
    for (int kt = kt0; kt < kt1; kt += 2) {
      step(s0, kt);
      if (kt + 1 < kt1) step(s1, kt + 1);
    }

    const float l = fa_sum_halves(l_run);
    if (row >= r.rows) continue;
    if (kt0 == 0 && kt1 == tiles)
      store_whole<M, D>(
          (uint16_t*)a.out + ((int64_t)(r.first + tok) * a.H + at.hk * G + hg) * D, o, l, g);
    else
      store_part<D>(a.work + ((int64_t)w * 2 + (kt0 == 0)) * part_floats(pd::kRows, D), pd::kRows,
                    c, o, m_run, l, g);
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
  at.find(line, from, runs.x, runs.sum);
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

// Workers of a launch: no more than the tiles that the table's width allows.
static int64_t decode_workers(const PackedArgs& a) {
  const int64_t keys = ((int64_t)a.width << a.log_page) / pd::BK + 1;
  const int64_t items = max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pd::kRows) * a.Hkv;
  return std::min<int64_t>(pd::workers(a.D), (items * keys + pd::kLeast - 1) / pd::kLeast);
}
size_t decode_ws_floats(const PackedArgs& a) {
  return (size_t)decode_workers(a) * 2 * part_floats(pd::kRows, a.D);
}

template <class M, int D>
static void launch_decode(const PackedArgs& a, hipStream_t stream) {
  const unsigned W = (unsigned)decode_workers(a);
  hipLaunchKernelGGL((decode_kernel<M, D>), dim3(W), dim3(64), 0, stream, a);
  if (W == 1) return;
  // the rows that a block is expected to hold, 1024 / D of them per workgroup
  const int64_t most = (a.max_new > 0 ? std::min(a.max_new, a.T) : a.T) * (a.H / a.Hkv);
  const unsigned y = (unsigned)((std::min<int64_t>(pd::kRows, most) * D + 1023) / 1024);
  hipLaunchKernelGGL((decode_join_kernel<M, D>), dim3(W - 1, y), dim3(256), 0, stream, a,
                     (int)W);
}
template <class M>
static void launch_decode_t(const PackedArgs& a, hipStream_t stream) {
  if (a.D == 32) launch_decode<M, 32>(a, stream);
  else if (a.D == 64) launch_decode<M, 64>(a, stream);
  else launch_decode<M, 128>(a, stream);
}

void launch_paged_decode(const PackedArgs& a, hipStream_t stream) {
  if (a.f16) launch_decode_t<MmaF16>(a, stream);
  else launch_decode_t<MmaBf16>(a, stream);
}

}  // namespace rew
