// Paged attention of few rows: decode steps (PackedArgs in kernels.h).
//
// A request's rows (its new tokens times the H / Hkv heads of a KV head) are
// columns of one 32-column MFMA block, so each key and value is read once per
// KV head and 32 rows; what bounds the kernel is that stream.  Lengths differ
// by orders of magnitude and only the device knows them, so the work is cut
// by key tiles, not by requests: all tiles of all (request, KV head, row block)
// items stand in one line, and worker w of W, a workgroup of one wave, takes
// the w-th of W equal runs of it.  A worker finds its run by summing the
// requests' tile counts (a wave, 64 requests a step), walks it with two LDS
// stages of its own, no barrier anywhere, and keeps 32 KiB of keys and values in
// flight (D = 128; two workers per CU).  An item that lies inside one run is
// written at once; of one that is cut, each run leaves its maximum, sum and
// unnormalised output (float32), at most two per worker, and a second launch
// joins them in order.  The partial results lie behind the output in its own
// block: two captured launches never share them.
#include <algorithm>

#include "attn_device.h"
#include "kernels.h"

namespace rew {

namespace pd {
constexpr int kRows = kDecodeRows;
constexpr int kLeast = 2;  // key tiles that are worth a worker
// workers: what the LDS of 256 CUs holds (4 tiles of 64 x D values each)
constexpr int workers(int D) { return 256 * (D == 128 ? 2 : D == 64 ? 4 : 8); }
// floats of a partial result: O [kRows][D], then (max, sum) per row
constexpr int part(int D) { return kRows * D + 2 * kRows; }
}  // namespace pd

size_t paged_ws_bytes(int D) { return (size_t)pd::workers(D) * 2 * pd::part(D) * 4; }

// A request's rows and keys, as the kernels of a step see them.
struct Request {
  int first, n, rows, len, cap;  // cap: keys that can have a page
  __device__ __forceinline__ int limit(const PackedArgs& a, int G, int row) const {
    const int t = min(row, rows - 1) / G;
    return min(max(a.causal ? len - n + t + 1 : len, 0), cap);
  }
};
// s: -1 .. n_seq (the rows of no request, as in SeqTile)
__device__ __forceinline__ Request request_at(const PackedArgs& a, int G, int s) {
  Request r;
  r.first = seq_bound(a.starts, a.n_seq, (int)a.T, s);
  r.n = s > a.n_seq ? 0 : max(seq_bound(a.starts, a.n_seq, (int)a.T, s + 1) - r.first, 0);
  r.rows = r.n * G;
  const bool real = s >= 0 && s < a.n_seq;
  r.len = real ? max(a.lens[s], 0) : 0;
  r.cap = real ? (int)min((int64_t)r.len, (int64_t)a.width << a.log_page) : 0;
  return r;
}

// The line of tiles: each item has at least one, so that rows without keys are
// written too.
struct TileLine {
  const PackedArgs& a;
  int G;
  bool all;  // requests of any size, or only those of one row block
  __device__ __forceinline__ int item_tiles(const Request& r, int qt) const {
    return max((r.limit(a, G, qt * pd::kRows + pd::kRows - 1) + pa::BK - 1) / pa::BK, 1);
  }
  // tiles of one KV head of a request
  __device__ __forceinline__ int head_tiles(const Request& r) const {
    if (!all && r.rows > pd::kRows) return 0;
    int t = 0;
    for (int qt = 0; qt * pd::kRows < r.rows; ++qt) t += item_tiles(r, qt);
    return t;
  }
  __device__ __forceinline__ int lane_tiles(int base) const {
    const int s = base + (int)(threadIdx.x & 63);
    return s > a.n_seq ? 0 : head_tiles(request_at(a, G, s)) * a.Hkv;
  }
};
// Where a tile of the line lies.
struct TilePlace {
  int s, hk, qt, kt;
  Request r;
  // (the line's total < 2^31 was checked on the host; x, sum: the first 64
  // requests' tiles and their running sum, which the total needed already)
  __device__ __forceinline__ void find(const TileLine& L, int t, int x, int sum) {
    int base = -1;
    for (;;) {
      const int total = __builtin_amdgcn_readlane(sum, 63);
      if (t < total || base + 64 > L.a.n_seq) break;
      t -= total;
      base += 64;
      x = L.lane_tiles(base);
      sum = wave_scan(x);
    }
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > t));
    t -= __builtin_amdgcn_readlane(sum - x, at);
    s = base + at;
    r = request_at(L.a, L.G, s);
    const int head = __builtin_amdgcn_readlane(x, at) / L.a.Hkv;
    hk = t / head;
    t -= hk * head;
    for (qt = 0;; ++qt) {
      const int k = L.item_tiles(r, qt);
      if (t < k) break;
      t -= k;
    }
    kt = t;
  }
  // the item after this one
  __device__ __forceinline__ void next(const TileLine& L) {
    kt = 0;
    if ((qt + 1) * pd::kRows < r.rows) {
      ++qt;
      return;
    }
    qt = 0;
    if (++hk < L.a.Hkv) return;
    hk = 0;
    do {
      ++s;
      r = request_at(L.a, L.G, s);
    } while (s <= L.a.n_seq && L.head_tiles(r) == 0);
  }
};
// The cut of the line into runs, as even as whole tiles allow; run w is
// [start(w), start(w + 1)).
struct Runs {
  int x, sum;  // of the first 64 requests, for TilePlace::find
  int total, count, each, more;
  __device__ __forceinline__ Runs(const TileLine& L, int most) {
    x = L.lane_tiles(-1);
    sum = wave_scan(x);
    total = __builtin_amdgcn_readlane(sum, 63);
    for (int base = 63; base <= L.a.n_seq; base += 64) total += wave_sum(L.lane_tiles(base));
    count = min(most, max((total + pd::kLeast - 1) / pd::kLeast, 1));
    each = total / count;
    more = total - each * count;
  }
  __device__ __forceinline__ int start(int w) const {
    return w >= count ? total : each * w + min(w, more);
  }
};

template <class M, int D>
__global__ void __launch_bounds__(64, D == 32 ? 2 : 1) decode_kernel(PackedArgs a, int all) {
  using namespace pa;
  typedef typename M::frag frag;
  constexpr int CPR = D / 8, NT = D / 16, DT = D / 32, TILE = BK * D;
  constexpr int RPD = 64 / CPR;     // key rows per DMA instruction
  constexpr int NDMA = TILE / 512;  // instructions per K (or V) tile
  __shared__ __attribute__((aligned(1024))) uint16_t S0[2 * TILE], S1[2 * TILE];
  typedef __attribute__((address_space(3))) uint16_t lds_u16;
  const int lane = threadIdx.x, c = lane & 31, g = lane >> 5;
  const int G = a.H / a.Hkv, w = blockIdx.x;
  const TileLine line{a, G, all != 0};
  const Runs runs(line, gridDim.x);
  const int from = runs.start(w), to = runs.start(w + 1);
  if (from >= to) return;
  TilePlace at;
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
  const float sl2 = a.scale * kLog2e;

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
    auto dma_tile = [&](lds_u16* st, int kt) __attribute__((always_inline)) {
      win.reach(kt * BK);
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
    // tile kt from stage st while the next one moves into the other, whose
    // reads are done
    auto step = [&](lds_u16* st, lds_u16* next, int kt) __attribute__((always_inline)) {
      const PageWindow here = win;
      const bool holes = here.any_missing(kt * BK, r.cap);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (kt + 1 < kt1) {
        dma_tile(next, kt + 1);
        if constexpr (NDMA == 16) asm volatile("s_waitcnt vmcnt(32)" ::: "memory");
        else if constexpr (NDMA == 8) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16_t s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s[0] = M::mma(*(__attribute__((address_space(3))) const frag*)(st + k_off[t]), qf[t], s[0]);
        s[1] = M::mma(*(__attribute__((address_space(3))) const frag*)(st + (k_off[t] + 32 * D)),
                      qf[t], s[1]);
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
                                    [&](int off) { return here.missing(k0 + off); });
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        union {
          uint32_t x[4];
          frag v;
        } pf;
#pragma unroll
        for (int i = 0; i < 4; ++i) pf.x[i] = pk[u >> 1][(u & 1) * 4 + i];
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
    dma_tile((lds_u16*)S0, kt0);
    int kt = kt0;
    for (; kt + 2 <= kt1; kt += 2) {
      step((lds_u16*)S0, (lds_u16*)S1, kt);
      step((lds_u16*)S1, (lds_u16*)S0, kt + 1);
    }
    if (kt < kt1) step((lds_u16*)S0, (lds_u16*)S1, kt);

    const float l = fa_sum_halves(l_run);
    if (kt0 == 0 && kt1 == tiles) {
      const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays NaN)
      if (row < r.rows) {
        uint16_t* O = (uint16_t*)a.out + ((int64_t)(r.first + tok) * a.H + at.hk * G + hg) * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(uint2*)(O + dt * 32 + i * 8 + g * 4) =
                make_uint2(M::pack(o[dt][i * 4] * inv, o[dt][i * 4 + 1] * inv),
                           M::pack(o[dt][i * 4 + 2] * inv, o[dt][i * 4 + 3] * inv));
      }
    } else if (row < r.rows) {  // slot 0: the item began in an earlier run; 1: it begins here
      float* p = a.work + ((int64_t)w * 2 + (kt0 == 0)) * pd::part(D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(float4*)(p + c * D + dt * 32 + i * 8 + g * 4) =
              make_float4(o[dt][i * 4], o[dt][i * 4 + 1], o[dt][i * 4 + 2], o[dt][i * 4 + 3]);
      if (g == 0) *(float2*)(p + pd::kRows * D + 2 * c) = make_float2(m_run, l);
    }
  }
}

// Workgroup w joins the item that run w is the first to continue, a wave per
// row in turn: the piece that run w - 1 left in slot 1, then those of runs w,
// w + 1, .. in slot 0.
template <class M, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(PackedArgs a, int all, int workers) {
  constexpr int L = D / 4;  // lanes of a row, four values each
  const int G = a.H / a.Hkv, w = blockIdx.x + 1;
  const TileLine line{a, G, all != 0};
  const Runs runs(line, workers);
  const int from = runs.start(w);
  if (from >= runs.total) return;
  TilePlace at;
  at.find(line, from, runs.x, runs.sum);
  const int first = from - at.kt;  // the item's first tile
  if (at.kt == 0 || first < runs.start(w - 1)) return;
  const int end = first + line.item_tiles(at.r, at.qt);
  int n = 1;  // pieces after the first
  while (runs.start(w + n) < end) ++n;
  const int rows = min(at.r.rows - at.qt * pd::kRows, pd::kRows);
  const int d = (threadIdx.x % L) * 4;
  for (int i = threadIdx.x / L; i < rows; i += 256 / L) {
    auto piece = [&](int k) {  // k = 0: slot 1 of run w - 1, then slot 0
      return a.work + ((int64_t)(w - 1 + k) * 2 + (k == 0)) * pd::part(D);
    };
    float m = -INFINITY;
#pragma unroll 8
    for (int k = 0; k <= n; ++k) m = fmaxf(m, piece(k)[pd::kRows * D + 2 * i]);
    const float mu = m == -INFINITY ? 0.0f : m;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
#pragma unroll 8
    for (int k = 0; k <= n; ++k) {
      const float* p = piece(k);
      const float2 ml = *(const float2*)(p + pd::kRows * D + 2 * i);
      const float4 o = *(const float4*)(p + i * D + d);
      const float s = fa_exp2(ml.x - mu);
      l = fmaf(ml.y, s, l);
      x[0] = fmaf(o.x, s, x[0]);
      x[1] = fmaf(o.y, s, x[1]);
      x[2] = fmaf(o.z, s, x[2]);
      x[3] = fmaf(o.w, s, x[3]);
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    const int row = at.qt * pd::kRows + i, tok = row / G, hg = row - tok * G;
    uint16_t* O = (uint16_t*)a.out + ((int64_t)(at.r.first + tok) * a.H + at.hk * G + hg) * D + d;
    *(uint2*)O = make_uint2(M::pack(x[0] * inv, x[1] * inv), M::pack(x[2] * inv, x[3] * inv));
  }
}

template <class M, int D>
static void launch_decode(const PackedArgs& a, int all, hipStream_t stream) {
  constexpr int W = pd::workers(D);
  hipLaunchKernelGGL((decode_kernel<M, D>), dim3(W), dim3(64), 0, stream, a, all);
  hipLaunchKernelGGL((decode_join_kernel<M, D>), dim3(W - 1), dim3(256), 0, stream, a, all, W);
}
template <class M>
static void launch_decode_t(const PackedArgs& a, int all, hipStream_t stream) {
  if (a.D == 32) launch_decode<M, 32>(a, all, stream);
  else if (a.D == 64) launch_decode<M, 64>(a, all, stream);
  else launch_decode<M, 128>(a, all, stream);
}

void launch_paged_decode(const PackedArgs& a, bool all, hipStream_t stream) {
  const int64_t keys = std::max<int64_t>(((int64_t)a.width << a.log_page) / pa::BK + 1, 1);
  if ((max_seq_tiles(a.T, a.n_seq, a.H / a.Hkv, pd::kRows) * keys) >= (1ll << 31) / a.Hkv)
    fail(REW_MI355X_ERR_UNSUPPORTED, "paged attention: 2^31 key tiles or more");
  if (a.f16) launch_decode_t<MmaF16>(a, all, stream);
  else launch_decode_t<MmaBf16>(a, all, stream);
}

}  // namespace rew
