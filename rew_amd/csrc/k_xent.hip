// Softmax cross entropy of a linear head and its gradients (XentArgs and
// XentGradArgs in kernels.h), without keeping the logits.
//
// Forward: a workgroup holds 256 tokens and walks a run of 256-column tiles of
// the vocabulary.  The logits of a tile are formed in the accumulators and
// reduced there: each lane keeps the running maximum m and the sum s of
// exp(z - m) of its columns per row, so only two floats per row and run of
// tiles reach memory.  A second launch joins the runs.
//
// Gradients: a piece of the vocabulary at a time, the logits are formed again,
// their gradient dz goes to working memory in 16 bits, and two products read
// it: dw's columns of the piece, x^T dz, are finished there; dx = dz w^T is
// added up over the pieces in float32.
//
// Bound: the matrix cores.  8192 x 4096 x 128256 bfloat16: the logits in 6.23 ms
// (1.37 PFLOP/s, as a large library product), matrix cores busy 78 % of the cycles
// at 1.66 GHz; per piece of 16384 words dz 0.86 ms, dw 0.81, dx 0.87 (1.28, 1.36 and
// 1.26 PFLOP/s; 67-75 %: dz's 270 MB of stores, dx's read and written sums).
// 4000 x 2048 x 32003 float16: 1.03 to 1.23 PFLOP/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_device.h"
#include "kernels.h"

namespace rew {

namespace {

constexpr int BM = 256, BN = 256, BK = 64;  // output tile, k-step
// eight waves, two per SIMD, of 128 x 64 outputs each: 128 accumulators a lane
// leave room for the fragments and an epilogue's own values (four waves of 128 x
// 128 spilled around theirs)
constexpr int kThreads = 512, NI = 4, NJ = 2;
constexpr int kBlocks = 4;  // 1 KiB blocks of an operand's k-step per wave
constexpr int kHalf = BM * BK * 2;          // bytes of an operand's k-step: 32 KiB
constexpr int SM = 64, kSmallHalf = SM * BK * 2;  // the small form's tile
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
// 1 / (kLog2e as it is rounded) less kLn2 as it is rounded.
constexpr float kLn2Rest = (float)(1.0 / (double)kLog2e - (double)kLn2);
constexpr float kMost = 3.402823466e38f;
// dz is stored as 2^14 g / max|g| (p - 1): below 2^14, so float16 keeps eleven
// bits of probabilities down to 2^-28 and the float32 sums have room.  (Its rounding makes
// the gradients' error 0.0022 for the 0.0017 of their own in bfloat16, 0.00028 for 0.00021
// in float16, relative to their norm; keeping the remainders of every token would double
// the k-steps of two of the three products.)
constexpr float kDzScale = 16384.0f;
// The gradients of few tokens are sums of few terms that matter, which do not average
// dz's rounding (2 tokens, 64 x 2 bfloat16: dx 0.0036 off relative to its norm, of which
// its own rounding is 0.0017).  Up to 32 tokens fill half of the products' least tile
// and k-step, and the other half carries what dz's rounding left.  Forward and
// gradients as called, without / with: 1 x 64 x 1000 35 / 38 us (the join of dx), 30 x
// 1000 x 20000 79 / 86, 32 x 4096 x 128256 915 / 929; 2 x 64 x 2 is off by its own
// rounding alone.
constexpr int64_t kRestRows = 32;
// Columns of the vocabulary at a time, at least (8192 x 4096 x 128256, all kernels: 26.7
// ms; 8192 columns 26.9; 32768 columns 26.5, with twice the working memory).
constexpr int64_t kPiece = 16384;

// An operand of a product: element (r, k) at p[r ld + k] (KC) or p[k ld + r].
// k counts up to `k`, a multiple of 8; `len` elements may be read from p.
struct Opnd {
  const uint16_t* p;
  int64_t ld, len, k;
};

struct Product {
  Opnd a, b;
  int64_t M, N, K;      // rows, columns; K: a multiple of BK, 0 past an operand's k
  int n0, V;            // first column in the vocabulary, its size
  int per;              // kStats: column tiles of a run; kSum: k-steps of a split
  int tiles_m, tiles_n, splits;
  int slot0;            // kStats: first of this launch's partial results
  int add;              // kSum: onto what is there
  const int32_t* target;  // kOut: null, or rows without a target are zeros
  const float *lse, *grad, *scale;  // scale: {max |grad|}
  float2* part;         // kStats: {m, s} of a run of tiles, [slot][M]
  float* zt;            // kStats: the target's logit
  void* out;            // kDz, kOut: row pitch ldo; kSum: float32 [split][M][N]
  int64_t ldo, rows_out;
  int64_t rest;         // kDz, kDzRest: rows from dz to its remainders, 0: none
};

// What becomes of the products: running softmax statistics; dz; a result in 16 bits;
// a float32 share of one.  kDzRest: dz and its remainders, by 256 x 256 tiles.
enum { kStats, kDz, kOut, kSum, kDzRest };
constexpr bool is_dz(int mode) { return mode == kDz || mode == kDzRest; }

// Workgroups whose indices agree mod 8 share an XCD and its L2: each XCD gets a
// contiguous range, walked in groups of 4 row tiles.
__device__ __forceinline__ void tile_at(uint32_t bid, uint32_t tiles_m, uint32_t tiles_n, int* tm,
                                        int* tn) {
  const uint32_t total = tiles_m * tiles_n, q = total / 8, r = total % 8, x = bid % 8;
  const uint32_t t = x * q + min(x, r) + bid / 8;
  const uint32_t group = 4 * tiles_n, g = t / group, i = t - g * group;
  const uint32_t size = min(4u, tiles_m - 4 * g);
  *tn = (int)(i / size);
  *tm = (int)(4 * g + i % size);
}

// One k-step (64) of an operand's R rows into LDS, Q 1 KiB blocks by each wave.
// KC: rows of 128 bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7).  Else rows
// of one k and R r's, for the transposing fragment reads: chunk c of row k at
// c ^ (4 (k & 3)) (R = 256) or c ^ (2 ((k >> 1) & 3)) (R = 64), so that the four
// rows that a read touches lie in different banks.  Past `len`, and past k in a KC
// row, zeros arrive.
template <bool KC, int R, int Q>
struct Fetch {
  static constexpr int kRowChunks = KC ? BK / 8 : R / 8;
  static constexpr int kBlockRows = 64 / kRowChunks;
  static constexpr uint32_t kPast = 0x80000000u;  // (behind any descriptor's end)
  const uint16_t* base;
  int64_t left;  // elements from base that may be read
  int64_t step;  // elements per k-step
  int64_t left_k;
  uint32_t off[Q], cols[KC ? Q : 1];  // KC: byte of the lane's chunk within its row

  __device__ __forceinline__ void start(const Opnd& o, int64_t r0, int64_t k0) {
    const int64_t at = KC ? r0 * o.ld + k0 : k0 * o.ld + r0;
    base = o.p + at;
    left = o.len - at;
    left_k = o.k - k0;
  }
  __device__ __forceinline__ void init(const Opnd& o, int first_block, int lane) {
    step = KC ? BK : BK * o.ld;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int r = (first_block + q) * kBlockRows + lane / kRowChunks;  // row, or k
      const int c = lane % kRowChunks;
      const int x = KC ? (r >> 1) & 7 : R == 256 ? 4 * (r & 3) : 2 * ((r >> 1) & 3);
      off[q] = (uint32_t)r * (uint32_t)(o.ld * 2);
      if constexpr (KC) cols[q] = (uint32_t)((c ^ x) * 16);
      else off[q] += (uint32_t)((c ^ x) * 16);
    }
  }
  // (`live` false: zeros, without a read)
  __device__ __forceinline__ void issue(uint8_t* lds, bool live) {
    const int64_t bytes = live && left > 0 ? min(left * 2, (int64_t)0x7fffffff) : 0;
    const __amdgpu_buffer_rsrc_t r = fa_rsrc(base, (uint32_t)bytes);
    const uint32_t lim = (uint32_t)(min(left_k, (int64_t)BK) * 2 - 16);
#pragma unroll
    for (int q = 0; q < Q; ++q)
      dma16_lds(r, !KC ? off[q] : cols[KC ? q : 0] <= lim ? off[q] + cols[KC ? q : 0] : kPast, 0,
                (lds_void*)(lds + q * 1024));
  }
  __device__ __forceinline__ void next(int n = 1) {
    base += n * step;
    left -= n * step;
    left_k -= n * BK;
  }
};

// Fragment i (32 rows from r0 + 32 i) of substep s (16 k): lane l gets row l % 32,
// k = 8 (l / 32) .. + 7.
template <bool KC, int R, int F>
struct Frags {
  int off[KC ? 4 : F];
  __device__ __forceinline__ void init(int r0, int lane) {
    if constexpr (KC) {
      const int r = r0 + (lane & 31);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        off[s] = r * 128 + (((2 * s + (lane >> 5)) ^ ((r >> 1) & 7)) * 16);
    } else {
      const int g = lane >> 4, s16 = lane & 15, k = 8 * (g >> 1) + (s16 >> 2);
      const int x = R == 256 ? 4 * (k & 3) : 2 * ((k >> 1) & 3);
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int c = r0 + i * 32 + 16 * (g & 1) + 4 * (s16 & 3);
        off[i] = k * (R * 2) + (((c >> 3) ^ x) * 16) + (c & 7) * 2;
      }
    }
  }
  template <class Frag>
  __device__ __forceinline__ void read(const uint8_t* lds, int s, Frag (&f)[F]) const {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if constexpr (KC) {
        f[i] = *(const Frag*)(lds + off[s] + i * 32 * 128);
      } else {
        // (k + 4 has k's swizzle in tiles of 256; in tiles of 64 the other half of it)
        const int at = off[i] + s * 16 * (R * 2);
        const uint8_t* hi_at = lds + (R == 256 ? at + 4 * (R * 2) : (at ^ 64) + 4 * (R * 2));
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds + at));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)hi_at);
        v4s both[2] = {lo, hi};
        __builtin_memcpy(&f[i], both, 16);
      }
    }
  }
};

__device__ __forceinline__ void wg_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes at any address (rows of an odd number of values).
struct __attribute__((packed, aligned(2))) Loose16 {
  uint32_t v[4];
};

// The first n of eight 16-bit values.
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v, int64_t n) {
  if (n >= 8) {
    *(Loose16*)p = {{v.x, v.y, v.z, v.w}};
  } else {
    const uint16_t* h = (const uint16_t*)&v;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = h[e];
  }
}

// The running maximum (of z log2 e, so that its rounding cancels) and sum of
// exponentials of one row's logits.  The maximum stays finite: an infinite logit
// gives an infinite exponential and no NaN.
__device__ __forceinline__ float stat_max(float z) {
  return fminf(fmaxf(z * kLog2e, -kMost), kMost);
}
__device__ __forceinline__ float stat_exp(float z, float m) {
  return fa_exp2(__builtin_fmaf(z, kLog2e, -m));
}

// What rounding two values to 16 bits leaves of them; none of an infinity.
template <class Ty>
__device__ __forceinline__ void rest_of(float& a, float& b) {
  const uint32_t h = Ty::pack(a, b);
  const float lo = Ty::lo(h), hi = Ty::hi(h);
  a = fabsf(lo) <= kMost ? a - lo : 0.0f;
  b = fabsf(hi) <= kMost ? b - hi : 0.0f;
}

// What a row's dz needs, loaded early; dz of a row without a target is zero.
struct DzRow {
  int32_t target;
  float grad, lse;
  __device__ __forceinline__ void load(const Product& g, int64_t row) {
    const bool in = row < g.M;
    const int64_t r = in ? row : g.M - 1;
    target = in ? g.target[r] : -1;
    grad = g.grad[r];
    lse = g.lse[r];
  }
  __device__ __forceinline__ bool live(const Product& g) const {
    return target >= 0 && target < g.V;
  }
  __device__ __forceinline__ float factor(float scale) const { return grad / scale * kDzScale; }
  __device__ __forceinline__ float lse2() const { return lse * kLog2e; }
  // .. of probabilities 2^(z log2 e - lse2): with what lse2's rounding took.
  __device__ __forceinline__ float factor_p(float f) const {
    const float d = __builtin_fmaf(lse, kLog2e, -lse2());
    return fabsf(d) < 1.0f ? __builtin_fmaf(-d * kLn2, f, f) : f;  // (not of an infinite lse)
  }
};

// 256 x 256 outputs at a time, from two stages of a k-step each.  Workgroups walk
// over tiles (kStats: a run of column tiles, else every gridDim.x-th), and the last
// k-steps of a tile already fetch the next one's first.
template <class Ty, bool AKC, bool BKC, int MODE>
__global__ void __launch_bounds__(kThreads, 1) xent_product_kernel(Product g) {
  // one array per stage and operand, so that the compiler sees that a DMA into one
  // does not meet fragment reads of another
  __shared__ __attribute__((aligned(1024))) uint8_t A0[kHalf], B0[kHalf], A1[kHalf], B1[kHalf];
  __shared__ __attribute__((aligned(1024))) uint8_t Turn[MODE == kStats ? 4 * BM * 8 : 8 * 4096];
  typedef typename Ty::frag frag;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  struct Tile {
    int tm, tn, split, k0, nk;
  };
  const uint32_t per_split = (uint32_t)g.tiles_m * g.tiles_n;
  const uint32_t total = MODE == kSum ? per_split * g.splits : per_split;
  const int nk_all = (int)(g.K / BK);
  auto tile_of = [&](uint32_t t) {
    Tile x;
    x.split = MODE == kSum ? t / per_split : 0;
    tile_at(t - x.split * per_split, g.tiles_m, g.tiles_n, &x.tm, &x.tn);
    x.k0 = MODE == kSum ? x.split * g.per : 0;
    x.nk = MODE == kSum ? min(g.per, nk_all - x.k0) : nk_all;
    return x;
  };
  Tile cur;
  uint32_t t = blockIdx.x;
  int tn_end = 0;
  if constexpr (MODE == kStats) {
    tile_at(blockIdx.x, g.tiles_m, g.splits, &cur.tm, &cur.split);
    cur.tn = cur.split * g.per;
    cur.k0 = 0;
    cur.nk = nk_all;
    tn_end = min(cur.tn + g.per, g.tiles_n);
  } else {
    cur = tile_of(t);
  }

  Frags<AKC, BM, NI> ra;
  Frags<BKC, BN, NJ> rb;
  ra.init(wm * 128, lane);
  rb.init(wn * 64, lane);
  Fetch<AKC, BM, kBlocks> fa;
  Fetch<BKC, BN, kBlocks> fb;
  fa.init(g.a, wave * kBlocks, lane);
  fb.init(g.b, wave * kBlocks, lane);
  const int at = wave * kBlocks * 1024;

  // rows of this lane: 256 tm + 128 wm + 32 i + lane % 32
  int tgt[NI];
  float run_m[NI], run_s[NI];
  if constexpr (MODE == kStats) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t row = (int64_t)cur.tm * BM + wm * 128 + i * 32 + (lane & 31);
      const int32_t v = row < g.M ? g.target[row] : -1;
      tgt[i] = v >= 0 && v < g.V ? v - g.n0 : -1;
      run_m[i] = -kMost;
      run_s[i] = 0.0f;
    }
  }
  float scale = 1.0f;
  if constexpr (is_dz(MODE) || MODE == kOut) scale = g.scale[0];

  fa.start(g.a, (int64_t)cur.tm * BM, (int64_t)cur.k0 * BK);
  fb.start(g.b, (int64_t)cur.tn * BN, (int64_t)cur.k0 * BK);
  fa.issue(A0 + at, cur.nk > 0);
  fb.issue(B0 + at, cur.nk > 0);
  fa.next();
  fb.next();
  fa.issue(A1 + at, cur.nk > 1);
  fa.next();
  __builtin_amdgcn_s_waitcnt(0x0f70 | kBlocks);  // (the second step's may be under way)
  wg_barrier();

  for (;;) {
    Tile nxt = cur;
    bool more;
    if constexpr (MODE == kStats) {
      nxt.tn = cur.tn + 1;
      more = nxt.tn < tn_end;
    } else {
      t += gridDim.x;
      more = t < total;
      if (more) nxt = tile_of(t);
    }
    const int64_t m0 = (int64_t)cur.tm * BM;
    DzRow dz[is_dz(MODE) ? NI : 1];
    if constexpr (is_dz(MODE))
#pragma unroll
      for (int i = 0; i < NI; ++i) dz[i].load(g, m0 + wm * 128 + i * 32 + (lane & 31));

    f32x16_t acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    frag x[2][NI], y[2][NJ];
    auto read = [&](const uint8_t* sa, const uint8_t* sb, int s) {
      ra.read(sa, s, x[s & 1]);
      rb.read(sb, s, y[s & 1]);
    };
    // (b first: lane l then holds row l % 32 of each 32 x 32 block and the columns
    // 8 (e / 4) + 4 (l / 32) + e % 4)
    auto products = [&](int s) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = Ty::mma(y[s & 1][j], x[s & 1][i], acc[i][j]);
    };
    // One substep's order: its products one by one, the fragment reads of the next and
    // four DMA instructions between them (left to itself the compiler reads right
    // before the use and issues all DMA together).
    auto pin = [&](bool dma, bool reads) {
      constexpr int kM = NI * NJ, kR = (AKC ? NI : 2 * NI) + (BKC ? NJ : 2 * NJ);
      constexpr int kEach = (kR + 5) / 6;  // (the last ones early enough to be there)
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (reads && r < kEach && m * kEach + r < kR)
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // DS read
        if (dma && m % (kM / 4) == 0) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // VMEM
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // A step with its first fragments already read: three substeps read the next one's
    // beside their products; then all waves have the last fragments of this stage and
    // their part of the next one's data has arrived, and beside the last substep's
    // products the next stage's first fragments are read (not at a tile's end: the
    // registers are the epilogue's).  A stage is filled with the step after the next:
    // a's half beside the last substep, b's beside the next step's first.
    auto step = [&](uint8_t* sa, uint8_t* sb, uint8_t* na, uint8_t* nb, bool live_b, bool live_a,
                    bool end) {
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        read(sa, sb, s + 1);
        if (s == 0) {
          fb.issue(nb + at, live_b);
          fb.next();
        }
        products(s);
        pin(s == 0, true);
      }
      __builtin_amdgcn_s_waitcnt(0x0070);  // (vmcnt 0, lgkmcnt 0)
      wg_barrier();
      if (!end) read(na, nb, 0);
      fa.issue(sa + at, live_a);
      fa.next();
      products(3);
      pin(true, !end);
    };
    read(A0, B0, 0);
    const int nk = cur.nk, even = max(2, (nk + 1) & ~1);  // (a last odd step: zeros)
    for (int kt = 0; kt + 2 < even; kt += 2) {
      step(A0, B0, A1, B1, true, true, false);
      step(A1, B1, A0, B0, true, kt + 3 < nk, false);
    }
    const bool last_b = even - 1 < nk, next0 = more && nxt.nk > 0, next1 = more && nxt.nk > 1;
    fa.start(g.a, (int64_t)nxt.tm * BM, (int64_t)nxt.k0 * BK);
    step(A0, B0, A1, B1, last_b, next0, false);
    fb.start(g.b, (int64_t)nxt.tn * BN, (int64_t)nxt.k0 * BK);
    step(A1, B1, A0, B0, next0, next1, true);

    const int n_base = cur.tn * BN + wn * 64;  // of this wave's columns
    const int n_lane = n_base + (lane >> 5) * 4;
    auto col_of = [&](int j, int e) { return n_lane + j * 32 + (e >> 2) * 8 + (e & 3); };

    if constexpr (MODE == kStats) {
      const bool edge = (cur.tn + 1) * BN > g.N;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (edge)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (col_of(j, e) >= g.N) acc[i][j][e] = -INFINITY;
        // the target's logit, where it lies in these 64 columns
        const int d = tgt[i] - n_base;
        if (__any(tgt[i] >= 0 && d >= 0 && d < 64 && tgt[i] < g.N)) {
          const int64_t row = m0 + wm * 128 + i * 32 + (lane & 31);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (tgt[i] == col_of(j, e) && tgt[i] < g.N) g.zt[row] = acc[i][j][e];
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
        const float m = fmaxf(run_m[i], stat_max(top));
        float s0 = run_s[i] * fa_exp2(run_m[i] - m), s1 = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            s0 += stat_exp(acc[i][j][e], m);
            s1 += stat_exp(acc[i][j][e + 1], m);
          }
        run_m[i] = m;
        run_s[i] = s0 + s1;
      }
    } else {
      // 32 rows at a time through 4 KiB of LDS of the wave's own, so that whole lines
      // of 128 bytes are stored: 16-byte chunk c of row r at c ^ (r & 7).  In passes of
      // 8 rows, lane l then has chunk l % 8 of row l / 8.
      uint8_t* turn = Turn + wave * 4096;
      const int r32 = lane & 31, r8 = lane >> 3, ch = lane & 7;
      auto put_at = [&](int c) { return turn + r32 * 128 + ((c ^ (r32 & 7)) * 16); };
      auto get_at = [&](int p) { return turn + (p * 8 + r8) * 128 + ((ch ^ r8) * 16); };
      const float gain = scale / kDzScale;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int64_t row0 = m0 + wm * 128 + i * 32;
        if constexpr (is_dz(MODE) || MODE == kOut) {
          uint64_t alive = ~0ull;
          if constexpr (is_dz(MODE)) {
            alive = __ballot(dz[i].live(g));
            const float f = dz[i].factor(scale), lse2 = dz[i].lse2(), fp = dz[i].factor_p(f);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                acc[i][j][e] = fp * fa_exp2(__builtin_fmaf(acc[i][j][e], kLog2e, -lse2));
            const int c = dz[i].target - g.n0;
            if (__any(dz[i].target >= g.n0 && c >= n_base && c < n_base + 64))
#pragma unroll
              for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  if (c == col_of(j, e)) acc[i][j][e] -= f;
          } else if (g.target) {
            const int64_t row = row0 + r32;
            const int32_t v = g.target[row < g.M ? row : g.M - 1];
            alive = __ballot(v >= 0 && v < g.V);
          }
          auto emit = [&](auto part) {
            constexpr bool rest = decltype(part)::value;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  v[e] = MODE == kOut ? acc[i][j][q * 4 + e] * gain : acc[i][j][q * 4 + e];
                if constexpr (rest) {
#pragma unroll
                  for (int e = 0; e < 4; e += 2) rest_of<Ty>(v[e], v[e + 1]);
                }
                *(uint2*)(put_at(j * 4 + q) + (lane >> 5) * 8) =
                    make_uint2(Ty::pack(v[0], v[1]), Ty::pack(v[2], v[3]));
              }
            const int64_t cols = g.N - (n_base + ch * 8);  // (dz: zeros behind)
            uint16_t* out =
                (uint16_t*)g.out + (row0 + r8 + (rest ? g.rest : 0)) * g.ldo + n_base + ch * 8;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              uint4 v = *(const uint4*)get_at(p);
              if (!(alive >> (p * 8 + r8) & 1)) v = make_uint4(0, 0, 0, 0);
              if (row0 + p * 8 + r8 >= g.rows_out) continue;
              if constexpr (is_dz(MODE)) {
                if (cols < 8) {
                  uint16_t* h = (uint16_t*)&v;
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    if (e >= cols) h[e] = 0;
                }
                *(uint4*)(out + p * 8 * g.ldo) = v;
              } else {
                store8(out + p * 8 * g.ldo, v, cols);
              }
            }
          };
          emit(std::false_type());
          if constexpr (MODE == kDzRest) emit(std::true_type());
        } else {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *(float4*)put_at(q * 2 + (lane >> 5)) =
                  make_float4(acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2],
                              acc[i][j][q * 4 + 3]);
            const int n = n_base + j * 32 + ch * 4;
            const int64_t cols = g.N - n;
            float* out = (float*)g.out + ((int64_t)cur.split * g.M + row0 + r8) * g.N + n;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              float4 v = *(const float4*)get_at(p);
              float* o = out + p * 8 * g.N;
              if (row0 + p * 8 + r8 >= g.M || cols <= 0) continue;
              if (g.N % 4 == 0) {
                if (g.add) {
                  const float4 w = *(const float4*)o;
                  v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                }
                *(float4*)o = v;
              } else {
                const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (e < cols) o[e] = g.add ? o[e] + f[e] : f[e];
              }
            }
          }
        }
      }
    }
    if (!more) break;
    cur = nxt;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // (the last fetches' zeros still land in the stages)

  if constexpr (MODE == kStats) {
    // both lanes of a row, then the four waves of its columns
    float2* tmp = (float2*)Turn;  // [4][BM]
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float om = __shfl_xor(run_m[i], 32), os = __shfl_xor(run_s[i], 32);
      const float m = fmaxf(run_m[i], om);
      const float s = run_s[i] * fa_exp2(run_m[i] - m) + os * fa_exp2(om - m);
      if (lane < 32) tmp[wn * BM + wm * 128 + i * 32 + lane] = make_float2(m, s);
    }
    __syncthreads();
    const int64_t row = (int64_t)cur.tm * BM + tid;
    if (tid < BM && row < g.M) {
      float m = tmp[tid].x, s = 0.0f;
#pragma unroll
      for (int w = 1; w < 4; ++w) m = fmaxf(m, tmp[w * BM + tid].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) s += tmp[w * BM + tid].y * fa_exp2(tmp[w * BM + tid].x - m);
      g.part[(int64_t)(g.slot0 + cur.split) * g.M + row] = make_float2(m, s);
    }
  }
}

// 64 x 64 outputs per workgroup, every eighth k-step to each wave, which fills and
// reads LDS of its own; the waves' sums are joined in LDS.  For products of few
// 256 x 256 tiles, whose k-steps would follow one another on a few CUs.
template <class Ty, bool AKC, bool BKC, int MODE>
__device__ __forceinline__ void small_product(const Product& g, uint32_t bid, float scale,
                                              uint8_t (*L)[2 * kSmallHalf]) {
  typedef typename Ty::frag frag;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t *sa = L[wave], *sb = L[wave] + kSmallHalf;

  int tm, tn, split = 0, nk = (int)(g.K / BK), k_first = 0;
  if constexpr (MODE == kStats) {
    tile_at(bid, g.tiles_m, g.splits, &tm, &split);
    tn = split * g.per;
  } else if constexpr (MODE == kSum) {
    const uint32_t tiles = g.tiles_m * g.tiles_n;
    split = bid / tiles;
    tile_at(bid - split * tiles, g.tiles_m, g.tiles_n, &tm, &tn);
    k_first = split * g.per;
    nk = min(g.per, nk - k_first);
  } else {
    tile_at(bid, g.tiles_m, g.tiles_n, &tm, &tn);
  }
  const int64_t m0 = (int64_t)tm * SM;
  const int tn_end = MODE == kStats ? min(tn + g.per, g.tiles_n) : tn + 1;
  Frags<AKC, SM, 2> ra;
  Frags<BKC, SM, 2> rb;
  ra.init(0, lane);
  rb.init(0, lane);
  // after the join: row tid / 8, columns 8 (tid % 8) ..
  const int jr = tid >> 3, jc = (tid & 7) * 8;
  const int64_t row = m0 + jr;
  float run_m = -kMost, run_s = 0.0f, gain = 0.0f;
  int tgt = -1;
  DzRow d;
  float f = 0.0f, fp = 0.0f;
  if constexpr (MODE == kStats) {
    const int32_t t = row < g.M ? g.target[row] : -1;
    if (t >= 0 && t < g.V) tgt = t - g.n0;
  }
  if constexpr (is_dz(MODE)) {
    d.load(g, row);
    f = d.factor(scale);
    fp = d.factor_p(f);
  }
  bool alive = true;
  if constexpr (MODE == kOut) {
    gain = scale / kDzScale;
    if (g.target) alive = row < g.M && g.target[row] >= 0 && g.target[row] < g.V;
  }

  for (; tn < tn_end; ++tn) {
    f32x16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    Fetch<AKC, SM, 8> fa;
    Fetch<BKC, SM, 8> fb;
    fa.init(g.a, 0, lane);
    fb.init(g.b, 0, lane);
    fa.start(g.a, m0, (int64_t)(k_first + wave) * BK);
    fb.start(g.b, (int64_t)tn * SM, (int64_t)(k_first + wave) * BK);
    for (int kt = wave; kt < nk; kt += 8) {
      fa.issue(sa, true);
      fb.issue(sb, true);
      fa.next(8);
      fb.next(8);
      __builtin_amdgcn_s_waitcnt(0x0f70);
      asm volatile("" ::: "memory");
      frag x[4][2], y[4][2];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        ra.read(sa, s, x[s]);
        rb.read(sb, s, y[s]);
      }
      // (in the registers before the next step's data takes their place)
      __builtin_amdgcn_s_waitcnt(0xc07f);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = Ty::mma(y[s][j], x[s][i], acc[i][j]);
    }
    // this wave's 64 x 64 sums: 256-byte rows, 16-byte chunk c of row r at c ^ (r & 15)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 32 + (lane & 31);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = (j * 32 + q * 8 + (lane >> 5) * 4) >> 2;
          *(float4*)(L[wave] + r * 256 + ((c ^ (r & 15)) * 16)) =
              make_float4(acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2],
                          acc[i][j][q * 4 + 3]);
        }
    }
    __syncthreads();
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const int live = min(8, nk);  // (waves with a k-step)
    for (int w = 0; w < live; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = (jc >> 2) + h;
        const float4 f = *(const float4*)(L[w] + jr * 256 + ((c ^ (jr & 15)) * 16));
        v[h * 4] += f.x, v[h * 4 + 1] += f.y, v[h * 4 + 2] += f.z, v[h * 4 + 3] += f.w;
      }
    __syncthreads();
    const int n = tn * SM + jc, cols = (int)min((int64_t)8, g.N - n);
    if constexpr (MODE == kStats) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e >= cols) v[e] = -INFINITY;
        else if (n + e == tgt) g.zt[row] = v[e];
        top = fmaxf(top, v[e]);
      }
      const float m = fmaxf(run_m, stat_max(top));
      run_s *= fa_exp2(run_m - m);
#pragma unroll
      for (int e = 0; e < 8; ++e) run_s += stat_exp(v[e], m);
      run_m = m;
    } else if constexpr (is_dz(MODE) || MODE == kOut) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (is_dz(MODE)) {
          v[e] = fp * fa_exp2(__builtin_fmaf(v[e], kLog2e, -d.lse2()));
          if (n + e == d.target - g.n0) v[e] -= f;
          if (e >= cols || !d.live(g)) v[e] = 0.0f;
        } else {
          v[e] = alive ? v[e] * gain : 0.0f;
        }
      }
      const uint4 h = make_uint4(Ty::pack(v[0], v[1]), Ty::pack(v[2], v[3]),
                                 Ty::pack(v[4], v[5]), Ty::pack(v[6], v[7]));
      if (row < g.rows_out) {
        uint16_t* out = (uint16_t*)g.out + row * g.ldo + n;
        if constexpr (is_dz(MODE)) {
          *(uint4*)out = h;
          if (g.rest) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) rest_of<Ty>(v[e], v[e + 1]);
            *(uint4*)(out + g.rest * g.ldo) =
                make_uint4(Ty::pack(v[0], v[1]), Ty::pack(v[2], v[3]), Ty::pack(v[4], v[5]),
                           Ty::pack(v[6], v[7]));
          }
        } else {
          store8(out, h, cols);
        }
      }
    } else if (row < g.M) {
      float* o = (float*)g.out + ((int64_t)split * g.M + row) * g.N + n;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < cols) o[e] = g.add ? o[e] + v[e] : v[e];
    }
  }
  if constexpr (MODE == kStats) {
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) {
      const float om = __shfl_xor(run_m, x), os = __shfl_xor(run_s, x);
      const float m = fmaxf(run_m, om);
      run_s = run_s * fa_exp2(run_m - m) + os * fa_exp2(om - m);
      run_m = m;
    }
    if (jc == 0 && row < g.M)
      g.part[(int64_t)(g.slot0 + split) * g.M + row] = make_float2(run_m, run_s);
  }
}

// The largest finite |grad| of a token with a target, 1 if none is above 0; in every
// thread.
template <int Threads>
__device__ __forceinline__ float largest_grad(const int32_t* target, const float* grad, int64_t T,
                                              int64_t V, float* tmp) {
  float m = 0.0f;
  for (int64_t t = threadIdx.x; t < T; t += Threads) {
    const float f = fabsf(grad[t]);
    if (target[t] >= 0 && target[t] < V && f < INFINITY) m = fmaxf(m, f);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Threads / 64; ++i) m = fmaxf(m, tmp[i]);
  __syncthreads();
  return m > 0.0f ? m : 1.0f;
}

// x with zeros in rows without a target (`all`: every row as it is), in rows behind T
// and columns behind H: 16 bytes from every `step`-th thread.  twice (the rows that dz's
// remainders multiply): row r once more in row r + kRestRows.
struct Copy {
  const uint16_t* x;
  const int32_t* target;
  uint16_t* out;
  int64_t T, H, V, Tp, Hp, ld;
  int all, twice;
};
__device__ __forceinline__ void copy_x(const Copy& c, int64_t first, int64_t step) {
  const int64_t per = c.Hp / 8, total = c.Tp * per;
  for (int64_t i = first; i < total; i += step) {
    const int64_t to = total >> 32 ? i / per : (int64_t)((uint32_t)i / (uint32_t)per);
    const int64_t k = (i - to * per) * 8;
    const int64_t r = c.twice && to >= kRestRows ? to - kRestRows : to;
    const bool live = r < c.T && (c.all || (c.target[r] >= 0 && c.target[r] < c.V));
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live) {
      const uint16_t* p = c.x + r * c.H + k;
      if (k + 8 <= c.H) {
        const Loose16 h = *(const Loose16*)p;
        v = make_uint4(h.v[0], h.v[1], h.v[2], h.v[3]);
      } else {
        uint16_t* h = (uint16_t*)&v;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < c.H) h[e] = p[e];
      }
    }
    *(uint4*)(c.out + to * c.ld + k) = v;
  }
}

template <class Ty, bool AKC, bool BKC, int MODE>
__global__ void __launch_bounds__(kThreads, 1) xent_small_kernel(Product g) {
  __shared__ __attribute__((aligned(1024))) uint8_t L[8][2 * kSmallHalf];
  small_product<Ty, AKC, BKC, MODE>(g, blockIdx.x, is_dz(MODE) || MODE == kOut ? g.scale[0] : 1.0f,
                                    L);
}

// The small form's first launch of a gradient where x needs no copy for dz: dz from x
// as it is (its rows without a target are zeros whatever x holds), the largest gradient
// by each workgroup itself, and the copy that dw reads by the workgroups behind
// `tiles`.  A launch less.
template <class Ty, bool BKC>
__global__ void __launch_bounds__(kThreads, 1) xent_first_kernel(Product g, Copy c, uint32_t tiles,
                                                                 float* scale) {
  __shared__ __attribute__((aligned(1024))) uint8_t L[8][2 * kSmallHalf];
  if (blockIdx.x >= tiles) {
    copy_x(c, (int64_t)(blockIdx.x - tiles) * kThreads + threadIdx.x,
           (int64_t)(gridDim.x - tiles) * kThreads);
    return;
  }
  const float m = largest_grad<kThreads>(g.target, g.grad, g.M, g.V, (float*)L);
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[0] = m;
  small_product<Ty, true, BKC, kDz>(g, blockIdx.x, m, L);
}

// dw and dx in one launch: `tiles` workgroups for dw, the others for dx.
template <class Ty, bool TIED, int MW, int MX>
__global__ void __launch_bounds__(kThreads, 1) xent_pair_kernel(Product w, Product x,
                                                                uint32_t tiles) {
  __shared__ __attribute__((aligned(1024))) uint8_t L[8][2 * kSmallHalf];
  const float scale = w.scale[0];
  if (blockIdx.x < tiles) small_product<Ty, false, false, MW>(w, blockIdx.x, scale, L);
  else small_product<Ty, true, !TIED, MX>(x, blockIdx.x - tiles, scale, L);
}

// lse and loss of every row from its `slots` partial results: 256 / rows threads
// a row, joined in order.
__global__ void __launch_bounds__(256) xent_join_kernel(XentArgs a, const float2* part,
                                                        const float* zt, int slots, int rows) {
  __shared__ float2 tmp[256];
  const int own = threadIdx.x % rows, share = threadIdx.x / rows, shares = 256 / rows;
  const int64_t row = (int64_t)blockIdx.x * rows + own;
  float m = -kMost, s = 0.0f;
  auto put = [&](float2 p) {
    const float n = fmaxf(m, p.x);
    s = s * fa_exp2(m - n) + p.y * fa_exp2(p.x - n);
    m = n;
  };
  if (row < a.T)
    for (int i = share; i < slots; i += shares) put(part[i * a.T + row]);
  for (int half = shares / 2; half > 0; half /= 2) {
    tmp[threadIdx.x] = make_float2(m, s);
    __syncthreads();
    if (share < half) put(tmp[threadIdx.x + half * rows]);
    __syncthreads();
  }
  if (share || row >= a.T) return;
  const float ls = log2f(s);
  const int32_t t = a.target[row];
  // Not lse - z: lse has been rounded at its own size, which leaves nothing of the loss of a
  // confident token (logits near 300: 6e-5 off).  m is the rounded z log2 e of the largest
  // logit and s has what that rounding took, so that they cancel to a few roundings of 1.
  float loss = 0.0f;
  if (t >= 0 && t < a.V) loss = (__builtin_fmaf(-zt[row], kLog2e, m) + ls) * kLn2;
  a.loss[row] = loss < 0.0f ? 0.0f : loss;  // (those roundings)
  if (!a.lse) return;
  // (m + ls) ln 2, rounded once: the gradient's probabilities are off by a step of it.
  // lo: what the sum's rounding took.
  const float sum = m + ls, of_ls = sum - m, lo = (m - (sum - of_ls)) + (ls - of_ls);
  a.lse[row] = fabsf(sum) <= kMost
                   ? __builtin_fmaf(sum, kLn2, __builtin_fmaf(sum, kLn2Rest, lo * kLn2))
                   : sum;
}

// Block 0 (scale set): the largest gradient.  The others: the copy of x.
__global__ void __launch_bounds__(1024) xent_prepare_kernel(Copy c, const float* grad,
                                                            float* scale) {
  __shared__ float tmp[16];
  const int first = scale ? 1 : 0;
  if (scale && blockIdx.x == 0) {
    const float m = largest_grad<1024>(c.target, grad, c.T, c.V, tmp);
    if (threadIdx.x == 0) scale[0] = m;
    return;
  }
  copy_x(c, (int64_t)(blockIdx.x - first) * 1024 + threadIdx.x,
         (int64_t)(gridDim.x - first) * 1024);
}

// A [rows, cols] window of w (row pitch ld) as [rows, pitch] with zeros behind cols.
__global__ void __launch_bounds__(256) xent_pack_kernel(const uint16_t* w, int64_t ld,
                                                        int64_t rows, int64_t cols, int64_t pitch,
                                                        uint16_t* out) {
  const uint32_t per = (uint32_t)(pitch / 8);
  const uint64_t total = (uint64_t)rows * per;  // (a piece of 2^21 x 16384: 2^32)
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * 256) {
    const int64_t r = total >> 32 ? (int64_t)(i / per) : (int64_t)((uint32_t)i / per);
    const int64_t c = (int64_t)(i - r * per) * 8;
    const uint16_t* p = w + r * ld + c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c + 8 <= cols) {
      const Loose16 h = *(const Loose16*)p;
      v = make_uint4(h.v[0], h.v[1], h.v[2], h.v[3]);
    } else {
      uint16_t* h = (uint16_t*)&v;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) h[e] = p[e];
    }
    *(uint4*)(out + r * pitch + c) = v;
  }
}

// A matrix [rows, cols] in 16 bits (row pitch ldo) from its splits' float32 sums.
// target set (dx): rows without a target are zeros.
// rest: the sums of row r lie in rows r and r + rest.
template <class Ty>
__global__ void __launch_bounds__(256) xent_round_kernel(const float* sums, int64_t rows,
                                                         int64_t cols, int splits, int64_t rest,
                                                         const float* scale,
                                                         const int32_t* target, int64_t V,
                                                         uint16_t* out, int64_t ldo) {
  const uint32_t per = (uint32_t)((cols + 7) / 8);
  const uint64_t total = (uint64_t)rows * per;
  const float gain = scale[0] / kDzScale;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * 256) {
    const int64_t r = total >> 32 ? (int64_t)(i / per) : (int64_t)((uint32_t)i / per);
    const int64_t c = (int64_t)(i - r * per) * 8;
    const int n = (int)min((int64_t)8, cols - c);
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const int32_t t = target ? target[r] : 0;
    if (t >= 0 && t < V) {
      for (int p = 0; p < (rest ? 2 * splits : splits); ++p) {
        // (a split has 2 rest rows)
        const float* s = sums + (rest ? p * rest + r : p * rows + r) * cols + c;
        if (cols % 4 == 0 && n == 8) {
          const float4 lo = *(const float4*)s, hi = *(const float4*)(s + 4);
          v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
          v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) v[e] += s[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= gain;
    }
    store8(out + r * ldo + c,
           make_uint4(Ty::pack(v[0], v[1]), Ty::pack(v[2], v[3]), Ty::pack(v[4], v[5]),
                      Ty::pack(v[6], v[7])), n);
  }
}

// ---- plans (sizes alone) --------------------------------------------------------------

constexpr int64_t kCus = 256;
// Tokens whose gradients each workgroup looks through itself: kernels of 100 tokens 22.8 us
// instead of 25.0, of 500 30.0 for 31.2, of 2000 45.6 for 44.2, and a launch less.
constexpr int64_t kFirstTokens = 2048;
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t cdiv(int64_t n, int64_t m) { return (n + m - 1) / m; }

// How a product of M x N over nk k-steps is cut: 256 x 256 or (small) 64 x 64
// tiles, k `splits` ways of `per` steps.  One workgroup runs on a CU at a time.
// Forward and gradients, all kernels, as chosen / 256 x 256 alone / 64 x 64 alone:
// 100 x 256 x 1000 23 / 59 / 23 us, 400 x 1024 x 8000 106 / 121 / 113, 1000 x 1024 x
// 8000 126 / 143 / 183, 16 x 4096 x 32000 256 / 363 / 477.
struct Cut {
  bool small = false;
  int64_t tiles_m = 0, tiles_n = 0, splits = 1, per = 0;
};

// us of a tile of n k-steps.
double tile_us(bool small, int64_t n) {
  return small ? 5.0 + 2.0 * (double)cdiv(n, 8) : 7.0 + 1.6 * (double)n;
}

// The cut that finishes soonest.  most: at most so many splits; their sums are
// written and read again.
Cut choose_cut(int64_t M, int64_t N, int64_t nk, int64_t most) {
  Cut best;
  double least = 1e300;
  for (int small = 0; small < 2; ++small) {
    const int64_t size = small ? SM : BM;
    const int64_t tm = cdiv(M, size), tn = cdiv(N, size);
    for (int rounds = 0; rounds <= 4; ++rounds) {  // of workgroups on all CUs
      const int64_t cus = rounds * kCus / std::max<int64_t>(tm * tn, 1);
      const int64_t s = std::max<int64_t>(1, std::min({cus, nk, most}));
      const int64_t per = cdiv(nk, s);
      double us = (double)cdiv(tm * tn * s, kCus) * tile_us(small, per);
      if (s > 1) us += 4.0 + (double)(M * N * s) * 8.0 / 4.0e6;
      if (us < least * 0.99) {
        least = us;
        best = {small != 0, tm, tn, std::max<int64_t>(1, cdiv(nk, std::max<int64_t>(per, 1))), per};
      }
    }
  }
  return best;
}

// The forward product: `splits` runs of `per` column tiles for each row of tiles.
Cut choose_runs(int64_t M, int64_t N, int64_t nk) {
  Cut best;
  double least = 1e300;
  for (int small = 0; small < 2; ++small) {
    const int64_t size = small ? SM : BM;
    const int64_t tm = cdiv(M, size), tn = cdiv(N, size);
    for (int rounds = 1; rounds <= 8; ++rounds) {
      const int64_t cus = rounds * kCus / std::max<int64_t>(tm, 1);
      const int64_t s = std::max<int64_t>(1, std::min(cus, tn));
      const int64_t per = cdiv(tn, s);
      const double us = (double)cdiv(tm * s, kCus) * (3.0 + (double)per * tile_us(small, nk));
      if (us < least * 0.99) {
        least = us;
        best = {small != 0, tm, tn, cdiv(tn, per), per};
      }
    }
  }
  return best;
}

struct XentPlan {
  bool pack_w, copy_x;     // w's pitch is no multiple of 8; x's no multiple of 64
  int64_t Hp, Tp;          // H and T padded
  int64_t ldx, ldz;        // pitches of the copy of x and of dz
  int64_t piece, pieces;   // columns of the vocabulary at a time
  Cut z, dw, dx;           // of a whole piece
  bool dx_sums;            // dx is added up in float32
  bool rest;               // dz and x lie in rows 0 .. 31, dz's remainders and x in 32 .. 63
  int64_t dz_rows;         // of the product for dx
  // offsets of the working memory
  size_t part, zt, x, w, dz, sums, dw_sums, scale, bytes;
};

XentPlan make_plan(int64_t T, int64_t H, int64_t V, int tied, bool grad) {
  XentPlan p;
  std::memset(&p, 0, sizeof p);
  p.pack_w = (tied ? H : V) % 8 != 0;
  p.copy_x = grad || H % BK != 0;
  p.Hp = up(H, BK);
  p.Tp = up(T, BK);
  p.piece = V;
  if (grad) {
    // dz of a piece: 2^25 values at least, 2^31 at most beyond 2^17 tokens
    const int64_t t = std::max<int64_t>(T, 1);
    p.piece = std::max(std::min(kPiece, ((int64_t)1 << 31) / t), ((int64_t)1 << 25) / t);
    p.piece = std::max<int64_t>(p.piece, BN);
  }
  if (!grad && p.pack_w) p.piece = kPiece;
  p.piece = std::min(up(p.piece, BN), up(V, BN));
  p.pieces = cdiv(V, p.piece);
  // (rows a power of two apart would meet in the same channels of the L2: dx 895 us for
  // 874 a piece, dw 801 for 808)
  p.ldx = p.Hp + 64;
  p.ldz = p.piece + 64;
  const int64_t n = std::min(p.piece, V);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
  };
  if (grad) {
    p.z = choose_cut(T, n, p.Hp / BK, 1);
    p.dw = choose_cut(tied ? n : H, tied ? H : n, p.Tp / BK, 16);
    p.rest = T > 0 && T <= kRestRows;
    p.dz_rows = p.rest ? 2 * kRestRows : T;
    p.dx = choose_cut(p.dz_rows, H, up(n, BK) / BK, 64);
    p.dx_sums = p.rest || p.pieces > 1 || p.dx.splits > 1;
    p.dz = take((size_t)p.Tp * p.ldz * 2);
    if (p.dx_sums) p.sums = take((size_t)p.dx.splits * p.dz_rows * H * 4);
    if (p.dw.splits > 1) p.dw_sums = take((size_t)p.dw.splits * n * H * 4);
    p.scale = take(4);
  } else {
    p.z = choose_runs(T, n, p.Hp / BK);
    p.part = take((size_t)p.pieces * p.z.splits * T * sizeof(float2));
    p.zt = take((size_t)T * 4);
  }
  if (p.copy_x) p.x = take((size_t)p.Tp * p.ldx * 2);
  if (p.pack_w) p.w = take((size_t)(tied ? p.piece * p.Hp : H * p.piece) * 2);
  p.bytes = at;
  return p;
}

template <class Ty, bool AKC, bool BKC, int MODE>
void launch_product(Product g, const Cut& c, hipStream_t stream) {
  const int64_t size = c.small ? SM : BM;
  g.tiles_m = (int)cdiv(g.M, size);
  g.tiles_n = (int)cdiv(g.N, size);
  g.per = (int)c.per;
  int64_t blocks = (int64_t)g.tiles_m * g.tiles_n;
  if (MODE == kStats) blocks = (int64_t)g.tiles_m * g.splits;
  if (MODE == kSum) blocks *= g.splits;
  if (blocks == 0) return;
  if (c.small)
    hipLaunchKernelGGL((xent_small_kernel<Ty, AKC, BKC, MODE>), dim3((unsigned)blocks),
                       dim3(kThreads), 0, stream, g);
  else
    hipLaunchKernelGGL((xent_product_kernel<Ty, AKC, BKC, MODE>),
                       dim3((unsigned)(MODE == kStats ? blocks : std::min(blocks, kCus))),
                       dim3(kThreads), 0, stream, g);
  REW_HIP(hipGetLastError());
}

// dw and dx of small cuts.
template <class Ty>
void launch_pair(Product w, Product x, const XentPlan& p, int tied, hipStream_t stream) {
  for (Product* g : {&w, &x}) {
    g->tiles_m = (int)cdiv(g->M, SM);
    g->tiles_n = (int)cdiv(g->N, SM);
  }
  w.per = (int)p.dw.per;
  x.per = (int)p.dx.per;
  const int64_t nw = (int64_t)w.tiles_m * w.tiles_n * (p.dw.splits > 1 ? w.splits : 1);
  const int64_t nx = (int64_t)x.tiles_m * x.tiles_n * (p.dx_sums ? x.splits : 1);
  auto launch = [&](auto t, auto mw, auto mx) {
    hipLaunchKernelGGL(
        (xent_pair_kernel<Ty, decltype(t)::value, decltype(mw)::value, decltype(mx)::value>),
        dim3((unsigned)(nw + nx)), dim3(kThreads), 0, stream, w, x, (uint32_t)nw);
  };
  auto by_x = [&](auto t, auto mw) {
    if (p.dx_sums) launch(t, mw, std::integral_constant<int, kSum>());
    else launch(t, mw, std::integral_constant<int, kOut>());
  };
  auto by_w = [&](auto t) {
    if (p.dw.splits > 1) by_x(t, std::integral_constant<int, kSum>());
    else by_x(t, std::integral_constant<int, kOut>());
  };
  if (tied) by_w(std::true_type());
  else by_w(std::false_type());
  REW_HIP(hipGetLastError());
}

template <class Ty>
void launch_round(const float* sums, int64_t rows, int64_t cols, int64_t splits, int64_t rest,
                  const float* scale, const int32_t* target, int64_t V, void* out, int64_t ldo,
                  hipStream_t stream) {
  const int64_t blocks = std::min<int64_t>(cdiv(rows * cdiv(cols, 8), 256), kCus * 16);
  hipLaunchKernelGGL((xent_round_kernel<Ty>), dim3((unsigned)blocks), dim3(256), 0, stream, sums,
                     rows, cols, (int)splits, rest, scale, target, V, (uint16_t*)out, ldo);
  REW_HIP(hipGetLastError());
}

// A piece of w, columns v0 .. v0 + n of the vocabulary, packed first where its
// rows are not 16-byte aligned.
struct Piece {
  const uint16_t* p;
  int64_t ld, len;
};
template <class A>
Piece piece_of(const A& a, const XentPlan& p, int64_t v0, int64_t n, uint8_t* work,
               hipStream_t stream, int* launches) {
  const uint16_t* w = (const uint16_t*)a.w + (a.tied ? v0 * a.H : v0);
  if (!p.pack_w) return {w, a.tied ? a.H : a.V, a.H * a.V - (a.tied ? v0 * a.H : v0)};
  const int64_t rows = a.tied ? n : a.H, cols = a.tied ? a.H : n, pitch = a.tied ? p.Hp : p.piece;
  uint16_t* out = (uint16_t*)(work + p.w);
  const int64_t blocks = std::min<int64_t>(cdiv(rows * pitch / 8, 256), kCus * 16);
  hipLaunchKernelGGL(xent_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, w,
                     a.tied ? a.H : a.V, rows, cols, pitch, out);
  REW_HIP(hipGetLastError());
  ++*launches;
  return {out, pitch, rows * pitch};
}

template <class Ty>
int run_xent(const XentArgs& a, hipStream_t stream) {
  const XentPlan p = make_plan(a.T, a.H, a.V, a.tied, false);
  uint8_t* work = (uint8_t*)a.work;
  int launches = 0;
  Product g;
  std::memset(&g, 0, sizeof g);
  g.a = {(const uint16_t*)a.x, a.H, a.T * a.H, a.H};
  if (p.copy_x) {
    uint16_t* x = (uint16_t*)(work + p.x);
    const Copy c = {(const uint16_t*)a.x, a.target, x, a.T, a.H, a.V, p.Tp, p.Hp, p.ldx, 1, 0};
    const int64_t blocks = std::min<int64_t>(cdiv(p.Tp * p.Hp / 8, 1024), kCus * 4);
    hipLaunchKernelGGL(xent_prepare_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream, c,
                       (const float*)nullptr, (float*)nullptr);
    REW_HIP(hipGetLastError());
    ++launches;
    g.a = {x, p.ldx, p.Tp * p.ldx, p.Hp};
  }
  g.M = a.T;
  g.K = p.Hp;
  g.V = (int)a.V;
  g.target = a.target;
  g.part = (float2*)(work + p.part);
  g.zt = (float*)(work + p.zt);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(p.piece, a.V - v0);
    const Piece w = piece_of(a, p, v0, n, work, stream, &launches);
    g.n0 = (int)v0;
    g.N = n;
    g.splits = (int)cdiv(cdiv(n, p.z.small ? SM : BN), p.z.per);
    g.b = {w.p, w.ld, w.len, a.tied && p.pack_w ? p.Hp : a.H};
    if (a.tied) launch_product<Ty, true, true, kStats>(g, p.z, stream);
    else launch_product<Ty, true, false, kStats>(g, p.z, stream);
    ++launches;
    g.slot0 += g.splits;
  }
  int rows = 64;  // of a workgroup of the join
  while (rows > 1 && a.T < rows * kCus) rows /= 2;
  hipLaunchKernelGGL(xent_join_kernel, dim3((unsigned)cdiv(a.T, rows)), dim3(256), 0, stream, a,
                     g.part, g.zt, g.slot0, rows);
  REW_HIP(hipGetLastError());
  return launches + 1;
}

template <class Ty>
int run_xent_grad(const XentGradArgs& a, hipStream_t stream) {
  const XentPlan p = make_plan(a.T, a.H, a.V, a.tied, true);
  uint8_t* work = (uint8_t*)a.work;
  int launches = 0;
  uint16_t* x = (uint16_t*)(work + p.x);
  uint16_t* dz = (uint16_t*)(work + p.dz);
  float* scale = (float*)(work + p.scale);
  const Copy copy = {(const uint16_t*)a.x, a.target, x, a.T, a.H, a.V, p.Tp, p.Hp, p.ldx, 0, p.rest};
  const bool first = a.T && p.z.small && p.pieces == 1 && !p.pack_w && a.H % BK == 0 &&
                     a.T <= kFirstTokens;
  if (!first) {
    const int64_t blocks = 1 + std::min<int64_t>(cdiv(p.Tp * p.Hp / 8, 1024), kCus * 4);
    hipLaunchKernelGGL(xent_prepare_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream, copy,
                       a.grad, scale);
    REW_HIP(hipGetLastError());
    ++launches;
  }
  const Opnd xk = {x, p.ldx, p.Tp * p.ldx, p.Hp};   // k = embed
  const Opnd xt = {x, p.ldx, p.Tp * p.ldx, p.Tp};   // k = tokens
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(p.piece, a.V - v0);
    const Piece w = piece_of(a, p, v0, n, work, stream, &launches);
    Product g;
    std::memset(&g, 0, sizeof g);
    g.n0 = (int)v0;
    g.V = (int)a.V;
    g.lse = a.lse;
    g.grad = a.grad;
    g.scale = scale;
    if (a.T) {
      // dz, zeros behind its n columns up to the next multiple of BN
      Product d = g;
      d.a = xk;
      d.b = {w.p, w.ld, w.len, a.tied && p.pack_w ? p.Hp : a.H};
      d.M = a.T;
      d.N = n;
      d.K = p.Hp;
      d.target = a.target;
      d.out = dz;
      d.ldo = p.ldz;
      d.rows_out = p.rest ? kRestRows : p.Tp;
      d.rest = p.rest ? kRestRows : 0;
      if (first) {
        d.a = {(const uint16_t*)a.x, a.H, a.T * a.H, a.H};
        d.tiles_m = (int)p.z.tiles_m;
        d.tiles_n = (int)p.z.tiles_n;
        const uint32_t tiles = (uint32_t)(d.tiles_m * d.tiles_n);
        const uint32_t blocks =
            tiles + (uint32_t)std::min<int64_t>(cdiv(p.Tp * p.Hp / 8, kThreads), kCus);
        if (a.tied)
          hipLaunchKernelGGL((xent_first_kernel<Ty, true>), dim3(blocks), dim3(kThreads), 0, stream,
                             d, copy, tiles, scale);
        else
          hipLaunchKernelGGL((xent_first_kernel<Ty, false>), dim3(blocks), dim3(kThreads), 0,
                             stream, d, copy, tiles, scale);
        REW_HIP(hipGetLastError());
      } else if (p.rest && !p.z.small) {
        if (a.tied) launch_product<Ty, true, true, kDzRest>(d, p.z, stream);
        else launch_product<Ty, true, false, kDzRest>(d, p.z, stream);
      } else if (a.tied) {
        launch_product<Ty, true, true, kDz>(d, p.z, stream);
      } else {
        launch_product<Ty, true, false, kDz>(d, p.z, stream);
      }
      ++launches;
    }
    Product dw = g;
    {
      Product& d = dw;
      const Opnd dzt = {dz, p.ldz, p.Tp * p.ldz, p.Tp};
      d.a = a.tied ? dzt : xt;
      d.b = a.tied ? xt : dzt;
      d.M = d.rows_out = a.tied ? n : a.H;
      d.N = a.tied ? a.H : n;
      d.K = p.Tp;
      d.out = (uint16_t*)a.dw + (a.tied ? v0 * a.H : v0);
      d.ldo = a.tied ? a.H : a.V;
      d.splits = (int)p.dw.splits;
    }
    const bool dw_sums = dw.splits > 1;
    void* dw_out = dw.out;
    if (dw_sums) dw.out = work + p.dw_sums;
    Product dx = g;
    if (a.T) {
      Product& d = dx;
      d.K = up(n, BK);
      d.a = {dz, p.ldz, p.Tp * p.ldz, d.K};
      // (a packed piece has zeros behind n; else the rows' or columns' end is w's own)
      d.b = {w.p, w.ld, w.len, a.tied ? n : p.pack_w ? d.K : n};
      d.M = d.rows_out = p.dz_rows;
      d.N = a.H;
      d.splits = (int)cdiv(d.K / BK, p.dx.per);  // (the first piece has the most)
      d.add = i > 0;
      d.out = p.dx_sums ? (void*)(work + p.sums) : a.dx;
      d.ldo = a.H;
      d.target = p.dx_sums ? nullptr : a.target;
    }
    if (a.T && p.dw.small && p.dx.small) {
      launch_pair<Ty>(dw, dx, p, a.tied, stream);
      ++launches;
    } else {
      if (dw_sums) launch_product<Ty, false, false, kSum>(dw, p.dw, stream);
      else launch_product<Ty, false, false, kOut>(dw, p.dw, stream);
      ++launches;
      if (a.T) {
        if (p.dx_sums && a.tied) launch_product<Ty, true, false, kSum>(dx, p.dx, stream);
        else if (p.dx_sums) launch_product<Ty, true, true, kSum>(dx, p.dx, stream);
        else if (a.tied) launch_product<Ty, true, false, kOut>(dx, p.dx, stream);
        else launch_product<Ty, true, true, kOut>(dx, p.dx, stream);
        ++launches;
      }
    }
    if (dw_sums) {
      launch_round<Ty>((const float*)dw.out, dw.M, dw.N, dw.splits, 0, scale, nullptr, 1,
                       dw_out, dw.ldo, stream);
      ++launches;
    }
  }
  if (a.T && p.dx_sums) {
    launch_round<Ty>((const float*)(work + p.sums), a.T, a.H, p.dx.splits, p.rest ? kRestRows : 0,
                     scale, a.target, a.V, a.dx, a.H, stream);
    ++launches;
  }
  return launches;
}

}  // namespace

size_t xent_ws_bytes(const XentArgs& a) { return make_plan(a.T, a.H, a.V, a.tied, false).bytes; }

int launch_xent(const XentArgs& a, hipStream_t stream) {
  if (a.T == 0) return 0;
  return a.f16 ? run_xent<MmaF16>(a, stream) : run_xent<MmaBf16>(a, stream);
}

size_t xent_grad_ws_bytes(const XentGradArgs& a) {
  return make_plan(a.T, a.H, a.V, a.tied, true).bytes;
}

int launch_xent_grad(const XentGradArgs& a, hipStream_t stream) {
  return a.f16 ? run_xent_grad<MmaF16>(a, stream) : run_xent_grad<MmaBf16>(a, stream);
}

}  // namespace rew
