// Device helpers shared by the attention kernels: MFMA operand types, the hardware
// exp2 and max, packing to 16 bits, and the DMA from memory into LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rew {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) void lds_void;

// 2^x with the hardware v_exp_f32 (1 ulp) and no denormal-range fix-up:
// every argument here is <= 0 (a score minus its running max), and results
// below 2^-126 are probabilities far under one bf16 ulp of the row sum.
// (The library exp2f wraps the instruction in a range test and two
// rescales; on the Llama shape the flash kernel ran 9 % faster without.)
__device__ __forceinline__ float fa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// max(a, b, c) in one v_max3_f32.  fmaxf would first quiet signalling NaNs
// with a v_max_f32 x, x per operand (MFMA results are not known to be
// canonical); a quiet NaN operand is ignored either way.  The compiler does
// not see that this reads a register: the wait states between a MFMA and the
// first use of its result must come from other code before it.
__device__ __forceinline__ float fa_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// max(a, b, c) in one v_maximum3_f32, which the compiler knows and schedules; NaN
// if one is.
__device__ __forceinline__ float fa_maximum3(float a, float b, float c) {
  return __builtin_elementwise_maximum(a, __builtin_elementwise_maximum(b, c));
}

// Two fp32 values rounded to bf16 (RNE; v_cvt_pk_bf16_f32), packed.
__device__ __forceinline__ uint32_t cvt_bf16x2(float a, float b) {
  const bf16x2_t v = __builtin_convertvector((f32x2_t){a, b}, bf16x2_t);
  uint32_t u;
  __builtin_memcpy(&u, &v, 4);
  return u;
}

__device__ __forceinline__ void dma16(const void* src, uint16_t* lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)lds, 16, 0, 0);
}

// Buffer descriptor over `bytes` bytes at `base`; a read past them returns
// zeros and touches no memory.  Both are wave-uniform and readfirstlane says
// so, which keeps the descriptor in SGPRs.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fa_rsrc(const void* base,
                                                          uint32_t bytes = 0x7fffffff) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  void* p = (void*)(uintptr_t)(((uint64_t)hi << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)__builtin_amdgcn_readfirstlane(bytes),
                                           0x00020000);
}
// 16 bytes per lane from base + voff + soff into LDS (buffer_load ... lds):
// the per-lane offset is fixed, the tile advance is the scalar `soff`.
__device__ __forceinline__ void dma16_buf(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff,
                                          uint16_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, voff, soff, 0, 0);
}

__device__ __forceinline__ void dma16_lds(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff,
                                          lds_void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, voff, soff, 0, 0);
}

// Workgroup barrier without the memory fence of __syncthreads (which would
// also wait for every DMA in flight); callers wait for what they need first.
// No instruction is scheduled across it: the ping-pong phases it separates
// must keep their own MFMA or VALU work.
__device__ __forceinline__ void block_barrier_fa() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// ---- operand types of the packed and paged kernels --------------------------------
//
// The 16-bit type of Q, K, V and of the probabilities that feed the second
// product.  kShift: the probabilities are stored as 2^kShift p, and kLazy2:
// the running max of the softmax moves only when a row's max grew by more
// than 2^kLazy2.  bfloat16 has float32's range, so it needs no shift; float16
// is normal from 2^-14 to 2^16: 2^11 p stays below 2^15 and keeps 11 bits
// down to p = 2^-25, where an unshifted probability would have lost them at
// 2^-14.
struct MmaBf16 {
  typedef bf16x8_t frag;
  static constexpr float kShift = 0.0f, kLazy2 = 11.5f, kGradShift = 0.0f;
  static constexpr bool kScaled = false;  // dS is stored scaled (k_packed_grad.hip)
  // PackedArgs::rest: a step, by the row's max, and the least max that counts
  static constexpr float kRestStep = 0x1p-8f / 127.0f, kRestLeast = 0x1p-100f;
  static constexpr uint32_t kInf = 0x7f80;
  static __device__ __forceinline__ f32x16_t mma(frag a, frag b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return cvt_bf16x2(a, b); }
  static __device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float hi(uint32_t u) {
    return __uint_as_float(u & 0xffff0000u);
  }
};
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
struct MmaF16 {
  typedef f16x8_t frag;
  static constexpr float kShift = 11.0f, kLazy2 = 4.0f, kGradShift = 15.0f;
  static constexpr bool kScaled = true;
  // (below 2^-14 a rounding takes up to 2^-25, whatever the value)
  static constexpr float kRestStep = 0x1p-11f / 127.0f, kRestLeast = 0x1p-14f;
  static constexpr uint32_t kInf = 0x7c00;
  static __device__ __forceinline__ f32x16_t mma(frag a, frag b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const f16x2_t v = __builtin_convertvector((f32x2_t){a, b}, f16x2_t);
    uint32_t u;
    __builtin_memcpy(&u, &v, 4);
    return u;
  }
  static __device__ __forceinline__ float lo(uint32_t u) {
    f16x2_t v;
    __builtin_memcpy(&v, &u, 4);
    return (float)v[0];
  }
  static __device__ __forceinline__ float hi(uint32_t u) {
    f16x2_t v;
    __builtin_memcpy(&v, &u, 4);
    return (float)v[1];
  }
};

// max over lanes l and l ^ 32
__device__ __forceinline__ float fa_max_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __builtin_elementwise_maximum(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float fa_sum_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// A value that is the same in every lane, as the compiler does not know.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Sums over the wave with the data-parallel moves of the vector ALU (a shuffle
// through LDS per step takes ten times as long): rows of 16 lanes by shifts,
// then lanes 15, 31 and 47 onto the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_moved(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {  // inclusive
  x = add_moved<0x111, 0xf>(x);
  x = add_moved<0x112, 0xf>(x);
  x = add_moved<0x114, 0xf>(x);
  x = add_moved<0x118, 0xf>(x);
  x = add_moved<0x142, 0xa>(x);
  return add_moved<0x143, 0xc>(x);
}
__device__ __forceinline__ int wave_sum(int x) {
  return __builtin_amdgcn_readlane(wave_scan(x), 63);
}
// likewise the running max of values >= 0
template <int CTRL, int ROWS>
__device__ __forceinline__ int max_moved(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_max_scan(int x) {
  x = max_moved<0x111, 0xf>(x);
  x = max_moved<0x112, 0xf>(x);
  x = max_moved<0x114, 0xf>(x);
  x = max_moved<0x118, 0xf>(x);
  x = max_moved<0x142, 0xa>(x);
  return max_moved<0x143, 0xc>(x);
}
// ---- packed sequences ---------------------------------------------------------------
//
// Sequence s owns rows [starts[s], starts[s + 1]) of T.  The rows before the
// first and behind the last sequence belong to none: they count as sequences
// -1 and n_seq, without keys.  starts is device data that the host does not
// see, so every value is clamped into [0, T], and one below an earlier value
// counts as that: no row outside the tensors is touched, no row belongs to two
// sequences, and the host's bounds on tiles, whose sums fit 31 bits, hold for any
// starts.
struct SeqTile {
  int seq;     // -1 .. n_seq; -2: there is no such tile
  int first;   // its first row
  int n;       // its rows
  int tile;    // the tile's index in the sequence
  __device__ __forceinline__ bool real(int n_seq) const { return seq >= 0 && seq < n_seq; }
};
__device__ __forceinline__ int seq_bound(const int32_t* starts, int n_seq, int T, int s) {
  if (s < 0) return 0;
  if (s > n_seq) return T;
  return min(max(starts[s], 0), T);
}
// The rows of the 64 sequences from `base`, one per lane (none past n_seq).
// floor: 0 for base -1, then what the step before left (the first row of
// sequence base).
struct SeqRows {
  int s, first, n;
  __device__ __forceinline__ SeqRows(const int32_t* starts, int n_seq, int T, int base, int& floor)
      : s(base + (int)(threadIdx.x & 63)) {
    first = max(wave_max_scan(seq_bound(starts, n_seq, T, s)), floor);
    const int end = max(seq_bound(starts, n_seq, T, s + 1), first);
    n = s > n_seq ? 0 : end - first;
    floor = __builtin_amdgcn_readlane(end, 63);
  }
};
// Tile `idx` of the sequences' tiles of `per` units, a row holding `units`
// (query heads of a KV head; 1 for keys), in sequence order.  One wave (every
// wave of a workgroup does the same): 64 sequences a step, their tile counts
// summed over the lanes.
__device__ __forceinline__ SeqTile find_tile(const int32_t* starts, int n_seq, int T, int units,
                                             int per, int idx) {
  SeqTile r;
  r.seq = -2;
  r.first = r.n = r.tile = 0;
  int floor = 0;
  for (int base = -1; base <= n_seq; base += 64) {
    const SeqRows x(starts, n_seq, T, base, floor);
    const int tiles = (int)(((int64_t)x.n * units + per - 1) / per);
    const int sum = wave_scan(tiles);
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (idx < total) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > idx));
      r.seq = base + at;
      r.first = __builtin_amdgcn_readlane(x.first, at);
      r.n = __builtin_amdgcn_readlane(x.n, at);
      r.tile = idx - __builtin_amdgcn_readlane(sum - tiles, at);
      return r;
    }
    idx -= total;
  }
  return r;
}
// The rank-th of the sequences' tiles in the order of falling level: a
// sequence's tiles have the levels lift + 1 .. lift + tiles (its own per
// lane; level by level, in sequence order), tile = level - lift - 1.  A level
// stands for the tile's work, so the heaviest tiles of all sequences start
// first.  At most 64 sequences (kLevelSeqs real ones), one per lane.
constexpr int kLevelSeqs = 62;
__device__ __forceinline__ SeqTile level_tile(int s, int first, int n, int tiles, int lift,
                                              int rank) {
  SeqTile r;
  r.seq = -2;
  r.first = r.n = r.tile = 0;
  if (rank >= wave_sum(tiles)) return r;
  auto above = [&](int level) { return min(max(lift + tiles - level + 1, 0), tiles); };
  int top = lift + tiles;  // the levels of all lanes end here
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = max(top, __shfl_xor(top, d));
  // the highest level that, with those above it, has more than `rank` tiles
  int lo = 1, hi = __builtin_amdgcn_readfirstlane(top) + 1;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (wave_sum(above(mid)) > rank) lo = mid;
    else hi = mid;
  }
  rank -= wave_sum(above(lo + 1));
  const uint64_t have = __builtin_amdgcn_ballot_w64(lift < lo && lo <= lift + tiles);
  const int lane = threadIdx.x & 63;
  const uint64_t before = have & ((1ull << lane) - 1);
  const int at = __builtin_ctzll(
      __builtin_amdgcn_ballot_w64(((have >> lane) & 1) && __builtin_popcountll(before) == rank));
  r.seq = __builtin_amdgcn_readlane(s, at);
  r.first = __builtin_amdgcn_readlane(first, at);
  r.n = __builtin_amdgcn_readlane(n, at);
  r.tile = lo - __builtin_amdgcn_readlane(lift, at) - 1;
  return r;
}
// level_tile over tiles of `per` units (find_tile's), the work growing with
// the tile's index.
__device__ __forceinline__ SeqTile rising_tile(const int32_t* starts, int n_seq, int T, int units,
                                               int per, int rank) {
  int floor = 0;
  const SeqRows x(starts, n_seq, T, -1, floor);
  return level_tile(x.s, x.first, x.n, (int)(((int64_t)x.n * units + per - 1) / per), 0, rank);
}

// r / g and r % g for 0 <= r < 2^31: one multiplication by floor((2^32 - 1) / g)
// falls short of the quotient by at most one.
struct DivBy {
  uint32_t g, m;
  __device__ __forceinline__ explicit DivBy(int d) : g(d), m(0xffffffffu / (uint32_t)d) {}
  __device__ __forceinline__ int div(int r, int& rem) const {
    uint32_t q = __umulhi((uint32_t)r, m);
    uint32_t x = (uint32_t)r - q * g;
    const bool up = x >= g;
    q += up;
    x -= up ? g : 0;
    rem = (int)x;
    return (int)q;
  }
};

// A bound on find_tile's tiles, known on the host.
inline int64_t max_seq_tiles(int64_t T, int64_t n_seq, int64_t units, int64_t per) {
  return T * units / per + n_seq + 2;
}

// Rows of D 16-bit values, `stride` elements apart, read a tile of `step_rows`
// at a time through a descriptor that ends with the last row: what lies
// behind it reads as zeros and touches no memory.
struct RowTiles {
  const uint16_t* p;
  int64_t step, left;  // elements per tile; bytes from p to the end of the last row
  __device__ __forceinline__ RowTiles(const uint16_t* base, int64_t row, int64_t rows,
                                      int64_t stride, int D, int step_rows)
      : p(base + row * stride), step(step_rows * stride),
        left(rows > row ? ((rows - 1 - row) * stride + D) * 2 : 0) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t next() {
    const __amdgpu_buffer_rsrc_t r =
        fa_rsrc(p, (uint32_t)(left < 0 ? 0 : left < 0x7fffffff ? left : 0x7fffffff));
    p += step;
    left -= step * 2;
    return r;
  }
};

// ---- keys of packed and paged attention ----------------------------------------------

namespace pa {
constexpr int BK = 64;  // keys per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
}  // namespace pa

// Zeros that stand for the rows of keys that are not there.
static __device__ __attribute__((aligned(256))) uint16_t g_zero_row[128];

// A request's block table, 64 entries at a time, one per lane; pages outside
// the cache (or the table) are -1.
struct PageWindow {
  const int32_t* row;
  int width, log_page, base, id;
  uint32_t pages;
  uint64_t bad;  // lanes without a page
  __device__ __forceinline__ PageWindow(const int32_t* r, int w, int lp, int64_t p)
      : row(r), width(w), log_page(lp), base(-64), id(-1), pages((uint32_t)min(p, (int64_t)0x7fffffff)),
        bad(~0ull) {}
  // makes the window hold the pages of the 64 keys from k0 (or 32, a multiple of it)
  __device__ __forceinline__ void reach(int k0) {
    const int b = (k0 >> log_page) & ~63;
    if (b == base) return;
    base = b;
    const int i = b + (int)(threadIdx.x & 63);
    const int v = i < width ? row[i] : -1;
    id = (uint32_t)v < pages ? v : -1;
    bad = __builtin_amdgcn_ballot_w64(id < 0);
  }
  // the page of key j (of a tile that the window holds)
  __device__ __forceinline__ int page(int j) const {
    return __builtin_amdgcn_ds_bpermute(((j >> log_page) - base) * 4, id);
  }
  // .. of a key j that is the same in all lanes
  __device__ __forceinline__ int page_uniform(int j) const {
    return __builtin_amdgcn_readlane(id, (j >> log_page) - base);
  }
  __device__ __forceinline__ bool missing(int j) const {
    return (bad >> ((j >> log_page) - base)) & 1;
  }
  // whether any of the `keys` keys from k0, up to key `end` - 1, has no page
  __device__ __forceinline__ bool any_missing(int k0, int keys, int end) const {
    const int first = (k0 >> log_page) - base;
    const int n = ((min(end - k0, keys) - 1) >> log_page) + 1;
    return end > k0 && ((bad >> first) & (n == 64 ? ~0ull : (1ull << n) - 1)) != 0;
  }
};

// The keys of a tile that a lane's row sees, one word per 32 keys: bit p for key
// p + g 4, below `seen` of the tile and with its bit in `none` clear.
template <int NB>
struct Seen {
  uint32_t bits[NB];
  __device__ __forceinline__ Seen(int seen, uint64_t none, int g) {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      const int n = seen - kb * 32 - g * 4;
      const uint32_t below = n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
      bits[kb] = below & ~(uint32_t)(none >> (kb * 32 + g * 4));
    }
  }
};

// One softmax step over a tile of S^T (32 NB keys x 32 rows): lane (c, g) holds
// row c's scores of keys kb 32 + (e / 4) 8 + g 4 + e % 4 in s[kb][e], of which
// `vis` are visible (all, if PLAIN).  The running max (of t = log2(e) scale s)
// moves, rescaling O and the sum, only when some row's max grew by more than
// 2^kLazy2; until then the probabilities stay below 2^(kLazy2 + kShift).
//
// First half: the scores masked, the max moved; the factor for O and the sum
// (1 in every lane of the wave, mostly).
template <class M, bool PLAIN, int NB>
__device__ __forceinline__ float soft_max(f32x16_t (&s)[NB], const Seen<NB>& vis, float sl2,
                                          float& m_run) {
  float mx[NB];
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      if constexpr (!PLAIN) {  // (two instructions per score, a bit's field and a bitwise select)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)vis.bits[kb],
                                                             ((e >> 2) * 8 + (e & 3)) + i, 1);
          s[kb][e + i] =
              __uint_as_float((__float_as_uint(s[kb][e + i]) & m) | (0xff800000u & ~m));
        }
      }
      float& m = mx[kb];
      m = e == 0 ? __builtin_elementwise_maximum(s[kb][0], s[kb][1])
                 : fa_maximum3(m, s[kb][e], s[kb][e + 1]);
    }
  const float mt =
      fa_max_halves(NB == 1 ? mx[0] : __builtin_elementwise_maximum(mx[0], mx[NB - 1])) * sl2;
  const float m_new = __builtin_elementwise_maximum(m_run, mt);
  const bool grow = !(m_new - m_run <= M::kLazy2);  // (also while m_run is -inf)
  const bool rescale = __builtin_amdgcn_ballot_w64(grow) != 0;
  const float m_use = m_new == -INFINITY ? 0.0f : m_new;
  const float alpha = rescale ? fa_exp2(m_run - m_use) : 1.0f;
  m_run = rescale ? m_new : m_run;
  return alpha;
}
// Second half: the probabilities, packed for the second product, and their sum.
template <class M, int NB>
__device__ __forceinline__ void soft_exp(const f32x16_t (&s)[NB], float sl2, float m_run,
                                         uint32_t (&pk)[NB][8], float& l_run) {
  const float base = M::kShift - (m_run == -INFINITY ? 0.0f : m_run);
  float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float p0 = fa_exp2(fmaf(s[kb][e], sl2, base));
      const float p1 = fa_exp2(fmaf(s[kb][e + 1], sl2, base));
      pk[kb][e >> 1] = M::pack(p0, p1);
      ps[e & 2] += p0;
      ps[(e & 2) + 1] += p1;
    }
  l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
}
// A value that a row does not see must not reach its output, and 0 times an
// infinity or NaN would.  Where some row of a block does not see all keys of a
// tile (the last tiles of causal blocks), the tile of V is looked through
// first; the infinities and NaN found are added to the rows that see them
// by themselves, and are zeros in the product.
//
// The largest magnitude (as bits) of the values seen, two by two.
template <class M>
struct Largest {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
  __device__ __forceinline__ void add(uint32_t w) {
    const uint32_t x = w & 0x7fff7fffu;
    u16x2 y;
    __builtin_memcpy(&y, &x, 4);
    most = __builtin_elementwise_max(most, y);
  }
  __device__ __forceinline__ bool special() const {
    return most[0] >= M::kInf || most[1] >= M::kInf;
  }
};
// Whether an LDS tile of KEYS rows of D holds an infinity or NaN.
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
template <class M, int KEYS, int D, class P>
__device__ __forceinline__ bool any_special(P tile, int lane = threadIdx.x & 63) {
  Largest<M> most;
#pragma unroll
  for (int i = 0; i < KEYS * D / 512; ++i) {
    const u32x4_t w = *(__attribute__((address_space(3))) const u32x4_t*)(
        tile + i * 512 + lane * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) most.add(w[j]);
  }
  return __builtin_amdgcn_ballot_w64(most.special()) != 0;
}
// The infinities and NaN of two values, zeros for others.
template <class M>
__device__ __forceinline__ uint32_t special(uint32_t w) {
  const uint32_t lo = (w & 0x7fffu) >= M::kInf ? 0xffffu : 0u;
  const uint32_t hi = (w & 0x7fff0000u) >= M::kInf << 16 ? 0xffff0000u : 0u;
  return w & (lo | hi);
}
// Key j's chunk x of 8 columns of a V tile lies at x ^ value_swizzle(j).
template <int D>
__device__ __forceinline__ int value_swizzle(int j) {
  return (4 * (j & 3)) % (D / 8);
}
// o += the infinities and NaN of the rows [from, to) of a tile's KEYS rows
// (o[dt][r 4 + i]: column dt 32 + r 8 + g 4 + i; row j's chunk x of 8 columns at
// x ^ swizzle(j)).
template <class M, int KEYS, int D, class P, class Swizzle>
__device__ __forceinline__ void add_special(f32x16_t (&o)[D / 32], P tile, int from, int to, int g,
                                            Swizzle swizzle) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll 1
      for (int j = 0; j < KEYS; ++j) {
        const int ch = (dt * 4 + r) ^ swizzle(j);
        const u32x2 w =
            *(__attribute__((address_space(3))) const u32x2*)(tile + j * D + ch * 8 + g * 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = j >= from && j < to ? special<M>(w[i]) : 0u;
          o[dt][r * 4 + i * 2] += M::lo(x);
          o[dt][r * 4 + i * 2 + 1] += M::hi(x);
        }
      }
}
// The tile's infinities and NaN become zeros; thread t of N has its part.
template <class M, int KEYS, int D, int N, class P>
__device__ __forceinline__ void clear_special(P tile, int t) {
#pragma unroll 1
  for (int i = t; i < KEYS * D / 2; i += N) {
    auto* p = (__attribute__((address_space(3))) uint32_t*)tile + i;
    *p ^= special<M>(*p);
  }
}
// O and the sum take the factor of soft_max.
template <int DT>
__device__ __forceinline__ void soft_rescale(f32x16_t (&o)[DT], float& l_run, float alpha) {
  if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) == 0) return;
  l_run *= alpha;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
}

}  // namespace rew
