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
#include <hip/hip_runtime.h>

#include <algorithm>

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
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMost = 3.402823466e38f;
// dz is stored as 2^14 g / max|g| (p - 1): below 2^14, so float16 keeps eleven
// bits of probabilities down to 2^-28 and the float32 sums have room.
constexpr float kDzScale = 16384.0f;
constexpr int64_t kPiece = 16384;  // columns of the vocabulary at a time, at least

// An operand of a product: element (r, k) at p[r ld + k] (KC) or p[k ld + r].
// k counts up to `k`, a multiple of 8; `len` elements may be read from p.
struct Opnd {
  const uint16_t* p;
  int64_t ld, len, k;
};

struct Product {
  Opnd a, b;
  int64_t M, N, K;      // rows, columns; K: a multiple of BK, 0 past an operand's k
  int64_t n0;           // first column in the vocabulary
  int64_t per;          // column tiles of a run (forward), k-steps of a split (dx)
  int64_t tiles_m, tiles_n, splits;
  const int32_t* target;
  const float *lse, *grad, *scale;  // scale: {max |grad|}
  float2* part;         // forward: {m, s} of a run of tiles, [slot][M]
  float* zt;            // forward: the target's logit
  int64_t V, slot0;
  void* out;            // dz, dw: 16 bits; dx: float32 [split][M][N]
  int64_t ldo, rows_out;
  int add;              // dx: onto what is there
};

enum { kStats, kDz, kDw, kDx };

// Workgroups whose indices agree mod 8 share an XCD and its L2: each XCD gets a
// contiguous range, walked in groups of 4 row tiles.
__device__ __forceinline__ void tile_at(int64_t bid, int64_t tiles_m, int64_t tiles_n, int64_t* tm,
                                        int64_t* tn) {
  const int64_t total = tiles_m * tiles_n, q = total / 8, r = total % 8, x = bid % 8;
  const int64_t t = x * q + (x < r ? x : r) + bid / 8;
  const int64_t group = 4 * tiles_n, first = t / group * 4;
  const int64_t size = min((int64_t)4, tiles_m - first), i = t % group;
  *tm = first + i % size;
  *tn = i / size;
}

// 32 KiB of an operand into LDS: rows r0 .. r0 + 255, k0 .. k0 + 63, the
// 1 KiB blocks of this wave.  KC: rows of 128 bytes, 16-byte chunk c of row r at
// c ^ ((r >> 1) & 7).  Else rows of one k and 256 r, chunk c of row k at
// c ^ (4 (k & 3)), for the transposing fragment reads.  Past `len` zeros arrive;
// a KC chunk past k is another of its row's (the other operand is zero there).
template <bool KC>
struct Fetch {
  const uint16_t* base;
  int64_t left;  // elements from base that may be read
  int64_t ld;
  uint32_t off[kBlocks];
  uint32_t cols[KC ? kBlocks : 1];  // KC: byte of the lane's chunk within its row

  __device__ __forceinline__ void init(const Opnd& o, int64_t r0, int64_t k0, int wave, int lane) {
    ld = o.ld;
    const int64_t at = KC ? r0 * ld + k0 : k0 * ld + r0;
    base = o.p + at;
    left = o.len - at;
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
      const int i = wave * kBlocks + q;
      if constexpr (KC) {
        const int r = 8 * i + (lane >> 3);
        off[q] = (uint32_t)(r * ld * 2);
        cols[q] = (uint32_t)(((lane & 7) ^ ((r >> 1) & 7)) * 16);
      } else {
        const int k = 2 * i + (lane >> 5);
        off[q] = (uint32_t)(k * ld * 2) + (uint32_t)(((lane & 31) ^ (4 * (k & 3))) * 16);
      }
    }
  }
  // blocks [q0, q1) of the k-step; `left_k`: k's from its first to the operand's last
  __device__ __forceinline__ void issue(uint8_t* lds, int wave, int q0, int q1, int64_t left_k) {
    const uint32_t bytes =
        left <= 0 ? 0u : (uint32_t)min(left * 2, (int64_t)0x7fffffff);
    const __amdgpu_buffer_rsrc_t r = fa_rsrc(base, bytes);
    const uint32_t lim = (uint32_t)(min(left_k, (int64_t)BK) * 2 - 16);
#pragma unroll
    for (int q = q0; q < q1; ++q) {
      const uint32_t v = KC ? off[q] + min(cols[KC ? q : 0], lim) : off[q];
      dma16_lds(r, v, 0, (lds_void*)(lds + (wave * kBlocks + q) * 1024));
    }
  }
  __device__ __forceinline__ void next() {
    const int64_t d = KC ? BK : BK * ld;
    base += d;
    left -= d;
  }
};

// Fragment i (32 rows from r0 + 32 i) of substep s (16 k): lane l gets row l % 32,
// k = 8 (l / 32) .. + 7.
template <bool KC, int F>
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
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int c = r0 + i * 32 + 16 * (g & 1) + 4 * (s16 & 3);
        off[i] = k * 512 + (((c >> 3) ^ (4 * (k & 3))) * 16) + (c & 7) * 2;
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
        const uint8_t* p = lds + off[i] + s * 16 * 512;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p);
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 4 * 512));
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

template <class Ty, bool AKC, bool BKC, int MODE>
__global__ void __launch_bounds__(kThreads, 1) xent_product_kernel(Product g) {
  // two stages of both operands; one array each, so that the compiler sees that a
  // DMA into one does not meet fragment reads of another
  __shared__ __attribute__((aligned(1024))) uint8_t A0[kHalf], B0[kHalf], A1[kHalf], B1[kHalf];
  auto block = [&](int i) -> uint8_t* {  // the stages as 32 KiB blocks of an output tile
    return i == 0 ? A0 : i == 1 ? B0 : i == 2 ? A1 : B1;
  };
  typedef typename Ty::frag frag;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  int64_t tm, tn, split = 0;
  if constexpr (MODE == kStats) {
    tile_at(blockIdx.x, g.tiles_m, g.splits, &tm, &split);
    tn = split * g.per;
  } else if constexpr (MODE == kDx) {
    const int64_t tiles = g.tiles_m * g.tiles_n;
    split = blockIdx.x / tiles;
    tile_at(blockIdx.x - split * tiles, g.tiles_m, g.tiles_n, &tm, &tn);
  } else {
    tile_at(blockIdx.x, g.tiles_m, g.tiles_n, &tm, &tn);
  }
  const int64_t m0 = tm * BM;
  int64_t k_first = 0, nk = g.K / BK;
  if constexpr (MODE == kDx) {
    k_first = split * g.per;
    nk = min(g.per, nk - k_first);
  }
  const int64_t tn_end = MODE == kStats ? min(tn + g.per, g.tiles_n) : tn + 1;

  Frags<AKC, NI> ra;
  Frags<BKC, NJ> rb;
  ra.init(wm * 128, lane);
  rb.init(wn * 64, lane);

  // rows of this lane: m0 + wm 128 + 32 i + lane % 32
  int32_t tgt[NI];
  float run_m[NI], run_s[NI];
  if constexpr (MODE == kStats || MODE == kDz) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t row = m0 + wm * 128 + i * 32 + (lane & 31);
      tgt[i] = row < g.M ? g.target[row] : -1;
      run_m[i] = -kMost;
      run_s[i] = 0.0f;
    }
  }

  for (; tn < tn_end; ++tn) {
    f32x16_t acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    Fetch<AKC> fa;
    Fetch<BKC> fb;
    fa.init(g.a, m0, k_first * BK, wave, lane);
    fb.init(g.b, tn * BN, k_first * BK, wave, lane);
    int64_t la = g.a.k - k_first * BK, lb = g.b.k - k_first * BK;
    auto issue = [&](uint8_t* sa, uint8_t* sb) {
      fa.issue(sa, wave, 0, kBlocks, la);
      fb.issue(sb, wave, 0, kBlocks, lb);
      fa.next();
      fb.next();
      la -= BK;
      lb -= BK;
    };
    auto step = [&](uint8_t* sa, uint8_t* sb, uint8_t* na, uint8_t* nb, bool more) {
      __builtin_amdgcn_s_waitcnt(0xf70);  // (vmcnt 0)
      wg_barrier();
      if (more) issue(na, nb);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        frag x[NI], y[NJ];
        ra.read(sa, s, x);
        rb.read(sb, s, y);
        // (b first: lane l then holds row l % 32 of each 32 x 32 block and the columns
        // 8 (e / 4) + 4 (l / 32) + e % 4)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = Ty::mma(y[j], x[i], acc[i][j]);
      }
    };
    if (nk > 0) issue(A0, B0);
    for (int64_t kt = 0; kt < nk; kt += 2) {
      step(A0, B0, A1, B1, kt + 1 < nk);
      if (kt + 1 < nk) step(A1, B1, A0, B0, kt + 2 < nk);
    }
    __syncthreads();

    const int64_t n_base = tn * BN + wn * 64 + (lane >> 5) * 4;
    auto col_of = [&](int j, int e) { return n_base + j * 32 + (e >> 2) * 8 + (e & 3); };

    if constexpr (MODE == kStats) {
      const bool edge = (tn + 1) * BN > g.N;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (edge)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (col_of(j, e) >= g.N) acc[i][j][e] = -INFINITY;
        // the target's logit, where it lies in these 64 columns
        const int64_t t = (int64_t)tgt[i] - g.n0;
        const int64_t d = t - (tn * BN + wn * 64);
        if (__any(d >= 0 && d < 64)) {
          const int64_t row = m0 + wm * 128 + i * 32 + (lane & 31);
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (t == col_of(j, e) && t < g.N && row < g.M) g.zt[row] = acc[i][j][e];
        }
        float m = run_m[i];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
        m = fminf(m, kMost);  // (an infinite logit: its exponential is infinite, not NaN)
        float s = run_s[i] * fa_exp2((run_m[i] - m) * kLog2e);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) s += fa_exp2((acc[i][j][e] - m) * kLog2e);
        run_m[i] = m;
        run_s[i] = s;
      }
    } else if constexpr (MODE == kDz || MODE == kDw) {
      // 16 bits through LDS, so that whole rows of 512 bytes are stored: rows 64 b ..
      // in block b, 16-byte chunk c of row r at c ^ (r & 15)
      float gain = 0.0f;
      if constexpr (MODE == kDw) gain = g.scale[0] / kDzScale;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int lr = wm * 128 + i * 32 + (lane & 31);
        uint8_t* cb = block(wm * 2 + (i >> 1)) + (lr & 63) * 512;
        float f = 0.0f, lse = 0.0f;
        bool live = false;
        int64_t t = -1;
        if constexpr (MODE == kDz) {
          const int64_t row = m0 + lr;
          live = tgt[i] >= 0 && tgt[i] < g.V;
          t = (int64_t)tgt[i] - g.n0;
          if (live) {
            f = g.grad[row] / g.scale[0] * kDzScale;
            lse = g.lse[row];
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int e = q * 4 + x;
              v[x] = acc[i][j][e];
              if constexpr (MODE == kDz) {
                const int64_t c = col_of(j, e);
                v[x] = f * (fa_exp2((v[x] - lse) * kLog2e) - (c == t ? 1.0f : 0.0f));
                if (!live || c >= g.N) v[x] = 0.0f;
              } else {
                v[x] *= gain;
              }
            }
            const int col = wn * 64 + j * 32 + q * 8 + (lane >> 5) * 4;
            *(uint2*)(cb + (((col >> 3) ^ (lr & 15)) * 16) + ((col >> 2) & 1) * 8) =
                make_uint2(Ty::pack(v[0], v[1]), Ty::pack(v[2], v[3]));
          }
      }
      __syncthreads();
      uint16_t* out = (uint16_t*)g.out;
      const int64_t rows = min((int64_t)BM, g.rows_out - m0);
      auto lds_row = [&](int r) { return block(r >> 6) + (r & 63) * 512; };
      if (MODE == kDz || g.ldo % 8 == 0) {
        const int ch = tid & 31;
        const int64_t n = tn * BN + ch * 8;
        if (MODE == kDz || n < g.N)
          for (int r = tid >> 5; r < rows; r += kThreads / 32)
            *(uint4*)(out + (m0 + r) * g.ldo + n) =
                *(const uint4*)(lds_row(r) + ((ch ^ (r & 15)) * 16));
      } else {
        const int c = tid & 255;
        const int64_t n = tn * BN + c;
        if (n < g.N)
          for (int r = tid >> 8; r < rows; r += kThreads / 256)
            out[(m0 + r) * g.ldo + n] =
                *(const uint16_t*)(lds_row(r) + (((c >> 3) ^ (r & 15)) * 16) + (c & 7) * 2);
      }
    } else {
      // float32, 128 rows at a time: 1 KiB rows, 16-byte chunk c of row r at c ^ (r & 15)
      float* out = (float*)g.out + split * g.M * g.N;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h) __syncthreads();
        if (wm == h) {
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const int lr = i * 32 + (lane & 31);
            uint8_t* cb = block(i) + (lr & 31) * 1024;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int c = (wn * 64 + j * 32 + q * 8 + (lane >> 5) * 4) >> 2;
                *(float4*)(cb + ((c ^ (lr & 15)) * 16)) =
                    make_float4(acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2],
                                acc[i][j][q * 4 + 3]);
              }
          }
        }
        __syncthreads();
        const int64_t r0 = m0 + h * 128;
        const int rows = (int)min((int64_t)128, g.M - r0);
        for (int r = tid >> 6; r < rows; r += kThreads / 64) {
          const float4 v =
              *(const float4*)(block(r >> 5) + (r & 31) * 1024 + ((lane ^ (r & 15)) * 16));
          const int64_t n = tn * BN + lane * 4;
          float* o = out + (r0 + r) * g.N + n;
          const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (n + x < g.N) o[x] = g.add ? o[x] + f[x] : f[x];
        }
      }
    }
  }

  if constexpr (MODE == kStats) {
    // both lanes of a row, then the four waves of its columns
    float2* tmp = (float2*)A0;  // [4][BM]
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float om = __shfl_xor(run_m[i], 32), os = __shfl_xor(run_s[i], 32);
      const float m = fmaxf(run_m[i], om);
      const float s = run_s[i] * fa_exp2((run_m[i] - m) * kLog2e) +
                      os * fa_exp2((om - m) * kLog2e);
      if (lane < 32) tmp[wn * BM + wm * 128 + i * 32 + lane] = make_float2(m, s);
    }
    __syncthreads();
    if (tid < BM && m0 + tid < g.M) {
      float m = tmp[tid].x, s = 0.0f;
#pragma unroll
      for (int w = 1; w < 4; ++w) m = fmaxf(m, tmp[w * BM + tid].x);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        s += tmp[w * BM + tid].y * fa_exp2((tmp[w * BM + tid].x - m) * kLog2e);
      g.part[(g.slot0 + split) * g.M + m0 + tid] = make_float2(m, s);
    }
  }
}

// lse and loss of every row from its `slots` partial results.
__global__ void __launch_bounds__(256) xent_join_kernel(XentArgs a, const float2* part,
                                                        const float* zt, int64_t slots) {
  __shared__ float2 tmp[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 64 + lane;
  float m = -kMost, s = 0.0f;
  auto put = [&](float2 p) {
    const float n = fmaxf(m, p.x);
    s = s * expf(m - n) + p.y * expf(p.x - n);
    m = n;
  };
  if (row < a.T)
    for (int64_t i = wave; i < slots; i += 4) put(part[i * a.T + row]);
  tmp[wave][lane] = make_float2(m, s);
  __syncthreads();
  if (wave || row >= a.T) return;
  for (int w = 1; w < 4; ++w) put(tmp[w][lane]);
  const float lse = m + logf(s);
  const int32_t t = a.target[row];
  a.loss[row] = t >= 0 && t < a.V ? lse - zt[row] : 0.0f;
  if (a.lse) a.lse[row] = lse;
}

// Block 0: the largest finite |grad| of a row with a target (1 if there is none
// above 0).  The others: x with zeros in rows without a target, in rows behind T
// and columns behind H.
__global__ void __launch_bounds__(1024) xent_prepare_kernel(const uint16_t* x,
                                                            const int32_t* target,
                                                            const float* grad, int64_t T,
                                                            int64_t H, int64_t V, int64_t Tp,
                                                            int64_t Hp, uint16_t* out,
                                                            float* scale) {
  if (grad && blockIdx.x == 0) {
    __shared__ float tmp[16];
    float m = 0.0f;
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
      const float f = fabsf(grad[t]);
      if (target[t] >= 0 && target[t] < V && f < INFINITY) m = fmaxf(m, f);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 16; ++i) m = fmaxf(m, tmp[i]);
      scale[0] = m > 0.0f ? m : 1.0f;
    }
    return;
  }
  const int64_t first = grad ? 1 : 0;
  const int64_t per = Hp / 8, total = Tp * per;
  for (int64_t i = (blockIdx.x - first) * 1024 + threadIdx.x; i < total;
       i += (gridDim.x - first) * 1024) {
    const int64_t r = i / per, c = (i - r * per) * 8;
    // (without gradients every row is taken as it is)
    const bool live = r < T && (!grad || (target[r] >= 0 && target[r] < V));
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live) {
      if (H % 8 == 0) {
        if (c < H) v = *(const uint4*)(x + r * H + c);
      } else {
        uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = c + e < H ? x[r * H + c + e] : (uint16_t)0;
        __builtin_memcpy(&v, h, 16);
      }
    }
    *(uint4*)(out + r * Hp + c) = v;
  }
}

// A [rows, cols] window of w (row pitch ld) as [rows, pitch] with zeros behind cols.
__global__ void __launch_bounds__(256) xent_pack_kernel(const uint16_t* w, int64_t ld,
                                                        int64_t rows, int64_t cols, int64_t pitch,
                                                        uint16_t* out) {
  const int64_t per = pitch / 8, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = (i - r * per) * 8;
    uint16_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = c + e < cols ? w[r * ld + c + e] : (uint16_t)0;
    uint4 v;
    __builtin_memcpy(&v, h, 16);
    *(uint4*)(out + r * pitch + c) = v;
  }
}

// dx from its splits' sums; rows without a target zero.
template <class Ty>
__global__ void __launch_bounds__(256) xent_dx_kernel(XentGradArgs a, const float* sums,
                                                      int64_t splits, const float* scale) {
  const int64_t total = a.T * a.H;
  const float gain = scale[0] / kDzScale;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int32_t t = a.target[i / a.H];
    float s = 0.0f;
    if (t >= 0 && t < a.V) {
      for (int64_t p = 0; p < splits; ++p) s += sums[p * total + i];
      s *= gain;
    }
    ((uint16_t*)a.dx)[i] = (uint16_t)Ty::pack(s, 0.0f);
  }
}

// ---- plans (sizes alone) --------------------------------------------------------------

constexpr int64_t kCus = 256;
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t cdiv(int64_t n, int64_t m) { return (n + m - 1) / m; }

// How many ways to split `n` steps of each of `tiles` tiles, so that the CUs, one
// workgroup each, finish soonest; `most`: at most so many.  A split costs `extra`
// steps of its own.
int64_t choose_splits(int64_t tiles, int64_t n, int64_t most, double extra) {
  int64_t best = 1;
  double least = 1e300;
  for (int64_t s = 1; s <= std::min(n, most); ++s) {
    const double cost = (double)cdiv(tiles * s, kCus) * ((double)cdiv(n, s) + extra);
    if (cost < least * 0.999) {
      least = cost;
      best = s;
    }
  }
  return cdiv(n, cdiv(n, best));  // (none of them empty)
}

struct XentPlan {
  bool pack_w, copy_x;     // w's pitch is no multiple of 8; x's no multiple of 64
  int64_t Hp, Tp;          // H and T padded
  int64_t piece, pieces;   // columns of the vocabulary at a time
  int64_t splits, per;     // forward: runs of tiles per piece; gradient: splits of dx
  // offsets of the working memory
  size_t part, zt, x, w, dz, sums, scale, bytes;
};

XentPlan make_plan(int64_t T, int64_t H, int64_t V, int tied, bool grad) {
  XentPlan p;
  p.pack_w = (tied ? H : V) % 8 != 0;
  p.copy_x = grad || H % BK != 0;
  p.Hp = up(H, BK);
  p.Tp = up(T, BK);
  p.piece = V;
  if (grad) p.piece = std::max(kPiece, (int64_t)(1 << 25) / std::max<int64_t>(T, 1));
  else if (p.pack_w) p.piece = kPiece;
  p.piece = std::min(up(p.piece, BN), up(V, BN));
  p.pieces = cdiv(V, p.piece);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
  };
  const int64_t tiles_m = cdiv(T, BM);
  if (grad) {
    const int64_t nk = p.piece / BK;
    p.splits = choose_splits(tiles_m * cdiv(H, BN), nk, 16, 24.0);
    p.per = cdiv(nk, p.splits);
    p.part = p.zt = 0;
    p.dz = take((size_t)p.Tp * p.piece * 2);
    p.sums = take((size_t)p.splits * T * H * 4);
    p.scale = take(4);
  } else {
    const int64_t tiles = p.piece / BN;
    p.splits = choose_splits(tiles_m, tiles, 256, 0.1);
    p.per = cdiv(tiles, p.splits);
    p.part = take((size_t)p.pieces * p.splits * T * sizeof(float2));
    p.zt = take((size_t)T * 4);
    p.dz = p.sums = p.scale = 0;
  }
  p.x = p.copy_x ? take((size_t)p.Tp * p.Hp * 2) : 0;
  p.w = p.pack_w ? take((size_t)(tied ? p.piece * p.Hp : H * p.piece) * 2) : 0;
  p.bytes = at;
  return p;
}

template <class Ty, bool AKC, bool BKC, int MODE>
void launch_product(const Product& g, hipStream_t stream) {
  const int64_t blocks =
      MODE == kStats ? g.tiles_m * g.splits
                     : MODE == kDx ? g.tiles_m * g.tiles_n * g.splits : g.tiles_m * g.tiles_n;
  if (blocks == 0) return;
  hipLaunchKernelGGL((xent_product_kernel<Ty, AKC, BKC, MODE>), dim3((unsigned)blocks),
                     dim3(kThreads), 0, stream, g);
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
    const int64_t blocks = std::min<int64_t>(cdiv(p.Tp * p.Hp / 8, 1024), kCus * 4);
    hipLaunchKernelGGL(xent_prepare_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream,
                       (const uint16_t*)a.x, a.target, (const float*)nullptr, a.T, a.H, a.V, p.Tp,
                       p.Hp, x, (float*)nullptr);
    REW_HIP(hipGetLastError());
    ++launches;
    g.a = {x, p.Hp, p.Tp * p.Hp, p.Hp};
  }
  g.M = a.T;
  g.K = p.Hp;
  g.V = a.V;
  g.target = a.target;
  g.part = (float2*)(work + p.part);
  g.zt = (float*)(work + p.zt);
  g.tiles_m = cdiv(a.T, BM);
  g.per = p.per;
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(p.piece, a.V - v0);
    const Piece w = piece_of(a, p, v0, n, work, stream, &launches);
    g.n0 = v0;
    g.N = n;
    g.tiles_n = cdiv(n, BN);
    g.splits = cdiv(g.tiles_n, p.per);
    if (a.tied) {
      g.b = {w.p, w.ld, w.len, p.pack_w ? p.Hp : a.H};
      launch_product<Ty, true, true, kStats>(g, stream);
    } else {
      g.b = {w.p, w.ld, w.len, a.H};
      launch_product<Ty, true, false, kStats>(g, stream);
    }
    ++launches;
    g.slot0 += g.splits;
  }
  hipLaunchKernelGGL(xent_join_kernel, dim3((unsigned)cdiv(a.T, 64)), dim3(256), 0, stream, a,
                     g.part, g.zt, g.slot0);
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
  float* sums = (float*)(work + p.sums);
  float* scale = (float*)(work + p.scale);
  const int64_t blocks = 1 + std::min<int64_t>(cdiv(p.Tp * p.Hp / 8, 1024), kCus * 4);
  hipLaunchKernelGGL(xent_prepare_kernel, dim3((unsigned)blocks), dim3(1024), 0, stream,
                     (const uint16_t*)a.x, a.target, a.grad, a.T, a.H, a.V, p.Tp, p.Hp, x, scale);
  REW_HIP(hipGetLastError());
  ++launches;
  int64_t splits = 0;
  const Opnd xk = {x, p.Hp, p.Tp * p.Hp, p.Hp};   // k = embed
  const Opnd xt = {x, p.Hp, p.Tp * p.Hp, p.Tp};   // k = tokens
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(p.piece, a.V - v0);
    const Piece w = piece_of(a, p, v0, n, work, stream, &launches);
    const int64_t np = up(n, BN);  // columns of dz, zeros behind n
    Product g;
    std::memset(&g, 0, sizeof g);
    // dz
    g.a = xk;
    g.b = {w.p, w.ld, w.len, a.tied && p.pack_w ? p.Hp : a.H};
    g.M = a.T;
    g.N = n;
    g.K = p.Hp;
    g.n0 = v0;
    g.V = a.V;
    g.target = a.target;
    g.lse = a.lse;
    g.grad = a.grad;
    g.scale = scale;
    g.tiles_m = cdiv(a.T, BM);
    g.tiles_n = np / BN;
    g.out = dz;
    g.ldo = p.piece;
    g.rows_out = p.Tp;
    if (a.T) {
      if (a.tied) launch_product<Ty, true, true, kDz>(g, stream);
      else launch_product<Ty, true, false, kDz>(g, stream);
      ++launches;
    }
    // dw
    const Opnd dzt = {dz, p.piece, p.Tp * p.piece, p.Tp};
    g.a = a.tied ? dzt : xt;
    g.b = a.tied ? xt : dzt;
    g.M = g.rows_out = a.tied ? n : a.H;
    g.N = a.tied ? a.H : n;
    g.K = p.Tp;
    g.tiles_m = cdiv(g.M, BM);
    g.tiles_n = cdiv(g.N, BN);
    g.out = (uint16_t*)a.dw + (a.tied ? v0 * a.H : v0);
    g.ldo = a.tied ? a.H : a.V;
    launch_product<Ty, false, false, kDw>(g, stream);
    ++launches;
    // dx
    if (!a.T) continue;
    g.a = {dz, p.piece, p.Tp * p.piece, np};
    // (a packed piece has zeros behind n; else the rows' or columns' end is w's own)
    g.b = {w.p, w.ld, w.len, a.tied ? n : p.pack_w ? np : up(n, 8)};
    g.M = a.T;
    g.N = a.H;
    g.K = up(n, BK);
    g.tiles_m = cdiv(g.M, BM);
    g.tiles_n = cdiv(g.N, BN);
    g.out = sums;
    g.per = p.per;
    g.splits = cdiv(g.K / BK, p.per);
    if (i == 0) splits = g.splits;  // (of all pieces the most)
    g.add = i > 0;
    if (a.tied) launch_product<Ty, true, false, kDx>(g, stream);
    else launch_product<Ty, true, true, kDx>(g, stream);
    ++launches;
  }
  if (a.T) {
    const int64_t nb = std::min<int64_t>(cdiv(a.T * a.H, 256), kCus * 16);
    hipLaunchKernelGGL((xent_dx_kernel<Ty>), dim3((unsigned)nb), dim3(256), 0, stream, a, sums,
                       splits, scale);
    REW_HIP(hipGetLastError());
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
