// The key tiles of a step's paged attention as one line, cut into equal runs.
//
// Requests differ in length by orders of magnitude and only the device knows
// them, so the work is cut by key tiles: an item is a row block of one KV head
// of one request, its tiles are the key tiles that its last row sees, and worker
// w of a launch takes the w-th of equal runs of all items' tiles.  An item that
// lies inside one run is finished by its worker; of one that is cut, each
// worker leaves its maximum, sum and unnormalised output in float32, at most
// two per worker, and a second launch joins them in order.  A worker finds its
// run by summing the requests' tile counts, 64 requests a step, one per lane.
#pragma once

#include "attn_device.h"
#include "kernels.h"

namespace rew {

// A request's rows and keys, as the kernels of a step see them.
struct Request {
  int first, n, rows, len, cap;  // cap: keys that can have a page
  __device__ __forceinline__ int limit(const PackedArgs& a, int G, int row) const {
    const int t = min(row, rows - 1) / G;
    return min(max(a.causal ? len - n + t + 1 : len, 0), cap);
  }
};
// s: -1 .. n_seq (the rows of no request, as in SeqTile); its n rows from `first`
__device__ __forceinline__ Request request_of(const PackedArgs& a, int G, int s, int first, int n) {
  Request r;
  r.first = first;
  r.n = n;
  r.rows = n * G;
  const bool real = s >= 0 && s < a.n_seq;
  r.len = real ? max(a.lens[s], 0) : 0;
  r.cap = real ? (int)min((int64_t)r.len, (int64_t)a.width << a.log_page) : 0;
  return r;
}
// The 64 requests from `base`, one per lane (floor: SeqRows).
__device__ __forceinline__ Request lane_request(const PackedArgs& a, int G, int base, int& floor) {
  const SeqRows x(a.starts, a.n_seq, (int)a.T, base, floor);
  return request_of(a, G, x.s, x.first, x.n);
}
// Lane `at`'s request, in every lane.
__device__ __forceinline__ Request request_from(const Request& x, int at) {
  Request r;
  r.first = __builtin_amdgcn_readlane(x.first, at);
  r.n = __builtin_amdgcn_readlane(x.n, at);
  r.rows = __builtin_amdgcn_readlane(x.rows, at);
  r.len = __builtin_amdgcn_readlane(x.len, at);
  r.cap = __builtin_amdgcn_readlane(x.cap, at);
  return r;
}

// The line for row blocks of ROWS rows and tiles of BK keys.  Each item has at
// least one tile, so that rows without keys are written too.
template <int ROWS, int BK>
struct TileLine {
  const PackedArgs& a;
  int G;
  static constexpr int kRows = ROWS;
  __device__ __forceinline__ int item_tiles(const Request& r, int qt) const {
    return max((r.limit(a, G, qt * ROWS + ROWS - 1) + BK - 1) / BK, 1);
  }
  // tiles of one KV head of a request
  __device__ __forceinline__ int head_tiles(const Request& r) const {
    int t = 0;
    for (int qt = 0; qt * ROWS < r.rows; ++qt) t += item_tiles(r, qt);
    return t;
  }
};
// 64 requests of the line, one per lane: their tiles and the running sum.
struct LineStep {
  Request r;
  int x, sum;
  template <class Line>
  __device__ __forceinline__ LineStep(const Line& L, int base, int& floor)
      : r(lane_request(L.a, L.G, base, floor)), x(L.head_tiles(r) * L.a.Hkv), sum(wave_scan(x)) {}
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(sum, 63); }
};
// Where a tile of the line lies.
template <class Line>
struct TilePlace {
  int s, hk, qt, kt;
  Request r;
  // (the line's total < 2^31 was checked on the host; step, floor: the first 64
  // requests, which the total needed already)
  __device__ __forceinline__ void find(const Line& L, int t, LineStep step, int floor) {
    int base = -1;
    for (;;) {
      if (t < step.total() || base + 64 > L.a.n_seq) break;
      t -= step.total();
      base += 64;
      step = LineStep(L, base, floor);
    }
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(step.sum > t));
    t -= __builtin_amdgcn_readlane(step.sum - step.x, at);
    s = base + at;
    r = request_from(step.r, at);
    const int head = __builtin_amdgcn_readlane(step.x, at) / L.a.Hkv;
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
  __device__ __forceinline__ void next(const Line& L) {
    kt = 0;
    if ((qt + 1) * Line::kRows < r.rows) {
      ++qt;
      return;
    }
    qt = 0;
    if (++hk < L.a.Hkv) return;
    hk = 0;
    do {
      ++s;
      const int first = r.first + r.n;
      const int end = max(seq_bound(L.a.starts, L.a.n_seq, (int)L.a.T, s + 1), first);
      r = request_of(L.a, L.G, s, first, end - first);
    } while (s <= L.a.n_seq && L.head_tiles(r) == 0);
  }
};
// The cut of the line into runs, as even as whole tiles allow and of at least
// `least` tiles; run w is [start(w), start(w + 1)).
struct Runs {
  int floor = 0;  // behind the first 64 requests, `step`, for TilePlace::find
  LineStep step;
  int total, count, each, more;
  template <class Line>
  __device__ __forceinline__ Runs(const Line& L, int most, int least) : step(L, -1, floor) {
    total = step.total();
    int at = floor;
    for (int base = 63; base <= L.a.n_seq; base += 64) total += LineStep(L, base, at).total();
    count = min(most, max((total + least - 1) / least, 1));
    each = total / count;
    more = total - each * count;
  }
  __device__ __forceinline__ int start(int w) const {
    return w >= count ? total : each * w + min(w, more);
  }
};

// Floats of a partial result: O [rows][D], then (max, sum) per row; worker w's
// are at 2 w (of an item that an earlier run began) and 2 w + 1 (of one that
// begins in its run).
constexpr int part_floats(int rows, int D) { return rows * D + 2 * rows; }

// Stores what lane (c, g) holds of its row: the result at `out`, or row `row`
// of a partial result.
template <class M, int D>
__device__ __forceinline__ void store_whole(uint16_t* out, const f32x16_t (&o)[D / 32], float l,
                                            int g) {
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays NaN)
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(uint2*)(out + dt * 32 + i * 8 + g * 4) =
          make_uint2(M::pack(o[dt][i * 4] * inv, o[dt][i * 4 + 1] * inv),
                     M::pack(o[dt][i * 4 + 2] * inv, o[dt][i * 4 + 3] * inv));
}
template <int D>
__device__ __forceinline__ void store_part(float* part, int rows, int row,
                                           const f32x16_t (&o)[D / 32], float m, float l, int g) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(float4*)(part + row * D + dt * 32 + i * 8 + g * 4) =
          make_float4(o[dt][i * 4], o[dt][i * 4 + 1], o[dt][i * 4 + 2], o[dt][i * 4 + 3]);
  if (g == 0) *(float2*)(part + rows * D + 2 * row) = make_float2(m, l);
}

// Joins rows [0, rows) of an item from the n partial results piece(0 .. n - 1)
// (of ROWS rows) into the result rows out(i): of a workgroup of 256 threads D / 4
// lanes take a row, workgroup y every gridDim.y-th 1024 / D rows, eight pieces in
// flight.
template <class M, int D, int ROWS, class Piece, class Out>
__device__ __forceinline__ void join_rows(int rows, int n, Piece piece, Out out) {
  constexpr int L = D / 4, B = 8;
  const int d = (threadIdx.x % L) * 4;
  for (int i = blockIdx.y * (256 / L) + threadIdx.x / L; i < rows; i += gridDim.y * (256 / L)) {
    float m = -INFINITY, l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < n; k0 += B) {
      float2 ml[B];
      float4 o[B];
#pragma unroll
      for (int j = 0; j < B; ++j) {  // (past the last: the last again, weighing nothing)
        const float* p = piece(min(k0 + j, n - 1));
        ml[j] = *(const float2*)(p + ROWS * D + 2 * i);
        o[j] = *(const float4*)(p + i * D + d);
      }
      float mb = m;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        if (k0 + j >= n) ml[j] = make_float2(-INFINITY, 0.0f);
        mb = fmaxf(mb, ml[j].x);
      }
      const float mu = mb == -INFINITY ? 0.0f : mb, s0 = fa_exp2(m - mu);
      l *= s0;
#pragma unroll
      for (int v = 0; v < 4; ++v) x[v] *= s0;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        if (k0 + j >= n) continue;
        const float s = fa_exp2(ml[j].x - mu);
        l = fmaf(ml[j].y, s, l);
        x[0] = fmaf(o[j].x, s, x[0]);
        x[1] = fmaf(o[j].y, s, x[1]);
        x[2] = fmaf(o[j].z, s, x[2]);
        x[3] = fmaf(o[j].w, s, x[3]);
      }
      m = mb;
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    *(uint2*)(out(i) + d) =
        make_uint2(M::pack(x[0] * inv, x[1] * inv), M::pack(x[2] * inv, x[3] * inv));
  }
}

}  // namespace rew
