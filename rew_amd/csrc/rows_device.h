// Element types of the row kernels (embeddings, layer norm): runs of values
// loaded as float32 and stored rounded once.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rew {

struct RowF32 {
  typedef float elem;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
struct RowBf16 {
  typedef __bf16 elem;
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};
struct RowF16 {
  typedef _Float16 elem;
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};

// Rows are walked in runs of N values: 16 bytes, or single values in rows of fewer.
// The run that would reach past a row's end, and any behind it, lies on the row's
// last N values instead: no access is under a condition (at whose end the compiler
// would wait for every load under way), and values that two runs hold are computed
// and stored twice, the same.  Sums over a row leave out what an earlier run holds.
template <class T>
constexpr int kRun = 16 / (int)sizeof(typename T::elem);

__device__ __forceinline__ int64_t run_start(int64_t i, int64_t n, int N) {
  return i < n - N ? i : n - N;
}

// (The address need not be a multiple of 16 in rows of an odd number of values: the
// access is one instruction all the same, since those of a wave may be unaligned.)
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(typename T::elem)))) RowRun {
  typename T::elem v[N];
};

template <class T, int N>
__device__ __forceinline__ RowRun<T, N> run_at(const void* base, int64_t i) {
  return *(const RowRun<T, N>*)((const typename T::elem*)base + i);
}

template <class T, int N>
__device__ __forceinline__ void run_load(const void* base, int64_t i, float (&f)[N]) {
  const RowRun<T, N> r = run_at<T, N>(base, i);
#pragma unroll
  for (int x = 0; x < N; ++x) f[x] = T::get(r.v[x]);
}

template <class T, int N>
__device__ __forceinline__ void run_store(void* base, int64_t i, const float (&f)[N]) {
  RowRun<T, N> r;
#pragma unroll
  for (int x = 0; x < N; ++x) r.v[x] = T::put(f[x]);
  *(RowRun<T, N>*)((typename T::elem*)base + i) = r;
}

// Workgroups 0 .. n - 1 (and up to 2^16 - 1 more) in rows of 2^16: the x of a launch takes
// fewer than 2^32 threads.
inline dim3 grid_of(int64_t n) {
  const int64_t x = n < 1 << 16 ? (n > 0 ? n : 1) : 1 << 16;
  return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}
__device__ __forceinline__ int64_t block_of() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

}  // namespace rew
