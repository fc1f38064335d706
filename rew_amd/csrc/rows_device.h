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

// N values side by side, loaded and stored as one access (N * the element's
// size is 16 bytes or less, a power of two, and the address a multiple of it).
template <class T, int N>
struct alignas(sizeof(typename T::elem) * N) RowRun {
  typename T::elem v[N];
};

template <class T, int N>
__device__ __forceinline__ void run_load(const void* base, int64_t i, float (&f)[N]) {
  const RowRun<T, N> r = *(const RowRun<T, N>*)((const typename T::elem*)base + i);
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

}  // namespace rew
