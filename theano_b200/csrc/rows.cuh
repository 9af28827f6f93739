// Rows of channels in device memory: loads and stores of the sequence operators (layer_norm.cu, causal_conv.cu,
// selective_scan.cu, selective_scan_grad.cu) in float32, float16 and bfloat16, computing in float32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sequence.h"

namespace b200 {

template <typename T> __device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// One rounding, to the nearest even value of the type.
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES> struct Words;
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };

// V elements as they lie in memory, loaded at once: a load that is issued early costs registers of the tensor's type.
template <typename T, int V> struct Pack {
  using W = typename Words<V * sizeof(T)>::type;
  union { W w; T e[V]; };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const { return to_float(e[i]); }
  __device__ __forceinline__ void set(int i, float v) { e[i] = from_float<T>(v); }
};

template <typename T, int V> __device__ __forceinline__ void load_row(const T* p, float (&f)[V]) {
  Pack<T, V> k;
  k.load(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = k.get(i);
}
template <typename T, int V> __device__ __forceinline__ void store_row(T* p, const float (&f)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.set(i, f[i]);
  k.store(p);
}

// Parameters (weights, biases) are of the tensors' type or float32.
template <typename T> __device__ __forceinline__ float param(const void* p, long long i, int f32) {
  return f32 ? static_cast<const float*>(p)[i] : to_float(static_cast<const T*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void set_param(void* p, long long i, int f32, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_float<T>(v);
}

// V of them that lie on a boundary of V elements.
template <typename P, int V> __device__ __forceinline__ void load_params(const void* p, long long i, float (&f)[V]) {
  constexpr int kStep = V * sizeof(P) > 16 ? 16 / sizeof(P) : V;
#pragma unroll
  for (int k = 0; k < V; k += kStep) {
    Pack<P, kStep> v;
    v.load(static_cast<const P*>(p) + i + k);
#pragma unroll
    for (int q = 0; q < kStep; ++q) f[k + q] = v.get(q);
  }
}

// First row of sequence i of a packed tensor, kept inside of the tensor whatever the caller's offsets say.
__device__ __forceinline__ long long start_of(const int* starts, int i, long long rows) {
  const long long s = starts[i];
  return s < 0 ? 0 : s > rows ? rows : s;
}
// The last sequence that starts at or before `row`; -1 before the first.
__device__ __forceinline__ int sequence_of(const int* starts, int count, long long row, long long rows) {
  int lo = 0, hi = count;                        // sequences [lo, hi) are undecided
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (start_of(starts, mid, rows) <= row) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + __expf(-v)); }

}  // namespace b200
