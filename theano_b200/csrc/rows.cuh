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

// Two float32 in a 64-bit register: the packed operations take one issue slot for two results.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Two neighbouring elements of a 16-bit type in a word.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int BYTES> struct Words;
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };

// V elements as they lie in memory, loaded at once: a load that is issued early costs registers of the tensor's type.
template <typename T, int V> struct Pack {
  using W = typename Words<V * sizeof(T)>::type;
  union { W w; T e[V]; uint32_t u[V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1]; };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const { return to_float(e[i]); }
  __device__ __forceinline__ void set(int i, float v) { e[i] = from_float<T>(v); }
  // elements 2 i and 2 i + 1 (V > 1)
  __device__ __forceinline__ Pair get2(int i) const {
    if constexpr (sizeof(T) == 4) {
      return Pair(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    } else {
      const float2 f = unpack2<T>(u[i]);
      return Pair(f.x, f.y);
    }
  }
  __device__ __forceinline__ void set2(int i, Pair v) {
    const float2 f = v.get();
    if constexpr (sizeof(T) == 4) {
      u[2 * i] = __float_as_uint(f.x);
      u[2 * i + 1] = __float_as_uint(f.y);
    } else {
      u[i] = pack2<T>(f.x, f.y);
    }
  }
};

// The same for any V: with one element the pair's second half is `fill`, and nothing on the way back.
template <int V> constexpr int kPairs = V > 1 ? V / 2 : 1;
template <typename T, int V> __device__ __forceinline__ Pair pair_of(const Pack<T, V>& k, int i, float fill) {
  if constexpr (V > 1) return k.get2(i);
  else return Pair(k.get(0), fill);
}
template <typename T, int V> __device__ __forceinline__ void put_pair(Pack<T, V>& k, int i, Pair v) {
  if constexpr (V > 1) k.set2(i, v);
  else k.set(0, v.get().x);
}

template <typename T, int V> __device__ __forceinline__ void load_row(const T* p, float (&f)[V]) {
  Pack<T, V> k;
  k.load(p);
  if constexpr (V > 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 v = k.get2(i).get();
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
    f[0] = k.get(0);
  }
}
template <typename T, int V> __device__ __forceinline__ void store_row(T* p, const float (&f)[V]) {
  Pack<T, V> k;
  if constexpr (V > 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) k.set2(i, Pair(f[2 * i], f[2 * i + 1]));
  } else {
    k.set(0, f[0]);
  }
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
// The last sequence that starts at or before `row`; -1 before the first.  All lanes of the warp ask for the same row: 32 offsets at a
// time, one trip to memory for up to 32 sequences, two for 1024.
__device__ __forceinline__ int sequence_of(const int* starts, int count, long long row, long long rows) {
  int lo = 0, n = count;                         // the sequences before lo start at or before the row, [lo, lo + n) are undecided
  while (n > 0) {
    const int step = (n + 31) >> 5, i = (threadIdx.x & 31) * step;
    const int m = __popc(__ballot_sync(~0u, i < n && start_of(starts, lo + (i < n ? i : 0), rows) <= row));
    if (m == 0) break;
    const int end = m * step < n ? m * step : n;
    n = end - (m - 1) * step - 1;
    lo += (m - 1) * step + 1;
  }
  return lo - 1;
}

// 2^v, off by 2^-22 of the result; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// 1 / (1 + e^-v): zero where e^-v overflows
__device__ __forceinline__ float sigmoid(float v) { return reciprocal_fast(1.f + exp2_fast(-v * kLog2e)); }

}  // namespace b200
