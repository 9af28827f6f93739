// What the passes of the short causal convolution share: where a run of tokens lies, the window before a token, launch shapes.
#pragma once
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "rows.cuh"

namespace b200 {

__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }

// A block is 2^log_lanes (32 or 64) channel pieces x threads >> log_lanes runs; `channel_blocks` blocks side by side span the channels.
struct CausalGrid {
  int threads, log_lanes, channel_blocks;
  int run;                                       // tokens of a run
  int runs;                                      // runs of a sequence (packed: of the tensor)
  unsigned run_blocks;
};
// Runs as long as lets all blocks be resident at once (`slots` of them), `least` tokens at least: a few blocks more than fit would be a
// second round, and every run costs its filters and the tokens before it.
inline CausalGrid causal_grid(const CausalArgs& a, int V, int threads, long long slots, int least) {
  CausalGrid g = {};
  const long long vecs = a.d.C / V, sequences = a.d.packed ? 1 : a.d.sequences;
  g.threads = threads;
  g.log_lanes = 5;                               // a warp works on one run
  while (g.log_lanes < 6 && (1LL << g.log_lanes) < vecs) ++g.log_lanes;
  g.channel_blocks = static_cast<int>((vecs + (1LL << g.log_lanes) - 1) >> g.log_lanes);
  const long long per = threads >> g.log_lanes, at_once = std::max<long long>(1, slots / g.channel_blocks * per / std::max<long long>(1, sequences));
  g.run = static_cast<int>(std::max<long long>((a.d.length + at_once - 1) / at_once, least));
  g.runs = static_cast<int>((a.d.length + g.run - 1) / g.run);
  g.run_blocks = static_cast<unsigned>((sequences * g.runs + per - 1) / per * g.channel_blocks);
  return g;
}

struct RunPlace { long long seq, from, to; };    // tokens [from, to) of sequence seq (packed: rows of the tensor, seq 0)
__device__ __forceinline__ RunPlace place_run(const CausalArgs& a, const CausalGrid& g, long long run) {
  RunPlace p;
  p.seq = a.d.packed ? 0 : static_cast<uint32_t>(run) / static_cast<uint32_t>(g.runs);
  p.from = (run - p.seq * g.runs) * g.run;
  p.to = p.from + g.run < a.d.length ? p.from + g.run : a.d.length;
  if (p.seq >= a.d.sequences || p.from >= a.d.length) p.from = p.to = 0;
  return p;
}

// The sequence that a token belongs to, and the first token of the run that belongs to any.
struct Place { int seq; long long begin, end, token; };
// From sequence `seq` on, past empty ones and rows in front of the first.
__device__ __forceinline__ Place place_from(const CausalArgs& a, int seq, long long t) {
  Place at;
  const int n = static_cast<int>(a.d.sequences);
  at.seq = seq < 0 ? 0 : seq;
  at.begin = at.end = at.token = a.d.length;
  for (; at.seq < n; ++at.seq) {
    at.begin = start_of(a.starts, at.seq, a.d.length);
    at.end = start_of(a.starts, at.seq + 1, a.d.length);
    const long long first = at.begin > t ? at.begin : t;
    if (first < at.end) { at.token = first; break; }
  }
  return at;
}
// The place of a run's first token (all lanes of a warp call this, for the same run).
__device__ __forceinline__ Place place_run_start(const CausalArgs& a, const RunPlace& p) {
  if (a.d.packed) return place_from(a, sequence_of(a.starts, static_cast<int>(a.d.sequences), p.from, a.d.length), p.from);
  Place at;
  at.seq = static_cast<int>(p.seq);
  at.begin = 0; at.end = a.d.length; at.token = p.from;
  return at;
}
// Token t lies behind at's sequence: the one that it belongs to.  False where no later row belongs to any.
__device__ __forceinline__ bool next_sequence(const CausalArgs& a, long long t, Place* at) {
  if (!a.d.packed) return false;
  *at = place_from(a, at->seq + 1, t);
  return at->token == t;
}

// Coefficients by distance: w[k] meets the token k steps back.
template <typename T, int V, int K>
__device__ __forceinline__ void load_filter(const CausalArgs& a, int c, float (&w)[K][V], float (&bias)[V]) {
  float flat[K * V];
  if (V == 1) {
#pragma unroll
    for (int i = 0; i < K; ++i) flat[i] = param<T>(a.w, 1LL * c * K + i, a.d.param_f32);
    bias[0] = a.bias ? param<T>(a.bias, c, a.d.param_f32) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float part[V];
      if (a.d.param_f32 || sizeof(T) == 4) load_params<float, V>(a.w, 1LL * c * K + i * V, part);
      else load_params<T, V>(a.w, 1LL * c * K + i * V, part);
#pragma unroll
      for (int q = 0; q < V; ++q) flat[i * V + q] = part[q];
    }
#pragma unroll
    for (int q = 0; q < V; ++q) bias[q] = 0.f;
    if (a.bias) {
      if (a.d.param_f32 || sizeof(T) == 4) load_params<float, V>(a.bias, c, bias);
      else load_params<T, V>(a.bias, c, bias);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int q = 0; q < V; ++q) w[k][q] = a.d.flip ? flat[q * K + k] : flat[q * K + K - 1 - k];
}

// Coefficients and bias in pairs of channels.
template <typename T, int V, int K>
__device__ __forceinline__ void load_filter(const CausalArgs& a, int c, Pair (&w)[K][kPairs<V>], Pair (&bias)[kPairs<V>]) {
  constexpr int kNext = V > 1 ? 1 : 0;
  float fw[K][V], fb[V];
  load_filter<T, V, K>(a, c, fw, fb);
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    bias[i] = Pair(fb[2 * i], fb[2 * i + kNext]);
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = Pair(fw[k][2 * i], fw[k][2 * i + kNext]);
  }
}

// v sigmoid(v) of both
__device__ __forceinline__ Pair silu2(Pair v) {
  const float2 e = mul2(v, Pair(-kLog2e, -kLog2e)).get();
  const float2 d = add2(Pair(exp2_fast(e.x), exp2_fast(e.y)), Pair(1.f, 1.f)).get();
  return mul2(v, Pair(reciprocal_fast(d.x), reciprocal_fast(d.y)));
}

// The taps - 1 rows before token t of at's sequence, oldest first: tokens, rows of the initial state, zeros.
template <typename T, int V, int K>
__device__ __forceinline__ void load_window(const CausalArgs& a, const T* x, const Place& at, long long t, int c, float (&win)[K - 1][V]) {
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const long long u = t - (K - 1) + j;
    if (u >= at.begin) load_row<T, V>(x + u * a.d.x.row, win[j]);
    else if (a.initial) load_row<T, V>(static_cast<const T*>(a.initial) + ((K - 1LL) * at.seq + (K - 1) + (u - at.begin)) * a.d.C + c, win[j]);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = 0.f;
  }
}

template <typename T, int V, int K>
__device__ __forceinline__ void load_window(const CausalArgs& a, const T* x, const Place& at, long long t, int c, Pair (&win)[K - 1][kPairs<V>]) {
  constexpr int kNext = V > 1 ? 1 : 0;
  float f[K - 1][V];
  load_window<T, V, K>(a, x, at, t, c, f);
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) win[j][i] = Pair(f[j][2 * i], f[j][2 * i + kNext]);
}

// Rows of the final states: thread i of these blocks takes one piece of one row of one sequence.
template <typename T, int V, int K>
__device__ __forceinline__ void final_state(const CausalArgs& a, long long block) {
  const int vecs = a.d.C / V;
  const long long i = block * 256 + threadIdx.x;
  if (i >= a.d.sequences * (K - 1) * vecs) return;
  const int c = static_cast<int>(i % vecs) * V, j = static_cast<int>(i / vecs % (K - 1));
  const int seq = static_cast<int>(i / vecs / (K - 1));
  const long long begin = a.d.packed ? start_of(a.starts, seq, a.d.length) : 0;
  const long long end = a.d.packed ? start_of(a.starts, seq + 1, a.d.length) : a.d.length;
  const long long len = end > begin ? end - begin : 0, u = len - (K - 1) + j;
  Pack<T, V> v;
  if (u >= 0) v.load(static_cast<const T*>(a.x) + (a.d.packed ? 0 : seq * a.d.x.seq) + (begin + u) * a.d.x.row + c);
  else if (a.initial) v.load(static_cast<const T*>(a.initial) + ((K - 1LL) * seq + (K - 1) + u) * a.d.C + c);
  else v.clear();
  v.store(static_cast<T*>(a.final) + ((K - 1LL) * seq + j) * a.d.C + c);
}

// Whether pieces of V > 1 channels lie on their boundaries in all tensors of the call.
inline bool wide_causal(const CausalArgs& a) {
  const int dt = a.d.dtype;
  return a.d.C % (dt == B200CONV_F32 ? 4 : 8) == 0 && rows_aligned(a.x, a.d.x, dt) && rows_aligned(a.y, a.d.y, dt) && rows_aligned(a.dy, a.d.dy, dt) &&
         rows_aligned(a.dx, a.d.dx, dt) && aligned16({a.w, a.bias, a.initial, a.final, a.dinitial});
}
// f(type, pieces of V channels, taps) for the call's data type and filter width.
template <typename T, int V, class F> cudaError_t with_taps(int width, F f) {
  switch (width) {
#define B200_TAPS(K) case K: return f(T(), std::integral_constant<int, V>(), std::integral_constant<int, K>());
    B200_TAPS(2) B200_TAPS(3) B200_TAPS(4) B200_TAPS(5) B200_TAPS(6) B200_TAPS(7) B200_TAPS(8)
#undef B200_TAPS
  }
  return cudaErrorInvalidValue;
}
template <int WIDE16 = 8, class F> cudaError_t with_causal(const CausalArgs& a, bool wide, F f) {
  if (a.d.dtype == B200CONV_F32) return wide ? with_taps<float, 4>(a.d.width, f) : with_taps<float, 1>(a.d.width, f);
  if (a.d.dtype == B200CONV_F16) return wide ? with_taps<__half, WIDE16>(a.d.width, f) : with_taps<__half, 1>(a.d.width, f);
  return wide ? with_taps<__nv_bfloat16, WIDE16>(a.d.width, f) : with_taps<__nv_bfloat16, 1>(a.d.width, f);
}

}  // namespace b200
