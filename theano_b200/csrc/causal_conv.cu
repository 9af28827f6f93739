// The short causal convolution: every channel with its own filter of 2 to 8 taps, bias and SiLU in the same pass.
//
//   pre[t][c] = bias[c] + sum over k of w[c][k] x[t - k][c],   y = pre or pre * sigmoid(pre)
//
// (a true convolution; without `flip` the taps are counted from the oldest token).  Tokens before a sequence's first are
// the rows of its initial state, or zeros; the final state is the last taps - 1 rows of (initial state, x).
// x is read once and y written once: a thread takes four neighbouring channels and walks along a run of tokens with the last taps - 1 rows
// in registers; only those rows are read a second time, out of L2, by the next run.  Runs are as long as lets all blocks be
// resident at once, and the rows ahead are loaded while the present ones are computed.  8192 packed tokens of 2048 channels,
// 4 taps, bfloat16: 21 us (3.2 TB/s), bound by the issue slots and the special function unit together (18 instructions per element and
// lane, two trips for SiLU); with 8 channels per thread 33 us, without rows on their way 37.  4 x 2047 x 1024 float32: 12 us (5.6 TB/s).
#include "causal_conv.cuh"
#include "internal.h"

namespace b200 {
namespace {

constexpr int kAhead = 4;                        // rows whose loads a thread has in flight

template <typename T, int K> constexpr int kBlocks = K <= 4 && sizeof(T) == 2 ? 3 : 2;     // of an SM: what the registers allow
template <typename T, int V, int K>
__global__ void __launch_bounds__(256, kBlocks<T, K>) causal_conv_kernel(CausalArgs a, CausalGrid g) {
  pdl_enter();
  if (blockIdx.x >= g.run_blocks) {              // the states behind the sequences, in blocks of their own
    final_state<T, V, K>(a, blockIdx.x - g.run_blocks);
    return;
  }
  const int c = ((blockIdx.x % g.channel_blocks << g.log_lanes) + (threadIdx.x & ((1 << g.log_lanes) - 1))) * V;
  const long long run = (static_cast<long long>(blockIdx.x / g.channel_blocks) << (8 - g.log_lanes)) + (threadIdx.x >> g.log_lanes);
  const RunPlace p = place_run(a, g, run);
  Place at = place_run_start(a, p);
  if (c >= a.d.C || p.from >= p.to) return;
  Pair w[K][kPairs<V>], bias[kPairs<V>], win[K - 1][kPairs<V>];
  load_filter<T, V, K>(a, c, w, bias);
  const long long xr = a.d.x.row, yr = a.d.y.row;
  const T* x = static_cast<const T*>(a.x) + p.seq * a.d.x.seq + c;
  T* y = static_cast<T*>(a.y) + p.seq * a.d.y.seq + c;
  long long t = at.token;
  if (t >= p.to) return;                         // rows of no sequence
  Pack<T, V> in[kAhead], next[kAhead];
  auto fetch = [&](const T* from, int left, Pack<T, V> (&to)[kAhead]) {
    if (left >= kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) to[k].load(from + k * xr);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < left) to[k].load(from + k * xr);
    }
  };
  const T* from = x + t * xr;
  T* to = y + t * yr;
  int left = static_cast<int>(p.to - t), same = static_cast<int>((at.end < p.to ? at.end : p.to) - t);      // tokens of the run, of this sequence in it
  fetch(from, left, in);
  load_window<T, V, K>(a, x, at, t, c, win);
  const bool pads = c + V >= a.d.C && a.d.y.stored > a.d.C;
  auto token = [&](int k) {
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      const Pair now = pair_of(in[k], i, 0.f);
      Pair pre = fma2(w[0][i], now, bias[i]);
#pragma unroll
      for (int j = 1; j < K; ++j) pre = fma2(w[j][i], win[K - 1 - j][i], pre);
      put_pair(o, i, a.d.silu ? silu2(pre) : pre);
#pragma unroll
      for (int j = 0; j + 2 < K; ++j) win[j][i] = win[j + 1][i];
      win[K - 2][i] = now;
    }
    o.store(to + k * yr);
    if (pads)
      for (int z = V; c + z < a.d.y.stored; ++z) to[k * yr + z] = from_float<T>(0.f);
  };
  while (left > 0) {
    from += kAhead * xr;
    fetch(from, left - kAhead, next);            // on their way while these are computed
    if (same >= kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) token(k);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (k >= left) break;
        if (k >= same) {                         // packed sequences: the next one begins here, or rows of none
          if (!next_sequence(a, t + k, &at)) return;
          load_window<T, V, K>(a, x, at, t + k, c, win);
          same = static_cast<int>((at.end < p.to ? at.end : p.to) - t);
        }
        token(k);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) in[k] = next[k];
    t += kAhead;
    left -= kAhead;
    same -= kAhead;
    to += kAhead * yr;
  }
}

// One token of every sequence: reads the state and the token, leaves y and the state moved on by a row.  64 x 2048 bfloat16: 3.9 us, the
// time of a launch and two trips to memory (2.1 MB); eight channels per thread, so that a row of the state is one load.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128) causal_step_kernel(CausalArgs a, int vecs) {
  pdl_enter();
  const long long i = blockIdx.x * 128LL + threadIdx.x;
  if (i >= a.d.sequences * vecs) return;
  const long long seq = i / vecs;
  const int c = static_cast<int>(i - seq * vecs) * V;
  T* state = static_cast<T*>(a.final) + seq * (K - 1) * a.d.C + c;
  Pack<T, V> old[K - 1], now;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) old[j].load(state + 1LL * j * a.d.C);
  now.load(static_cast<const T*>(a.x) + seq * a.d.x.seq + c);
  float w[K][V], bias[V], out[V];
  load_filter<T, V, K>(a, c, w, bias);
#pragma unroll
  for (int q = 0; q < V; ++q) {
    float pre = fmaf(w[0][q], now.get(q), bias[q]);       // in the order of a prompt
#pragma unroll
    for (int j = 1; j < K; ++j) pre = fmaf(w[j][q], old[K - 1 - j].get(q), pre);
    out[q] = a.d.silu ? silu(pre) : pre;
  }
#pragma unroll
  for (int j = 0; j + 2 < K; ++j) old[j + 1].store(state + 1LL * j * a.d.C);
  now.store(state + (K - 2LL) * a.d.C);
  T* y = static_cast<T*>(a.y) + seq * a.d.y.seq + c;
  store_row<T, V>(y, out);
  if (c + V >= a.d.C)
    for (int z = V; c + z < a.d.y.stored; ++z) y[z] = from_float<T>(0.f);
}

template <typename T, int V, int K>
cudaError_t forward(const CausalArgs& a, cudaStream_t s) {
  const CausalGrid g = causal_grid(a, V, 256, 148 * kBlocks<T, K>, kAhead);
  long long grid = g.run_blocks;
  if (a.final) grid += (a.d.sequences * (K - 1) * (a.d.C / V) + 255) / 256;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  if (grid) launch_streaming(causal_conv_kernel<T, V, K>, static_cast<unsigned>(grid), 256, 0, s, a, g);
  return cudaGetLastError();
}
template <typename T, int V, int K>
cudaError_t step(const CausalArgs& a, cudaStream_t s) {
  const int vecs = a.d.C / V;
  const long long grid = (a.d.sequences * vecs + 127) / 128;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  launch_streaming(causal_step_kernel<T, V, K>, static_cast<unsigned>(grid), 128, 0, s, a, vecs);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_causal_conv(const CausalArgs& a, cudaStream_t s) {
  return with_causal<4>(a, wide_causal(a), [&](auto t, auto v, auto k) { return forward<decltype(t), decltype(v)::value, decltype(k)::value>(a, s); });
}
cudaError_t launch_causal_step(const CausalArgs& a, cudaStream_t s) {
  return with_causal(a, wide_causal(a), [&](auto t, auto v, auto k) { return step<decltype(t), decltype(v)::value, decltype(k)::value>(a, s); });
}

}  // namespace b200
