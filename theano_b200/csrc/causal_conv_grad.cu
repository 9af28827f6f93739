// Gradients of the short causal convolution.
//
//   g[t] = dy[t] silu'(pre[t])  (pre from x again),   dx[t] = sum over k of w[k] g[t + k],
//   dw[k] = sum over tokens of g[t] x[t - k],  dbias = sum of g,  and the initial state's rows like tokens before the first
//
// HBM bound: x and dy are read once, dx is written once.  A thread walks along a run of tokens with the last taps - 1 rows of x
// and the unfinished sums of dx in registers, and taps - 1 tokens beyond its run for the sums that end there.  The
// filters' sums stay in registers too; a block adds its runs and leaves one row of partial sums, which a second kernel adds
// in block order.
#include "causal_conv.cuh"
#include "internal.h"

namespace b200 {
namespace {

// d(pre sigmoid(pre)) = sigmoid (1 + pre (1 - sigmoid))
__device__ __forceinline__ float silu_slope(float v) {
  const float s = sigmoid(v);
  return s * (1.f + v * (1.f - s));
}

// Gradient of the initial states: one thread per piece of a row of a sequence, taps terms each, from the first tokens.
template <typename T, int V, int K>
__device__ void initial_grad(const CausalArgs& a, long long block) {
  const int vecs = a.d.C / V;
  const long long i = block * 256 + threadIdx.x;
  if (i >= a.d.sequences * (K - 1) * vecs) return;
  const int c = static_cast<int>(i % vecs) * V, j = static_cast<int>(i / vecs % (K - 1));
  Place at;
  at.seq = static_cast<int>(i / vecs / (K - 1));
  at.begin = a.d.packed ? start_of(a.starts, at.seq, a.d.length) : 0;
  at.end = a.d.packed ? start_of(a.starts, at.seq + 1, a.d.length) : a.d.length;
  const long long seq = a.d.packed ? 0 : at.seq;
  const T* x = static_cast<const T*>(a.x) + seq * a.d.x.seq + c;
  const T* dy = static_cast<const T*>(a.dy) + seq * a.d.dy.seq + c;
  float w[K][V], bias[V], sum[V];
  load_filter<T, V, K>(a, c, w, bias);
#pragma unroll
  for (int q = 0; q < V; ++q) sum[q] = 0.f;
#pragma unroll
  for (int k = 1; k < K; ++k) {
    const long long t = at.begin + j - (K - 1) + k;          // the token that meets this row k steps later
    if (t < at.begin || t >= at.end) continue;
    float win[K - 1][V], now[V], g[V];
    load_window<T, V, K>(a, x, at, t, c, win);
    load_row<T, V>(x + t * a.d.x.row, now);
    load_row<T, V>(dy + t * a.d.dy.row, g);
#pragma unroll
    for (int q = 0; q < V; ++q) {
      float pre = bias[q] + w[0][q] * now[q];
#pragma unroll
      for (int m = 1; m < K; ++m) pre += w[m][q] * win[K - 1 - m][q];
      sum[q] += w[k][q] * (a.d.silu ? g[q] * silu_slope(pre) : g[q]);
    }
  }
  store_row<T, V>(static_cast<T*>(a.dinitial) + ((K - 1LL) * at.seq + j) * a.d.C + c, sum);
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(256) causal_grad_kernel(CausalArgs a, CausalGrid g) {
  pdl_enter();
  __shared__ float part[256][V + 1];
  if (blockIdx.x >= g.run_blocks) {
    initial_grad<T, V, K>(a, blockIdx.x - g.run_blocks);
    return;
  }
  const int lanes = 1 << g.log_lanes, lane = threadIdx.x & (lanes - 1);
  const int cb = blockIdx.x % g.channel_blocks, rb = blockIdx.x / g.channel_blocks;
  const int c = ((cb << g.log_lanes) + lane) * V;
  const bool inside = c < a.d.C;
  RunPlace p = place_run(a, g, (static_cast<long long>(rb) << (8 - g.log_lanes)) + (threadIdx.x >> g.log_lanes));
  float w[K][V], bias[V], dw[K][V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
  }
  if (inside && p.from < p.to) {
    load_filter<T, V, K>(a, c, w, bias);
    const T* x = static_cast<const T*>(a.x) + p.seq * a.d.x.seq + c;
    const T* dy = static_cast<const T*>(a.dy) + p.seq * a.d.dy.seq + c;
    T* dx = static_cast<T*>(a.dx) + p.seq * a.d.dx.seq + c;
    for (long long from = p.from; from < p.to;) {            // the piece of each sequence in the run
      const Place at = place_token(a, p, from);
      from = at.token;
      if (from >= p.to) break;
      const long long to = at.end < p.to ? at.end : p.to, last = to + K - 1;
      float win[K - 1][V], acc[K][V];
      load_window<T, V, K>(a, x, at, from, c, win);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[k][i] = 0.f;
      constexpr int kStep = 4;
      for (long long t0 = from; t0 < last; t0 += kStep) {
        Pack<T, V> px[kStep], pd[kStep];
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
          if (t0 + u < last && t0 + u < at.end) {
            px[u].load(x + (t0 + u) * a.d.x.row);
            pd[u].load(dy + (t0 + u) * a.d.dy.row);
          } else {
            px[u].clear();
            pd[u].clear();
          }
        }
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
          const long long t = t0 + u;
          if (t >= last) break;
          float done[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float now = px[u].get(i);
            float pre = bias[i] + w[0][i] * now;
#pragma unroll
            for (int k = 1; k < K; ++k) pre += w[k][i] * win[K - 1 - k][i];
            float gr = pd[u].get(i);
            if (a.d.silu) gr *= silu_slope(pre);
            if (t >= at.end) gr = 0.f;                       // behind the sequence: only sums that wait for their store
            if (t < to) {
              db[i] += gr;
              dw[0][i] += gr * now;
#pragma unroll
              for (int k = 1; k < K; ++k) dw[k][i] += gr * win[K - 1 - k][i];
            }
            done[i] = acc[K - 1][i] + w[K - 1][i] * gr;
#pragma unroll
            for (int k = K - 1; k > 0; --k) acc[k][i] = acc[k - 1][i] + w[k - 1][i] * gr;
#pragma unroll
            for (int j = 0; j + 2 < K; ++j) win[j][i] = win[j + 1][i];
            win[K - 2][i] = now;
          }
          const long long at_row = t - (K - 1);
          if (at_row >= from) {
            store_row<T, V>(dx + at_row * a.d.dx.row, done);
            if (c + V >= a.d.C)
              for (int z = V; c + z < a.d.dx.stored; ++z) dx[at_row * a.d.dx.row + z] = from_float<T>(0.f);
          }
        }
      }
      from = to;
    }
  }
  if (!a.partial) return;
  // the runs of the block in order, a tap at a time; the last round is the bias
  float* out = a.partial + static_cast<long long>(rb) * (K + 1) * a.d.C;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) part[threadIdx.x][i] = k < K ? dw[k < K ? k : 0][i] : db[i];
    __syncthreads();
    for (int e = threadIdx.x; e < lanes * V; e += 256) {
      const int l = e / V, i = e % V, ch = ((cb << g.log_lanes) + l) * V + i;
      float v = 0.f;
      for (int r = 0; r < 256 >> g.log_lanes; ++r) v += part[(r << g.log_lanes) + l][i];
      if (ch < a.d.C) out[1LL * k * a.d.C + ch] = v;
    }
    __syncthreads();
  }
}

// 32 channels of one tap (or the bias) per block; warp w adds the parts w, w + 16, ..., the warps' sums in warp order.
template <typename T>
__global__ void __launch_bounds__(512) causal_params_kernel(CausalArgs a, int parts) {
  pdl_enter();
  __shared__ float part[16][32];
  const int C = a.d.C, K = a.d.width, wp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, k = blockIdx.y;
  void* out = k < K ? a.dw : a.dbias;
  if (!out) return;
  float acc = 0.f;
  if (c < C)
#pragma unroll 10
    for (int b = wp; b < parts; b += 16) acc += a.partial[(1LL * b * (K + 1) + k) * C + c];
  part[wp][lane] = acc;
  __syncthreads();
  if (wp == 0 && c < C) {
    for (int q = 1; q < 16; ++q) acc += part[q][lane];
    set_param<T>(out, k == K ? c : 1LL * c * K + (a.d.flip ? k : K - 1 - k), a.d.param_f32, acc);
  }
}

// Runs that are long enough for few partial sums, short enough to occupy the SMs with two blocks each.
CausalGrid grad_grid(const CausalArgs& a, int V) { return causal_grid(a, V, 148 * 2 * 256, 16, 1 << 20); }

template <typename T, int V, int K>
cudaError_t backward(const CausalArgs& a, int* launches, cudaStream_t s) {
  const CausalGrid g = grad_grid(a, V);
  long long grid = g.run_blocks;
  if (a.dinitial) grid += (a.d.sequences * (K - 1) * (a.d.C / V) + 255) / 256;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  *launches = 1;
  launch_streaming(causal_grad_kernel<T, V, K>, static_cast<unsigned>(grid), 256, 0, s, a, g);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !a.partial) return e;
  launch_chained(causal_params_kernel<T>, dim3((a.d.C + 31) / 32, K + 1), 512, 0, s, a, static_cast<int>(g.run_blocks / g.channel_blocks));
  ++*launches;
  return cudaGetLastError();
}

}  // namespace

// Four channels per thread: filters, their sums, the window and the unfinished sums are 17 registers per channel.
int causal_grad_parts(const CausalArgs& a) {
  const CausalGrid g = grad_grid(a, wide_causal(a) ? 4 : 1);
  return g.channel_blocks ? static_cast<int>(g.run_blocks / g.channel_blocks) : 0;
}
cudaError_t launch_causal_grad(const CausalArgs& a, int* launches, cudaStream_t s) {
  return with_causal<4>(a, wide_causal(a),
                        [&](auto t, auto v, auto k) { return backward<decltype(t), decltype(v)::value, decltype(k)::value>(a, launches, s); });
}

}  // namespace b200
