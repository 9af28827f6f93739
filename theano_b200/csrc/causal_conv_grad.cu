// Gradients of the short causal convolution.
//
//   g[t] = dy[t] silu'(pre[t])  (pre from x again),   dx[t] = sum over k of w[k] g[t + k],
//   dw[k] = sum over tokens of g[t] x[t - k],  dbias = sum of g,  and the initial state's rows like tokens before the first
//
// x and dy are read once, dx is written once.  A thread walks along a run of tokens with the last taps - 1 rows of x and the unfinished sums
// of dx in registers, and taps - 1 tokens beyond its run for the sums that end there.  The filters' sums stay in registers too; a
// block adds its runs and leaves one row of partial sums, which a second kernel adds in block order.  4 x 2047 x 1024 float32, 4 taps:
// 25 us (4.0 TB/s) and 5 for the second kernel; four channels per thread take 166 registers, three blocks of 128 threads to an SM, which
// bounds the bytes on their way.  Blocks of 256 threads left one to an SM: 45 us.
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
  const long long i = block * blockDim.x + threadIdx.x;
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

// The slope of both
__device__ __forceinline__ Pair silu_slope2(Pair v) {
  const float2 e = mul2(v, Pair(-kLog2e, -kLog2e)).get();
  const Pair one(1.f, 1.f);
  const float2 d = add2(Pair(exp2_fast(e.x), exp2_fast(e.y)), one).get();
  const Pair s(reciprocal_fast(d.x), reciprocal_fast(d.y));
  return mul2(s, fma2(v, fma2(s, Pair(-1.f, -1.f), one), one));
}

constexpr int kGradThreads = 128;
template <int K> constexpr int kGradBlocks = K <= 4 ? 3 : 2;            // of an SM

template <typename T, int V, int K>
__global__ void __launch_bounds__(kGradThreads, kGradBlocks<K>) causal_grad_kernel(CausalArgs a, CausalGrid g) {
  constexpr int H = kPairs<V>;
  pdl_enter();
  __shared__ float part[kGradThreads][V + 1];
  if (blockIdx.x >= g.run_blocks) {
    initial_grad<T, V, K>(a, blockIdx.x - g.run_blocks);
    return;
  }
  const int lanes = 1 << g.log_lanes, lane = threadIdx.x & (lanes - 1), rows = kGradThreads >> g.log_lanes;
  const int cb = blockIdx.x % g.channel_blocks, rb = blockIdx.x / g.channel_blocks;
  const int c = ((cb << g.log_lanes) + lane) * V;
  const bool inside = c < a.d.C;
  const RunPlace p = place_run(a, g, 1LL * rb * rows + (threadIdx.x >> g.log_lanes));
  Place at = place_run_start(a, p);
  Pair dw[K][H], db[H];
#pragma unroll
  for (int i = 0; i < H; ++i) {
    db[i] = Pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][i] = Pair(0.f, 0.f);
  }
  if (inside && p.from < p.to) {
    Pair w[K][H], bias[H];
    load_filter<T, V, K>(a, c, w, bias);
    const long long xr = a.d.x.row, yr = a.d.dy.row, dr = a.d.dx.row;
    const T* x = static_cast<const T*>(a.x) + p.seq * a.d.x.seq + c;
    const T* dy = static_cast<const T*>(a.dy) + p.seq * a.d.dy.seq + c;
    T* dx = static_cast<T*>(a.dx) + p.seq * a.d.dx.seq + c;
    const bool pads = c + V >= a.d.C && a.d.dx.stored > a.d.C;
    for (long long from = p.from; from < p.to;) {            // the piece of each sequence in the run
      if (from > p.from && !next_sequence(a, from, &at)) break;
      from = at.token;
      if (from >= p.to) break;
      const long long to = at.end < p.to ? at.end : p.to;
      // tokens of the piece, tokens to read (those beyond it for the sums that end there), rounds until the last sum has left
      const int mine = static_cast<int>(to - from), read = static_cast<int>((at.end < to + K - 1 ? at.end : to + K - 1) - from), last = mine + K - 1;
      Pair win[K - 1][H], acc[K - 1][H];
      load_window<T, V, K>(a, x, at, from, c, win);
#pragma unroll
      for (int k = 0; k + 1 < K; ++k)
#pragma unroll
        for (int i = 0; i < H; ++i) acc[k][i] = Pair(0.f, 0.f);
      constexpr int kRound = 4;                  // rows on their way
      const T* px = x + from * xr;
      const T* py = dy + from * yr;
      T* pd = dx + (from - (K - 1)) * dr;
      Pack<T, V> nx[kRound], ny[kRound], cx[kRound], cy[kRound];
      auto fetch = [&](int left) {
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
          nx[u].clear();
          ny[u].clear();
          if (u < left) {
            nx[u].load(px + u * xr);
            ny[u].load(py + u * yr);
          }
        }
        px += kRound * xr;
        py += kRound * yr;
      };
      fetch(read);
      for (int t0 = 0; t0 < last; t0 += kRound) {
#pragma unroll
        for (int u = 0; u < kRound; ++u) { cx[u] = nx[u]; cy[u] = ny[u]; }
        fetch(read - t0 - kRound);               // on their way while these are computed
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
          const int t = t0 + u;
          if (t >= last) break;
          Pack<T, V> done;
          const bool behind = t >= read, sums = t < mine;
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const Pair now = pair_of(cx[u], i, 0.f);
            Pair gr = pair_of(cy[u], i, 0.f);
            if (a.d.silu) {
              Pair pre = fma2(w[0][i], now, bias[i]);
#pragma unroll
              for (int k = 1; k < K; ++k) pre = fma2(w[k][i], win[K - 1 - k][i], pre);
              gr = mul2(gr, silu_slope2(pre));
            }
            if (behind) gr = Pair(0.f, 0.f);                 // behind the sequence: only sums that wait for their store
            if (sums) {
              db[i] = add2(gr, db[i]);
              dw[0][i] = fma2(gr, now, dw[0][i]);
#pragma unroll
              for (int k = 1; k < K; ++k) dw[k][i] = fma2(gr, win[K - 1 - k][i], dw[k][i]);
            }
            put_pair(done, i, fma2(w[K - 1][i], gr, acc[K - 2][i]));
#pragma unroll
            for (int k = K - 2; k > 0; --k) acc[k][i] = fma2(w[k][i], gr, acc[k - 1][i]);
            acc[0][i] = mul2(w[0][i], gr);
#pragma unroll
            for (int j = 0; j + 2 < K; ++j) win[j][i] = win[j + 1][i];
            win[K - 2][i] = now;
          }
          if (t >= K - 1) {
            done.store(pd + u * dr);
            if (pads)
              for (int z = V; c + z < a.d.dx.stored; ++z) pd[u * dr + z] = from_float<T>(0.f);
          }
        }
        pd += kRound * dr;
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
    for (int i = 0; i < H; ++i) {
      const float2 v = (k < K ? dw[k < K ? k : 0][i] : db[i]).get();
      part[threadIdx.x][2 * i] = v.x;
      if (V > 1) part[threadIdx.x][2 * i + (V > 1 ? 1 : 0)] = v.y;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < lanes * V; e += kGradThreads) {
      const int l = e / V, i = e % V, ch = ((cb << g.log_lanes) + l) * V + i;
      float v = 0.f;
      for (int r = 0; r < rows; ++r) v += part[(r << g.log_lanes) + l][i];
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

CausalGrid grad_grid(const CausalArgs& a, int V) {
  return causal_grid(a, V, kGradThreads, 148LL * (a.d.width <= 4 ? kGradBlocks<4> : kGradBlocks<8>), 8);
}

template <typename T, int V, int K>
cudaError_t backward(const CausalArgs& a, int* launches, cudaStream_t s) {
  const CausalGrid g = grad_grid(a, V);
  long long grid = g.run_blocks;
  if (a.dinitial) grid += (a.d.sequences * (K - 1) * (a.d.C / V) + kGradThreads - 1) / kGradThreads;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  *launches = 1;
  launch_streaming(causal_grad_kernel<T, V, K>, static_cast<unsigned>(grid), kGradThreads, 0, s, a, g);
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
