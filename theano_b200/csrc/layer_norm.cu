// Layer norm over the channels of every row, forward and backward.
//
//   t = x + r (the residual stream, rounded to the tensors' type as it is stored)
//   mean = sum t / C,  rstd = 1 / sqrt(sum (t - mean)^2 / C + eps),  hat = (t - mean) rstd,  y = hat gamma + beta
//   dt = rstd (g - mean(g) - hat mean(g hat)) + dtotal  with g = dy gamma;  dgamma = sum over rows of dy hat, dbeta of dy
//
// Both passes move bytes: a row is read once and stays in registers, so that the variance is the mean of squared differences
// from the mean and not a difference of large sums.  All sums are float32.  What keeps them off the HBM rate is the issue slots (a forward
// row of 2048 takes 17 instructions per element and lane with everything, 58 % of the slots): elements change type and are
// computed two at a time, few threads share a row, and a row's sums meet at a barrier of its own threads.  16384 x 2048 bfloat16: forward
// 30 us (4.5 TB/s), backward 51 (3.9 TB/s) and 7 for the parameters' sums; 6003 x 1000 float16 with residual 11.9 us (4.0 TB/s).
#include "internal.h"
#include "rows.cuh"

namespace b200 {
namespace {

constexpr int kNormThreads = 256;                // of a block, unless a row takes more
constexpr int kGradThreads = 256;
constexpr int kGradBlocks = 2;                   // of an SM

__device__ __forceinline__ void locate(const b200conv_norm_desc& d, long long row, long long* seq, long long* tok) {
  if (d.sequences == 1) { *seq = 0; *tok = row; return; }         // rows that all follow each other
  if (row < (1LL << 31) && d.length < (1LL << 31)) {
    *seq = static_cast<uint32_t>(row) / static_cast<uint32_t>(d.length);
    *tok = row - *seq * d.length;
  } else {
    *seq = row / d.length;
    *tok = row - *seq * d.length;
  }
}
__device__ __forceinline__ long long at(const b200conv_rows& r, long long seq, long long tok) { return seq * r.seq + tok * r.row; }

// Sums of N values over the TPR threads of a row (TPR > 32: `shared` holds N floats per warp of the block; the caller
// alternates between two of them, so that one barrier per sum is enough).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*shared)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(~0u, v[n], o);
  if (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) shared[warp][n] = v[n];
    // a barrier for the row's threads alone: the block's other rows go on
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / TPR), "n"(TPR) : "memory");
    const int first = warp & ~(TPR / 32 - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = 0.f;
    // as wide as the parts lie together: two warps' pairs, four warps' single sums
    const float4* p = reinterpret_cast<const float4*>(&shared[first][0]);
#pragma unroll
    for (int w = 0; w < TPR / 32 * N / 4; ++w) {
      const float4 f = p[w];
      if (N == 2) { v[0] += f.x + f.z; v[N - 1] += f.y + f.w; }
      else v[0] += (f.x + f.y) + (f.z + f.w);
    }
    if (TPR / 32 * N < 4) {                      // two warps of single sums
      v[0] = shared[first][0] + shared[first + 1][0];
    }
  }
}

template <typename T>
__device__ __forceinline__ void zero_pads(T* row, int C, int stored, int lane, int lanes) {
  for (int c = C + lane; c < stored; c += lanes) row[c] = from_float<T>(0.f);
}

// TPR threads per row, VPT pieces of V channels per thread.  C is a multiple of V.
template <typename T, int V, int VPT, int TPR>
__global__ void __launch_bounds__(TPR < kNormThreads ? kNormThreads : TPR, VPT >= 4 && TPR < 128 ? (TPR == 64 ? 4 : 3) : 1) norm_kernel(NormArgs a) {
  constexpr int kThreads = TPR < kNormThreads ? kNormThreads : TPR;
  pdl_enter();
  __shared__ __align__(16) float part[2][kThreads / 32][1];
  const int C = a.d.C, lane = threadIdx.x % TPR;
  const long long rows = a.d.sequences * a.d.length;
  const long long row = 1LL * blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  const bool active = row < rows;
  long long seq = 0, tok = 0;
  if (active) locate(a.d, row, &seq, &tok);
  const T* x = static_cast<const T*>(a.x) + at(a.d.x, seq, tok);
  Pack<T, V> px[VPT], pr[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = (k * TPR + lane) * V;
    if (active && c < C) px[k].load(x + c);
    else px[k].clear();
  }
  if (a.residual) {
    const T* r = static_cast<const T*>(a.residual) + at(a.d.residual, seq, tok);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (k * TPR + lane) * V;
      if (active && c < C) pr[k].load(r + c);
      else pr[k].clear();
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int i = 0; i < kPairs<V>; ++i) put_pair(px[k], i, add2(pair_of(px[k], i, 0.f), pair_of(pr[k], i, 0.f)));
  }
  if (a.total && active) {
    T* t = static_cast<T*>(a.total) + at(a.d.total, seq, tok);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (k * TPR + lane) * V;
      if (c < C) px[k].store(t + c);
    }
    zero_pads(t, C, a.d.total.stored, lane, TPR);
  }
  Pair sums(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) sums = add2(sums, pair_of(px[k], i, 0.f));
  float sum[1] = {sums.get().x + sums.get().y};
  row_sum<TPR, 1>(sum, part[0]);
  const float mean = sum[0] / C;
  const Pair away(-mean, -mean);
  Pair squares(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if ((k * TPR + lane) * V < C)
#pragma unroll
      for (int i = 0; i < kPairs<V>; ++i) {
        const Pair d = add2(pair_of(px[k], i, mean), away);
        squares = fma2(d, d, squares);
      }
  float sq[1] = {squares.get().x + squares.get().y};
  row_sum<TPR, 1>(sq, part[1]);
  const float rstd = 1.f / sqrtf(sq[0] / C + a.d.eps);
  if (!active) return;
  if (a.stats && lane == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, rstd);
  T* y = static_cast<T*>(a.y) + at(a.d.y, seq, tok);
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = (k * TPR + lane) * V;
    if (c < C) {
      Pack<T, V> o;
      float gamma[V], beta[V];
#pragma unroll
      for (int i = 0; i < V; ++i) { gamma[i] = 1.f; beta[i] = 0.f; }
      if (a.d.param_f32 || sizeof(T) == 4) {
        if (a.gamma) load_params<float, V>(a.gamma, c, gamma);
        if (a.beta) load_params<float, V>(a.beta, c, beta);
      } else {
        if (a.gamma) load_params<T, V>(a.gamma, c, gamma);
        if (a.beta) load_params<T, V>(a.beta, c, beta);
      }
      const Pair scale(rstd, rstd);
#pragma unroll
      for (int i = 0; i < kPairs<V>; ++i) {
        constexpr int kNext = V > 1 ? 1 : 0;
        put_pair(o, i, fma2(mul2(add2(pair_of(px[k], i, mean), away), scale), Pair(gamma[2 * i], gamma[2 * i + kNext]),
                            Pair(beta[2 * i], beta[2 * i + kNext])));
      }
      o.store(y + c);
    }
  }
  zero_pads(y, C, a.d.y.stored, lane, TPR);
}

// Rows of any length: read three times, the last two from L2 (a row of 65536 float32 is 256 KB).
template <typename T>
__global__ void __launch_bounds__(512) norm_long_kernel(NormArgs a) {
  pdl_enter();
  __shared__ __align__(16) float part[2][16][1];
  const int C = a.d.C, lane = threadIdx.x;
  long long seq, tok;
  locate(a.d, blockIdx.x, &seq, &tok);
  const T* x = static_cast<const T*>(a.x) + at(a.d.x, seq, tok);
  const T* r = a.residual ? static_cast<const T*>(a.residual) + at(a.d.residual, seq, tok) : nullptr;
  T* t = a.total ? static_cast<T*>(a.total) + at(a.d.total, seq, tok) : nullptr;
  auto value = [&](int c) { return r ? to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))) : to_float(x[c]); };
  float sum[1] = {0.f}, sq[1] = {0.f};
  for (int c = lane; c < C; c += 512) sum[0] += value(c);
  row_sum<512, 1>(sum, part[0]);
  const float mean = sum[0] / C;
  for (int c = lane; c < C; c += 512) {
    const float d = value(c) - mean;
    sq[0] += d * d;
  }
  row_sum<512, 1>(sq, part[1]);
  const float rstd = 1.f / sqrtf(sq[0] / C + a.d.eps);
  if (a.stats && lane == 0) reinterpret_cast<float2*>(a.stats)[blockIdx.x] = make_float2(mean, rstd);
  T* y = static_cast<T*>(a.y) + at(a.d.y, seq, tok);
  for (int c = lane; c < C; c += 512) {
    const float v = value(c);
    if (t) t[c] = from_float<T>(v);              // a thread's own channels: total may be x or the residual
    const float g = a.gamma ? param<T>(a.gamma, c, a.d.param_f32) : 1.f, b = a.beta ? param<T>(a.beta, c, a.d.param_f32) : 0.f;
    y[c] = from_float<T>((v - mean) * rstd * g + b);
  }
  if (t) zero_pads(t, C, a.d.total.stored, lane, 512);
  zero_pads(y, C, a.d.y.stored, lane, 512);
}

// Backward: blocks stay and walk over the rows, each group of TPR threads with a stride, so that the sums for dgamma and
// dbeta stay in registers; a block leaves one row of partial sums, which grad_params_kernel adds in block order.
template <typename T, int V, int VPT, int TPR>
__global__ void __launch_bounds__(TPR < kGradThreads ? kGradThreads : TPR, TPR <= kGradThreads ? kGradBlocks : 1) norm_grad_kernel(NormArgs a) {
  constexpr int kThreads = TPR < kGradThreads ? kGradThreads : TPR, kGroups = kThreads / TPR;
  pdl_enter();
  extern __shared__ float sums[];                // [kGroups][TPR * VPT * V] of one parameter at a time
  __shared__ __align__(16) float part[2][kThreads / 32][2];
  const int C = a.d.C, lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const long long rows = a.d.sequences * a.d.length, step = 1LL * gridDim.x * kGroups;
  Pair weight[VPT][kPairs<V>], dg[VPT][kPairs<V>], db[VPT][kPairs<V>];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int i = 0; i < kPairs<V>; ++i) {
      float v[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < (V > 1 ? 2 : 1); ++e) {
        const int c = (k * TPR + lane) * V + 2 * i + e;
        if (c < C) v[e] = a.gamma ? param<T>(a.gamma, c, a.d.param_f32) : 1.f;
      }
      weight[k][i] = Pair(v[0], v[1]);
      dg[k][i] = db[k][i] = Pair(0.f, 0.f);
    }
  Pack<T, V> px[VPT], py[VPT], nx[VPT], ny[VPT];
  float2 st = make_float2(0.f, 0.f), ns = st;
  auto fetch = [&](long long row) {
    if (row >= rows) return;
    long long seq, tok;
    locate(a.d, row, &seq, &tok);
    const T* x = static_cast<const T*>(a.x) + at(a.d.x, seq, tok);
    const T* dy = static_cast<const T*>(a.dy) + at(a.d.dy, seq, tok);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (k * TPR + lane) * V;
      if (c < C) { nx[k].load(x + c); ny[k].load(dy + c); }
    }
    ns = reinterpret_cast<const float2*>(a.stats)[row];
  };
#pragma unroll
  for (int k = 0; k < VPT; ++k) { nx[k].clear(); ny[k].clear(); }
  const long long base = 1LL * blockIdx.x * kGroups;
  fetch(base + group);
  int turn = 0;
  for (long long b = base; b < rows; b += step, turn ^= 1) {
    const long long row = b + group;
    const bool active = row < rows;
#pragma unroll
    for (int k = 0; k < VPT; ++k) { px[k] = nx[k]; py[k] = ny[k]; }
    st = ns;
    fetch(row + step);                           // the next row is on its way all along
    const Pair away(-st.x, -st.x), scale(st.y, st.y);
    Pair g0(0.f, 0.f), g1(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (active && (k * TPR + lane) * V < C)
#pragma unroll
        for (int i = 0; i < kPairs<V>; ++i) {
          const Pair d = pair_of(py[k], i, 0.f), hat = mul2(add2(pair_of(px[k], i, st.x), away), scale), g = mul2(d, weight[k][i]);
          dg[k][i] = fma2(d, hat, dg[k][i]);
          db[k][i] = add2(d, db[k][i]);
          g0 = add2(g, g0);
          g1 = fma2(g, hat, g1);
        }
    float s[2] = {g0.get().x + g0.get().y, g1.get().x + g1.get().y};
    row_sum<TPR, 2>(s, part[turn]);
    if (!active) continue;
    const float m0 = s[0] / C, m1 = s[1] / C;
    long long seq, tok;
    locate(a.d, row, &seq, &tok);
    T* dx = static_cast<T*>(a.dx) + at(a.d.dx, seq, tok);
    const T* dt = a.dtotal ? static_cast<const T*>(a.dtotal) + at(a.d.dtotal, seq, tok) : nullptr;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (k * TPR + lane) * V;
      if (c < C) {
        Pack<T, V> o, more;
        if (dt) more.load(dt + c);
        else more.clear();
        const Pair less(-m0, -m0), slope(-m1, -m1);
#pragma unroll
        for (int i = 0; i < kPairs<V>; ++i) {
          const Pair hat = mul2(add2(pair_of(px[k], i, st.x), away), scale);
          const Pair d = fma2(hat, slope, fma2(pair_of(py[k], i, 0.f), weight[k][i], less));
          put_pair(o, i, fma2(d, scale, pair_of(more, i, 0.f)));
        }
        o.store(dx + c);
      }
    }
    zero_pads(dx, C, a.d.dx.stored, lane, TPR);
  }
  if (!a.partial) return;
  // the groups of the block in group order, first dgamma, then dbeta
  constexpr int kWide = TPR * VPT * V;
  float* out = a.partial + 2LL * blockIdx.x * C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int i = 0; i < kPairs<V>; ++i) {
        const float2 v = (which ? db[k][i] : dg[k][i]).get();
        float* to = sums + group * kWide + (k * TPR + lane) * V + 2 * i;
        to[0] = v.x;
        if (V > 1) to[1] = v.y;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) v += sums[q * kWide + c];
      out[which * C + c] = v;
    }
  }
}

// Rows of any length: dx from three readings, without the parameters' sums, which norm_grad_columns_kernel makes.
template <typename T>
__global__ void __launch_bounds__(512) norm_grad_long_kernel(NormArgs a) {
  pdl_enter();
  __shared__ __align__(16) float part[16][2];
  const int C = a.d.C, lane = threadIdx.x;
  long long seq, tok;
  locate(a.d, blockIdx.x, &seq, &tok);
  const T* x = static_cast<const T*>(a.x) + at(a.d.x, seq, tok);
  const T* dy = static_cast<const T*>(a.dy) + at(a.d.dy, seq, tok);
  const T* dt = a.dtotal ? static_cast<const T*>(a.dtotal) + at(a.d.dtotal, seq, tok) : nullptr;
  T* dx = static_cast<T*>(a.dx) + at(a.d.dx, seq, tok);
  const float2 st = reinterpret_cast<const float2*>(a.stats)[blockIdx.x];
  auto grad = [&](int c) { return to_float(dy[c]) * (a.gamma ? param<T>(a.gamma, c, a.d.param_f32) : 1.f); };
  float s[2] = {0.f, 0.f};
  for (int c = lane; c < C; c += 512) {
    const float g = grad(c);
    s[0] += g;
    s[1] += g * (to_float(x[c]) - st.x) * st.y;
  }
  row_sum<512, 2>(s, part);
  const float m0 = s[0] / C, m1 = s[1] / C;
  for (int c = lane; c < C; c += 512) {
    const float v = st.y * (grad(c) - m0 - (to_float(x[c]) - st.x) * st.y * m1);
    dx[c] = from_float<T>(dt ? v + to_float(dt[c]) : v);
  }
  zero_pads(dx, C, a.d.dx.stored, lane, 512);
}
// One thread per channel and slice of the rows: partial[slice][2][C].
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_columns_kernel(NormArgs a) {
  pdl_enter();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.d.C) return;
  const long long rows = a.d.sequences * a.d.length;
  float dg = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    long long seq, tok;
    locate(a.d, row, &seq, &tok);
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    const float dy = to_float(static_cast<const T*>(a.dy)[at(a.d.dy, seq, tok) + c]);
    dg += dy * (to_float(static_cast<const T*>(a.x)[at(a.d.x, seq, tok) + c]) - st.x) * st.y;
    db += dy;
  }
  a.partial[2LL * blockIdx.y * a.d.C + c] = dg;
  a.partial[(2LL * blockIdx.y + 1) * a.d.C + c] = db;
}

// dgamma and dbeta: 32 channels of one of them per block, warp w adds the parts w, w + 16, ... and the warps' sums are
// added in warp order (the same result on every run).
template <typename T>
__global__ void __launch_bounds__(512) norm_params_kernel(NormArgs a, int parts) {
  pdl_enter();
  __shared__ float part[16][32];
  const int C = a.d.C, wp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  void* out = blockIdx.y ? a.dbeta : a.dgamma;
  if (!out) return;
  float acc = 0.f;
  if (c < C)
#pragma unroll 10
    for (int b = wp; b < parts; b += 16) acc += a.partial[(2LL * b + blockIdx.y) * C + c];
  part[wp][lane] = acc;
  __syncthreads();
  if (wp == 0 && c < C) {
    for (int k = 1; k < 16; ++k) acc += part[k][lane];
    set_param<T>(out, c, a.d.param_f32, acc);
  }
}

// Tensors whose rows all follow each other are one long sequence: no row needs a division.
bool flat(const b200conv_norm_desc& d, const b200conv_rows& r, const void* p) { return !p || r.seq == d.length * r.row; }

template <typename T, int V>
cudaError_t forward(const NormArgs& a, cudaStream_t s) {
  const long long rows = a.d.sequences * a.d.length;
  const int vecs = a.d.C / V;
#define B200_NORM(VPT, TPR)                                                                                         \
  {                                                                                                                 \
    constexpr int kThreads = TPR < kNormThreads ? kNormThreads : TPR;                                               \
    const long long grid = (rows + kThreads / TPR - 1) / (kThreads / TPR);                                          \
    launch_streaming(norm_kernel<T, V, VPT, TPR>, static_cast<unsigned>(grid), kThreads, 0, s, a);                  \
    return cudaGetLastError();                                                                                      \
  }
  if (vecs <= 32) B200_NORM(1, 32)
  if (vecs <= 64) B200_NORM(2, 32)
  // one or two warps per row; with few rows four warps to a row end sooner
  if (rows >= 148 * 8) {
    if (vecs <= 128) B200_NORM(4, 32)
    if (vecs <= 256) B200_NORM(4, 64)
  }
  if (vecs <= 128) B200_NORM(1, 128)
  if (vecs <= 256) B200_NORM(2, 128)
  if (vecs <= 512) B200_NORM(4, 128)
  if (vecs <= 1024) B200_NORM(2, 512)
  if (vecs <= 2048) B200_NORM(4, 512)
#undef B200_NORM
  launch_streaming(norm_long_kernel<T>, static_cast<unsigned>(rows), 512, 0, s, a);
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t backward(const NormArgs& a, int* launches, cudaStream_t s) {
  const long long rows = a.d.sequences * a.d.length;
  const int vecs = a.d.C / V, parts = norm_grad_parts(a.d);
  cudaError_t e;
  *launches = 1;
#define B200_NORM(VPT, TPR)                                                                                         \
  {                                                                                                                 \
    constexpr int kThreads = TPR < kGradThreads ? kGradThreads : TPR, kSmem = kThreads * VPT * V * 4;   /* <= 32 KB */ \
    launch_streaming(norm_grad_kernel<T, V, VPT, TPR>, parts, kThreads, kSmem, s, a);                               \
    break;                                                                                                          \
  }
  do {
    // two pieces per thread: what a row costs beside its elements (its place, the sums' meeting) is shared by 16 of them; with
    // one piece and twice the threads 103 us for forward and backward of 16384 x 2048 bfloat16, with two 94, with four 97
    if (vecs <= 32) B200_NORM(1, 32)
    if (vecs <= 64) B200_NORM(2, 32)
    if (vecs <= 128) B200_NORM(2, 64)
    if (vecs <= 256) B200_NORM(2, 128)
    if (vecs <= 512) B200_NORM(2, 256)
    if (vecs <= 1024) B200_NORM(2, 512)
    if (a.partial) {                             // first: dx may lie over dy
      launch_streaming(norm_grad_columns_kernel<T>, dim3((a.d.C + 255) / 256, parts), 256, 0, s, a);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
      ++*launches;
    }
    launch_streaming(norm_grad_long_kernel<T>, static_cast<unsigned>(rows), 512, 0, s, a);
  } while (0);
#undef B200_NORM
  if ((e = cudaGetLastError()) != cudaSuccess || !a.partial) return e;
  launch_chained(norm_params_kernel<T>, dim3((a.d.C + 31) / 32, 2), 512, 0, s, a, parts);
  ++*launches;
  return cudaGetLastError();
}

}  // namespace

// Parts of the parameters' sums: one per block, two blocks per SM once there are rows for them.
int norm_grad_parts(const b200conv_norm_desc& d) {
  const long long rows = d.sequences * d.length;
  return static_cast<int>(rows < 1 ? 1 : rows < 148 * kGradBlocks ? rows : 148 * kGradBlocks);
}

cudaError_t launch_layer_norm(const NormArgs& args, cudaStream_t s) {
  NormArgs a = args;
  if (flat(a.d, a.d.x, a.x) && flat(a.d, a.d.residual, a.residual) && flat(a.d, a.d.y, a.y) && flat(a.d, a.d.total, a.total)) {
    a.d.length *= a.d.sequences;
    a.d.sequences = 1;
  }
  const int dt = a.d.dtype, V = dt == B200CONV_F32 ? 4 : 8;
  const bool wide = a.d.C % V == 0 && rows_aligned(a.x, a.d.x, dt) && rows_aligned(a.residual, a.d.residual, dt) && rows_aligned(a.y, a.d.y, dt) &&
                    rows_aligned(a.total, a.d.total, dt) && aligned16({a.gamma, a.beta});
  if (dt == B200CONV_F32) return wide ? forward<float, 4>(a, s) : forward<float, 1>(a, s);
  if (dt == B200CONV_F16) return wide ? forward<__half, 8>(a, s) : forward<__half, 1>(a, s);
  return wide ? forward<__nv_bfloat16, 8>(a, s) : forward<__nv_bfloat16, 1>(a, s);
}

cudaError_t launch_layer_norm_grad(const NormArgs& args, int* launches, cudaStream_t s) {
  NormArgs a = args;
  if (flat(a.d, a.d.x, a.x) && flat(a.d, a.d.dy, a.dy) && flat(a.d, a.d.dtotal, a.dtotal) && flat(a.d, a.d.dx, a.dx)) {
    a.d.length *= a.d.sequences;
    a.d.sequences = 1;
  }
  const int dt = a.d.dtype, V = dt == B200CONV_F32 ? 4 : 8;
  const bool wide = a.d.C % V == 0 && rows_aligned(a.x, a.d.x, dt) && rows_aligned(a.dy, a.d.dy, dt) && rows_aligned(a.dtotal, a.d.dtotal, dt) &&
                    rows_aligned(a.dx, a.d.dx, dt);
  if (dt == B200CONV_F32) return wide ? backward<float, 4>(a, launches, s) : backward<float, 1>(a, launches, s);
  if (dt == B200CONV_F16) return wide ? backward<__half, 8>(a, launches, s) : backward<__half, 1>(a, launches, s);
  return wide ? backward<__nv_bfloat16, 8>(a, launches, s) : backward<__nv_bfloat16, 1>(a, launches, s);
}

}  // namespace b200
