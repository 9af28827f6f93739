// Gradients of the selective state space scan.  With dy0 = dy silu(z) and lambda[t] the adjoint of h[t]:
//
//   lambda[t] = C[t] dy0[t] + a[t + 1] lambda[t + 1]   (a = exp(delta A);  the final state's gradient behind the last token)
//   through[t] = a[t] lambda[t] h[t - 1]
//   dx = delta sum_n(lambda B) + D dy0        ddelta = sum_n(through A) + x sum_n(lambda B)       ddt = ddelta softplus'
//   dB = sum over the group's channels of lambda delta x     dC = of dy0 h     dA = sum over tokens of through delta
//   dz = dy y0 silu'(z),  y0 = sum_n(C h) + D x               dinitial = a[first] lambda[first]
//
// A first kernel walks forward and leaves the states in front of every eighth token (and, where sequences are cut, what each
// piece makes of zero states and of a zero adjoint); the second walks backward in tiles of eight tokens, makes the eight states
// and decays of a tile again in registers and runs the adjoint over them.  Sums over the states meet by shuffles; dB and dC
// are kept per token and state in registers while the block goes through its channels, then meet over the block.
// Bound by arithmetic: 13 operations and an exponential per token, channel and state in the second kernel, 3 and an
// exponential in the first, against 24 bytes per token and channel.
#include "selective_scan.cuh"

namespace b200 {
namespace {

constexpr int kTrace = 32;                       // tokens of the forward walk's tiles
constexpr int kStep = 8;                         // tokens of the backward walk's tiles, and between kept states
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float silu_of(float z) { return __fdividef(z, 1.f + __expf(-z)); }

// Place of the state kept in front of a token: pieces overlap an eighth row at most, and each has a number of its own.
__device__ __forceinline__ long long kept_at(const ScanArgs& a, const Piece& p, int id, long long tok) {
  return (a.d.packed ? tok : p.base * a.d.length + tok) / kStep + id;
}

template <typename T, int P>
__device__ __forceinline__ void load_states(const void* src, const b200conv_rows& r, long long base, long long tok, long long to, int tokens, int group,
                                            int N, float* dst) {
  const T* p = static_cast<const T*>(src) + base * r.seq + 1LL * group * N;
  for (int i = threadIdx.x; i < tokens * 4 * P; i += kScanThreads) {
    const int t = i / (4 * P), n = i % (4 * P);
    dst[i] = n < N && tok + t < to ? to_float(p[(tok + t) * r.row + n]) : 0.f;
  }
}

// Forward walk.  CUT: from zero states, with the piece's own effect on states and adjoints; else from the initial states.
template <typename T, int V, int P, bool CUT>
__global__ void __launch_bounds__(kScanThreads) scan_trace_kernel(ScanArgs a) {
  constexpr int kWide = kScanThreads / P;
  constexpr int kParts = (kTrace * kWide / V + kScanThreads - 1) / kScanThreads;
  pdl_enter();
  __shared__ __align__(16) float4 in[kTrace][kWide];         // delta, delta x, dy0
  __shared__ __align__(16) float sb[kTrace * 4 * P], sc[CUT ? kTrace * 4 * P : 1];
  const int id = blockIdx.x / a.tiles;
  const ScanTile ct = scan_tile(a, blockIdx.x - id * a.tiles, kWide);
  const Piece p = piece_of(a, id);
  if (!p.valid) return;
  const int q = threadIdx.x % P, ch = threadIdx.x / P, c = ct.channel + ch, N = a.d.N;
  const bool mine = ch < ct.channels;
  float A[4], h[4], back[4], reach[4], sum = 0.f;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int n = 4 * q + s;
    A[s] = mine && n < N ? scaled_decay(a.A[1LL * c * N + n]) : 0.f;
    h[s] = !CUT && a.initial && mine && n < N ? a.initial[(1LL * p.seq * a.d.C + c) * N + n] : 0.f;
    back[s] = 0.f;
    reach[s] = 1.f;
  }
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + ct.channel;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + ct.channel;
  const T* z = CUT && a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + ct.channel : nullptr;
  const T* dy = CUT ? static_cast<const T*>(a.dy) + p.base * a.d.dy.seq + ct.channel : nullptr;
  for (long long tok = p.from; tok < p.to; tok += kTrace) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
      if (i >= kTrace * kWide / V) break;
      const bool inside = tok + t < p.to && cc < ct.channels;
      Pack<T, V> px, pd, pz, py;
      if (inside) {
        px.load(x + (tok + t) * a.d.x.row + cc);
        pd.load(dt + (tok + t) * a.d.dt.row + cc);
        if (CUT) py.load(dy + (tok + t) * a.d.dy.row + cc);
        if (z) pz.load(z + (tok + t) * a.d.z.row + cc);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside) {
          v.x = pd.get(e) + (a.dt_bias ? a.dt_bias[ct.channel + cc + e] : 0.f);
          if (a.d.softplus) v.x = softplus(v.x);
          v.y = v.x * px.get(e);
          if (CUT) v.z = z ? py.get(e) * silu_of(pz.get(e)) : py.get(e);
        }
        in[t][cc + e] = v;
      }
    }
    load_states<T, P>(a.B, a.d.B, p.base, tok, p.to, kTrace, ct.group, N, sb);
    if (CUT) load_states<T, P>(a.C, a.d.Cm, p.base, tok, p.to, kTrace, ct.group, N, sc);
    __syncthreads();
    const int n = p.to - tok < kTrace ? static_cast<int>(p.to - tok) : kTrace;
    for (int t0 = 0; t0 < n; t0 += kStep) {
      if (mine) {
        const long long at = kept_at(a, p, id, tok + t0) * a.d.C + c;
        *reinterpret_cast<float4*>(a.kept + at * 4 * P + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
        if (CUT && q == 0) a.kept_sum[at] = sum;
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const float4 v = in[t0 + k][ch];
        const float4 b = *reinterpret_cast<const float4*>(sb + (t0 + k) * 4 * P + 4 * q);
        const float bs[4] = {b.x, b.y, b.z, b.w};
        float cs[4];
        if (CUT) {
          const float4 w = *reinterpret_cast<const float4*>(sc + (t0 + k) * 4 * P + 4 * q);
          cs[0] = w.x; cs[1] = w.y; cs[2] = w.z; cs[3] = w.w;
          sum += v.x;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float d = exp2_fast(v.x * A[s]);
          h[s] = d * h[s] + v.y * bs[s];
          if (CUT) {
            reach[s] *= d;
            back[s] += reach[s] * (cs[s] * v.z);
          }
        }
      }
    }
  }
  if (!CUT || !mine) return;
  const long long at = 1LL * id * a.d.C + c;
  *reinterpret_cast<float4*>(a.piece_state + at * 4 * P + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<float4*>(a.piece_back + at * 4 * P + 4 * q) = make_float4(back[0], back[1], back[2], back[3]);
  if (q == 0) a.piece_sum[at] = sum;
}

// Sums of n values per lane over the lanes whose numbers differ in the bits of P, 2 P, ... 16; a lane keeps n / (32 / P) of
// them: those whose number has, at its highest bits, the lane's bits from 16 down to P.
template <int O, int P, int n>
__device__ __forceinline__ void fold_lanes(float* v) {
  if constexpr (O >= P) {
    const bool hi = threadIdx.x & O;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float keep = hi ? v[i + n / 2] : v[i], give = hi ? v[i] : v[i + n / 2];
      v[i] = keep + __shfl_xor_sync(~0u, give, O);
    }
    fold_lanes<O / 2, P, n / 2>(v);
  }
}

template <int P> struct GradShape {
  static constexpr int kPass = kScanThreads / P;                       // channels at a time
  static constexpr int kPasses = 4, kWide = kPass * kPasses;           // of a block
  static constexpr int kLeft = 64 / (32 / P);                          // values of dB and dC that a lane keeps
  static constexpr size_t kInputs = sizeof(float4) * kStep * kWide, kStates = sizeof(float) * 2 * kStep * 4 * P,
                          kCarry = sizeof(float4) * kPasses * kScanThreads, kSums = sizeof(float) * 4 * 2 * kStep * 4 * P;
  static constexpr size_t bytes(bool cut) { return kInputs + kStates + kCarry * (cut ? 3 : 2) + kSums; }
};

template <typename T, int V, int P, bool CUT>
__global__ void __launch_bounds__(kScanThreads) scan_grad_kernel(ScanArgs a) {
  using S = GradShape<P>;
  constexpr int kWide = S::kWide, kPass = S::kPass, kPasses = S::kPasses;
  constexpr int kParts = (kStep * kWide / V + kScanThreads - 1) / kScanThreads;
  pdl_enter();
  extern __shared__ __align__(16) unsigned char smem[];
  float4* io = reinterpret_cast<float4*>(smem);                                    // [kStep][kWide]: delta x, dy0, -, delta; then the sums over n
  float* sb = reinterpret_cast<float*>(smem + S::kInputs);                         // [kStep][4 P], B then C
  float* sc = sb + kStep * 4 * P;
  float4* carry = reinterpret_cast<float4*>(smem + S::kInputs + S::kStates);       // [kPasses][threads]: a[t + 1] lambda[t + 1]
  float4* da = carry + kPasses * kScanThreads;
  float4* before = da + kPasses * kScanThreads;                                    // CUT: the states in front of the piece
  float* meet = reinterpret_cast<float*>(smem + S::bytes(CUT) - S::kSums);         // [warps][2][kStep][4 P]
  const int id = blockIdx.x / a.tiles, tile = blockIdx.x - id * a.tiles;
  const ScanTile ct = scan_tile(a, tile, kWide);
  const Piece p = piece_of(a, id);
  const int q = threadIdx.x % P, N = a.d.N, tiles_per_group = a.tiles / a.d.groups;
  if (!p.valid) {
    clear_piece_sums<P>(a, id, ct);
    return;
  }
  for (int m = 0; m < kPasses; ++m) {
    const int ch = m * kPass + threadIdx.x / P, c = ct.channel + ch;
    float g[4] = {0.f, 0.f, 0.f, 0.f}, h[4] = {0.f, 0.f, 0.f, 0.f};
    if (ch < ct.channels) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = 4 * q + s;
        if (n >= N) continue;
        const long long at = (1LL * p.seq * a.d.C + c) * N + n;
        if (a.dfinal) g[s] = a.dfinal[at];
        if (CUT) {
          const float A = scaled_decay(a.A[1LL * c * N + n]);
          for (int j = p.last; j > id; --j) {
            const long long o = 1LL * j * a.d.C + c;
            g[s] = a.piece_back[o * 4 * P + n] + exp2_fast(A * a.piece_sum[o]) * g[s];
          }
          if (a.initial) h[s] = a.initial[at];
          for (int j = p.first; j < id; ++j) {
            const long long o = 1LL * j * a.d.C + c;
            h[s] = a.piece_state[o * 4 * P + n] + exp2_fast(A * a.piece_sum[o]) * h[s];
          }
        }
      }
    }
    carry[m * kScanThreads + threadIdx.x] = make_float4(g[0], g[1], g[2], g[3]);
    da[m * kScanThreads + threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (CUT) before[m * kScanThreads + threadIdx.x] = make_float4(h[0], h[1], h[2], h[3]);
  }
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + ct.channel;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + ct.channel;
  const T* z = a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + ct.channel : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + p.base * a.d.dy.seq + ct.channel;
  T* dx = static_cast<T*>(a.dx) + p.base * a.d.dx.seq + ct.channel;
  T* ddt = static_cast<T*>(a.ddt) + p.base * a.d.ddt.seq + ct.channel;
  T* dz = a.dz ? static_cast<T*>(a.dz) + p.base * a.d.dz.seq + ct.channel : nullptr;
  float sum_d[kParts][V], sum_b[kParts][V];
#pragma unroll
  for (int k = 0; k < kParts; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) sum_d[k][e] = sum_b[k][e] = 0.f;
  const long long steps = (p.to - p.from + kStep - 1) / kStep;
  for (long long tok = p.from + (steps - 1) * kStep; tok >= p.from; tok -= kStep) {
    Pack<T, V> px[kParts], pd[kParts], pz[kParts], py[kParts];
    __syncthreads();                             // the tile behind this one has been read
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
      if (i >= kStep * kWide / V) break;
      const bool inside = tok + t < p.to && cc < ct.channels;
      if (inside) {
        px[k].load(x + (tok + t) * a.d.x.row + cc);
        pd[k].load(dt + (tok + t) * a.d.dt.row + cc);
        py[k].load(dy + (tok + t) * a.d.dy.row + cc);
        if (z) pz[k].load(z + (tok + t) * a.d.z.row + cc);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside) {
          v.w = pd[k].get(e) + (a.dt_bias ? a.dt_bias[ct.channel + cc + e] : 0.f);
          if (a.d.softplus) v.w = softplus(v.w);
          v.x = v.w * px[k].get(e);
          v.y = z ? py[k].get(e) * silu_of(pz[k].get(e)) : py[k].get(e);
        }
        io[t * kWide + cc + e] = v;
      }
    }
    load_states<T, P>(a.B, a.d.B, p.base, tok, p.to, kStep, ct.group, N, sb);
    load_states<T, P>(a.C, a.d.Cm, p.base, tok, p.to, kStep, ct.group, N, sc);
    __syncthreads();
    float bc[64];                                // dB [token][state], then dC
#pragma unroll
    for (int i = 0; i < 64; ++i) bc[i] = 0.f;
#pragma unroll 1
    for (int m = 0; m < kPasses; ++m) {
      const int ch = m * kPass + threadIdx.x / P, c = ct.channel + ch;
      const bool mine = ch < ct.channels;
      float A[4], h0[4], h[kStep][4], d[kStep][4], delta[kStep], u[kStep], g[kStep];
      {
        float4 k4 = make_float4(0.f, 0.f, 0.f, 0.f), b4 = k4;
        float sum = 0.f;
        if (mine) {
          const long long at = kept_at(a, p, id, tok) * a.d.C + c;
          k4 = *reinterpret_cast<const float4*>(a.kept + at * 4 * P + 4 * q);
          if (CUT) sum = a.kept_sum[at];
        }
        if (CUT) b4 = before[m * kScanThreads + threadIdx.x];
        const float ks[4] = {k4.x, k4.y, k4.z, k4.w}, bs[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          A[s] = mine && 4 * q + s < N ? scaled_decay(a.A[1LL * c * N + 4 * q + s]) : 0.f;
          h0[s] = CUT ? ks[s] + exp2_fast(A[s] * sum) * bs[s] : ks[s];
        }
      }
#pragma unroll
      for (int t = 0; t < kStep; ++t) {
        const float4 v = io[t * kWide + ch], b = *reinterpret_cast<const float4*>(sb + t * 4 * P + 4 * q);
        const float bs[4] = {b.x, b.y, b.z, b.w};
        delta[t] = v.w; u[t] = v.x; g[t] = v.y;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          d[t][s] = exp2_fast(delta[t] * A[s]);
          h[t][s] = d[t][s] * (t ? h[t - 1][s] : h0[s]) + u[t] * bs[s];
        }
      }
      __syncwarp();                              // the sums take the place of these channels' inputs
      float4 cr = carry[m * kScanThreads + threadIdx.x], dr = da[m * kScanThreads + threadIdx.x];
      float ca[4] = {cr.x, cr.y, cr.z, cr.w}, dA[4] = {dr.x, dr.y, dr.z, dr.w};
#pragma unroll
      for (int t0 = kStep - 4; t0 >= 0; t0 -= 4) {
        float lb[4], ta[4], yy[4];
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          const int t = t0 + k;
          const float4 b = *reinterpret_cast<const float4*>(sb + t * 4 * P + 4 * q), w = *reinterpret_cast<const float4*>(sc + t * 4 * P + 4 * q);
          const float bs[4] = {b.x, b.y, b.z, b.w}, cs[4] = {w.x, w.y, w.z, w.w};
          lb[k] = ta[k] = yy[k] = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float lam = cs[s] * g[t] + ca[s];
            lb[k] += lam * bs[s];
            yy[k] += cs[s] * h[t][s];
            bc[t * 4 + s] += lam * u[t];
            bc[32 + t * 4 + s] += g[t] * h[t][s];
            ca[s] = d[t][s] * lam;
            const float through = ca[s] * (t ? h[t - 1][s] : h0[s]);
            ta[k] += through * A[s];
            dA[s] += through * delta[t];
          }
        }
        const float s1 = lane_sums<P>(lb), s2 = lane_sums<P>(ta), s3 = lane_sums<P>(yy);
        if (q < 4) {
          float4* to = io + (t0 + q) * kWide + ch;
          *reinterpret_cast<float2*>(to) = make_float2(s1, s2 * kLn2);
          to->z = s3;
        }
      }
      carry[m * kScanThreads + threadIdx.x] = make_float4(ca[0], ca[1], ca[2], ca[3]);
      da[m * kScanThreads + threadIdx.x] = make_float4(dA[0], dA[1], dA[2], dA[3]);
    }
    fold_lanes<16, P, 64>(bc);
    {
      // the number of the first value that this lane kept: its bits from 16 down to P, highest first
      int first = 0;
#pragma unroll
      for (int o = 16, half = 32; o >= P; o >>= 1, half >>= 1)
        if (threadIdx.x & o) first += half;
      float* out = meet + (threadIdx.x >> 5) * (2 * kStep * 4 * P);
#pragma unroll
      for (int i = 0; i < S::kLeft; ++i) {
        const int v = first + i, which = v >> 5, t = v >> 2 & 7, s = v & 3;
        out[(which * kStep + t) * 4 * P + 4 * q + s] = bc[i];
      }
    }
    __syncthreads();
    {
      float* out = a.partial_bc + ((static_cast<long long>(tile - ct.group * tiles_per_group) * a.rows + (a.d.packed ? tok : p.base * a.d.length + tok)) *
                                       a.d.groups + ct.group) * 2 * N;
      for (int i = threadIdx.x; i < 2 * kStep * 4 * P; i += kScanThreads) {
        const int n = i % (4 * P), t = i / (4 * P) % kStep, which = i / (4 * P * kStep);
        if (n >= N || tok + t >= p.to) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) v += meet[w * (2 * kStep * 4 * P) + i];
        out[(1LL * t * a.d.groups * 2 + which) * N + n] = v;
      }
    }
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
      if (i >= kStep * kWide / V || tok + t >= p.to || cc >= ct.channels) break;
      float ox[V], od[V], oz[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float4 v = io[t * kWide + cc + e];             // sum lambda B, sum through A, sum C h, delta
        const int c = ct.channel + cc + e;
        const float xv = px[k].get(e), dv = py[k].get(e), D = a.D ? a.D[c] : 0.f;
        float g = dv;
        if (z) {
          const float zv = pz[k].get(e), sg = __fdividef(1.f, 1.f + __expf(-zv));
          g = dv * silu_of(zv);
          oz[e] = dv * (v.z + D * xv) * sg * (1.f + zv * (1.f - sg));
        }
        ox[e] = v.w * v.x + D * g;
        od[e] = v.y + xv * v.x;
        if (a.d.softplus) od[e] *= __fdividef(1.f, 1.f + __expf(-(pd[k].get(e) + (a.dt_bias ? a.dt_bias[c] : 0.f))));
        sum_d[k][e] += g * xv;
        sum_b[k][e] += od[e];
      }
      store_row<T, V>(dx + (tok + t) * a.d.dx.row + cc, ox);
      store_row<T, V>(ddt + (tok + t) * a.d.ddt.row + cc, od);
      if (dz) store_row<T, V>(dz + (tok + t) * a.d.dz.row + cc, oz);
    }
  }
  // what is left per channel: dA and the gradient of the initial states from the lanes, dD and the bias's over the tile's tokens
  for (int m = 0; m < kPasses; ++m) {
    const int ch = m * kPass + threadIdx.x / P, c = ct.channel + ch;
    if (ch >= ct.channels) continue;
    const float4 dr = da[m * kScanThreads + threadIdx.x], cr = carry[m * kScanThreads + threadIdx.x];
    const float dA[4] = {dr.x, dr.y, dr.z, dr.w}, ca[4] = {cr.x, cr.y, cr.z, cr.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int n = 4 * q + s;
      if (n >= N) continue;
      a.partial_a[(1LL * id * a.d.C + c) * N + n] = dA[s];
      if (a.dinitial && id == p.first) a.dinitial[(1LL * p.seq * a.d.C + c) * N + n] = ca[s];
    }
  }
  __syncthreads();
  float2* sums = reinterpret_cast<float2*>(io);              // [kStep][kWide]
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
    if (i >= kStep * kWide / V) break;
#pragma unroll
    for (int e = 0; e < V; ++e) sums[t * kWide + cc + e] = make_float2(sum_d[k][e], sum_b[k][e]);
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < ct.channels; ch += kScanThreads) {
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int t = 0; t < kStep; ++t) {
      v.x += sums[t * kWide + ch].x;
      v.y += sums[t * kWide + ch].y;
    }
    a.partial_d[2LL * id * a.d.C + ct.channel + ch] = v.x;
    a.partial_d[(2LL * id + 1) * a.d.C + ct.channel + ch] = v.y;
  }
}

// dB and dC: the blocks that share a group's rows, in their order.
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(ScanArgs a, int tiles_per_group) {
  pdl_enter();
  const int N = a.d.N, wide = a.d.groups * 2 * N;
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= a.rows * wide) return;
  const long long row = i / wide;
  const int e = static_cast<int>(i - row * wide), n = e % N, which = e / N % 2, group = e / (2 * N);
  long long seq = 0, tok = row;
  if (!a.d.packed) {
    seq = row / a.d.length;
    tok = row - seq * a.d.length;
  } else {
    const long long lo = start_of(a.starts, 0, a.d.length), hi = start_of(a.starts, static_cast<int>(a.d.sequences), a.d.length);
    if (row < lo || row >= hi) return;           // rows of no sequence
  }
  float v = 0.f;
  for (int t = 0; t < tiles_per_group; ++t) v += a.partial_bc[(t * a.rows) * wide + i];
  const b200conv_rows& r = which ? a.d.dCm : a.d.dB;
  static_cast<T*>(which ? a.dC : a.dB)[seq * r.seq + tok * r.row + 1LL * group * N + n] = from_float<T>(v);
}

// dA, dD and the bias's gradient: the pieces in their order, 8 threads apart so that long batches do not wait for one sum.
__global__ void __launch_bounds__(256) scan_params_kernel(ScanArgs a) {
  pdl_enter();
  __shared__ float part[8][32];
  const long long wide = 1LL * a.d.C * a.d.N, all = wide + 2LL * a.d.C, i = blockIdx.x * 32LL + (threadIdx.x & 31);
  const int w = threadIdx.x >> 5;
  float v = 0.f;
  if (i < all)
    for (int p = w; p < a.pieces; p += 8) v += i < wide ? a.partial_a[p * wide + i] : a.partial_d[2LL * p * a.d.C + (i - wide)];
  part[w][threadIdx.x & 31] = v;
  __syncthreads();
  if (w || i >= all) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += part[k][threadIdx.x & 31];
  if (i < wide) a.dA[i] = v;
  else if (i < wide + a.d.C) { if (a.dD) a.dD[i - wide] = v; }
  else if (a.ddt_bias) a.ddt_bias[i - wide - a.d.C] = v;
}

}  // namespace

int scan_grad_slots(int N) { return 4 * scan_lanes(N); }
int scan_grad_channels(int N) { return 4 * (kScanThreads / scan_lanes(N)); }
long long scan_kept(const ScanArgs& a) { return a.rows / kStep + a.pieces + 1; }

// Pieces of the gradient's call: three blocks per SM.  Being cut costs two operations per state in the forward walk.
void plan_grad_pieces(ScanArgs* a) {
  const long long longest = a->d.packed ? (a->d.longest > 0 && a->d.longest < a->d.length ? a->d.longest : a->d.length) : a->d.length;
  const int wide = scan_grad_channels(a->d.N), per = a->d.C / a->d.groups;
  const long long tiles = 1LL * a->d.groups * ((per + wide - 1) / wide);
  a->rows = a->d.packed ? a->d.length : a->d.sequences * a->d.length;
  const long long even = a->d.packed ? (a->rows + longest - 1) / longest : a->d.sequences;
  long long piece = a->d.length;
  if (tiles * even < 148 * 3) {
    const long long want = (148 * 3 + tiles - 1) / tiles;
    piece = (a->rows + want - 1) / want;
    piece = (piece + kTrace - 1) / kTrace * kTrace;
    if (piece < 2 * kTrace) piece = 2 * kTrace;
  }
  if (piece >= longest) piece = a->d.length;
  a->piece = static_cast<int>(piece);
  a->pieces_per_seq = static_cast<int>((a->d.length + piece - 1) / piece);
  a->pieces = static_cast<int>(a->d.packed ? a->d.sequences + a->d.length / piece : a->d.sequences * a->pieces_per_seq);
  a->tiles = static_cast<int>(tiles);
}

cudaError_t launch_scan_grad(const ScanArgs& args, int* launches, cudaStream_t s) {
  ScanArgs a = args;
  const bool cut = a.piece < a.d.length;
  const int P = scan_lanes(a.d.N), narrow = kScanThreads / P, per = a.d.C / a.d.groups;
  const int trace_tiles = a.d.groups * ((per + narrow - 1) / narrow), grad_tiles = a.tiles;
  if (1LL * trace_tiles * a.pieces >= INT32_MAX) return cudaErrorInvalidValue;
  cudaError_t e = with_scan(a, wide_scan(a), [&](auto t, auto v, auto p) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, L = decltype(p)::value;
    using S = GradShape<L>;
    static PerDeviceOnce setup;
    cudaError_t e = setup.ensure([&] {
      const cudaError_t e = cudaFuncSetAttribute(scan_grad_kernel<T, V, L, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(true));
      return e != cudaSuccess ? e : cudaFuncSetAttribute(scan_grad_kernel<T, V, L, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(false));
    });
    if (e != cudaSuccess) return e;
    a.tiles = trace_tiles;
    if (cut) launch_streaming(scan_trace_kernel<T, V, L, true>, trace_tiles * a.pieces, kScanThreads, 0, s, a);
    else launch_streaming(scan_trace_kernel<T, V, L, false>, trace_tiles * a.pieces, kScanThreads, 0, s, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    a.tiles = grad_tiles;
    if (cut) launch_streaming(scan_grad_kernel<T, V, L, true>, grad_tiles * a.pieces, kScanThreads, S::bytes(true), s, a);
    else launch_streaming(scan_grad_kernel<T, V, L, false>, grad_tiles * a.pieces, kScanThreads, S::bytes(false), s, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    const long long bc = a.rows * a.d.groups * 2 * a.d.N;
    if ((bc + 255) / 256 >= INT32_MAX) return cudaErrorInvalidValue;
    launch_streaming(scan_bc_kernel<T>, static_cast<unsigned>((bc + 255) / 256), 256, 0, s, a, grad_tiles / a.d.groups);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  *launches = 4;
  const long long all = 1LL * a.d.C * (a.d.N + 2);
  launch_streaming(scan_params_kernel, static_cast<unsigned>((all + 31) / 32), 256, 0, s, a);
  return cudaGetLastError();
}

}  // namespace b200
