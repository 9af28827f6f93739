// The selective state space scan: prompts and single tokens.
//
//   delta = dt + dt_bias (softplus of it),  h[t] = exp(delta A) h[t - 1] + delta x B[t],  y = (sum over n of C[t] h[t] + D x) silu(z)
//
// with N states per channel and B, C shared by the channels of a group.  One exponential per token, channel and state:
// 16 per clock and SM, 4.6e12 a second at 1.965 GHz, which bounds prompts (at N = 16 the tensors' 8 bytes per token and channel
// take a third of that time).  A block takes 128 / P channels and walks along its tokens in tiles of 32: x, dt and z come
// in 16-byte pieces that stay in registers, delta and delta x, B and C go through shared memory as float32, the states stay
// in registers, the sums over the states meet by shuffles four tokens at a time.
#include "selective_scan.cuh"

namespace b200 {
namespace {

constexpr int kTile = 32;                        // tokens
constexpr int kPitch = kTile + 4;                // of a channel's tokens in shared memory

// Reads a piece's B or C rows into [kTile][4 P] float32, zeros beyond N and beyond the piece.
template <typename T, int P>
__device__ __forceinline__ void load_states(const void* src, const b200conv_rows& r, long long base, long long tok, long long to, int group, int N,
                                            float* dst) {
  const T* p = static_cast<const T*>(src) + base * r.seq + 1LL * group * N;
  for (int i = threadIdx.x; i < kTile * 4 * P; i += kScanThreads) {
    const int t = i / (4 * P), n = i % (4 * P);
    dst[i] = n < N && tok + t < to ? to_float(p[(tok + t) * r.row + n]) : 0.f;
  }
}

// LOCAL: what a piece makes of zero states, and the sum of its deltas; else the outputs, from the states that the pieces before leave.
template <typename T, int V, int P, bool LOCAL>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(ScanArgs a) {
  constexpr int kWide = kScanThreads / P;        // channels of a block
  constexpr int kParts = (kTile * kWide / V + kScanThreads - 1) / kScanThreads;
  pdl_enter();
  __shared__ __align__(16) float sd[kWide][kPitch], su[kWide][kPitch], sy[LOCAL ? 1 : kWide][kPitch];
  __shared__ __align__(16) float sb[kTile * 4 * P], sc[LOCAL ? 1 : kTile * 4 * P];
  const int id = blockIdx.x / a.tiles;
  const ScanTile ct = scan_tile(a, blockIdx.x - id * a.tiles, kWide);
  const Piece p = piece_of(a, id);
  if (!p.valid || (LOCAL && id == p.last)) return;
  const int q = threadIdx.x % P, ch = threadIdx.x / P, c = ct.channel + ch;
  const bool mine = ch < ct.channels;
  const int N = a.d.N;
  float A[4], h[4], sum = 0.f;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int n = 4 * q + s;
    A[s] = mine && n < N ? scaled_decay(a.A[1LL * c * N + n]) : 0.f;
    h[s] = 0.f;
    if (!LOCAL && a.initial && mine && n < N) h[s] = a.initial[(1LL * p.seq * a.d.C + c) * N + n];
  }
  if (!LOCAL && mine)
    for (int j = p.first; j < id; ++j) {         // what the pieces before this one made of it
      const float all = a.piece_sum[1LL * j * a.d.C + c];
      const float4 f = *reinterpret_cast<const float4*>(a.piece_state + (1LL * j * a.d.C + c) * 4 * P + 4 * q);
      h[0] = exp2_fast(A[0] * all) * h[0] + f.x;
      h[1] = exp2_fast(A[1] * all) * h[1] + f.y;
      h[2] = exp2_fast(A[2] * all) * h[2] + f.z;
      h[3] = exp2_fast(A[3] * all) * h[3] + f.w;
    }
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + ct.channel;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + ct.channel;
  const T* z = a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + ct.channel : nullptr;
  T* y = LOCAL ? nullptr : static_cast<T*>(a.y) + p.base * a.d.y.seq + ct.channel;
  for (long long tok = p.from; tok < p.to; tok += kTile) {
    Pack<T, V> px[kParts], pz[kParts];
    __syncthreads();                             // the tile before has been read
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
      if (i >= kTile * kWide / V) break;
      const bool in = tok + t < p.to && cc < ct.channels;
      Pack<T, V> pd;
      if (in) {
        px[k].load(x + (tok + t) * a.d.x.row + cc);
        pd.load(dt + (tok + t) * a.d.dt.row + cc);
        if (!LOCAL && z) pz[k].load(z + (tok + t) * a.d.z.row + cc);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float d = 0.f, u = 0.f;
        if (in) {
          d = pd.get(e) + (a.dt_bias ? a.dt_bias[ct.channel + cc + e] : 0.f);
          if (a.d.softplus) d = softplus(d);
          u = d * px[k].get(e);
        }
        sd[cc + e][t] = d;
        su[cc + e][t] = u;
      }
    }
    load_states<T, P>(a.B, a.d.B, p.base, tok, p.to, ct.group, N, sb);
    if (!LOCAL) load_states<T, P>(a.C, a.d.Cm, p.base, tok, p.to, ct.group, N, sc);
    __syncthreads();
#pragma unroll 2
    for (int t = 0; t < kTile; t += 4) {
      const float4 d4 = *reinterpret_cast<const float4*>(&sd[ch][t]), u4 = *reinterpret_cast<const float4*>(&su[ch][t]);
      const float d[4] = {d4.x, d4.y, d4.z, d4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
      float out[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 b4 = *reinterpret_cast<const float4*>(sb + (t + k) * 4 * P + 4 * q);
        const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) h[s] = exp2_fast(d[k] * A[s]) * h[s] + u[k] * b[s];
        if (LOCAL) {
          sum += d[k];
        } else {
          const float4 c4 = *reinterpret_cast<const float4*>(sc + (t + k) * 4 * P + 4 * q);
          out[k] = h[0] * c4.x + h[1] * c4.y + h[2] * c4.z + h[3] * c4.w;
        }
      }
      if (!LOCAL) {
        const float r = lane_sums<P>(out);
        if (q < 4) sy[ch][t + q] = r;
      }
    }
    if (LOCAL) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int i = threadIdx.x + k * kScanThreads, t = i / (kWide / V), cc = i % (kWide / V) * V;
      if (i >= kTile * kWide / V || tok + t >= p.to || cc >= ct.channels) break;
      float out[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        out[e] = sy[cc + e][t];
        if (a.D) out[e] += a.D[ct.channel + cc + e] * px[k].get(e);
        if (z) {
          const float zv = pz[k].get(e);
          out[e] *= __fdividef(zv, 1.f + __expf(-zv));
        }
      }
      store_row<T, V>(y + (tok + t) * a.d.y.row + cc, out);
    }
  }
  if (!mine) return;
  if (LOCAL) {
    *reinterpret_cast<float4*>(a.piece_state + (1LL * id * a.d.C + c) * 4 * P + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
    if (q == 0) a.piece_sum[1LL * id * a.d.C + c] = sum;
  } else if (a.final && id == p.last) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (4 * q + s < N) a.final[(1LL * p.seq * a.d.C + c) * N + 4 * q + s] = h[s];
  }
}

// One token of every sequence; the states are read, moved on and written where they lie.
template <typename T, int V, int P>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(ScanArgs a) {
  pdl_enter();
  const long long i = blockIdx.x * static_cast<long long>(kScanThreads / P) + threadIdx.x / P;
  const bool mine = i < a.d.sequences * a.d.C;
  const int q = threadIdx.x % P, N = a.d.N;
  const long long seq = mine ? i / a.d.C : 0;
  const int c = mine ? static_cast<int>(i - seq * a.d.C) : 0, group = c / (a.d.C / a.d.groups);
  float d = 0.f, x = 0.f, y = 0.f;
  if (mine) {
    d = to_float(static_cast<const T*>(a.dt)[seq * a.d.dt.seq + c]) + (a.dt_bias ? a.dt_bias[c] : 0.f);
    if (a.d.softplus) d = softplus(d);
    x = to_float(static_cast<const T*>(a.x)[seq * a.d.x.seq + c]);
    float* state = a.final + (seq * a.d.C + c) * N;
    const T* B = static_cast<const T*>(a.B) + seq * a.d.B.seq + 1LL * group * N;
    const T* C = static_cast<const T*>(a.C) + seq * a.d.Cm.seq + 1LL * group * N;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int n = 4 * q + s;
      if (n < N) {
        const float h = exp2_fast(d * scaled_decay(a.A[1LL * c * N + n])) * state[n] + d * x * to_float(B[n]);
        state[n] = h;
        y += h * to_float(C[n]);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < P; o <<= 1) y += __shfl_xor_sync(~0u, y, o);
  if (!mine || q) return;
  if (a.D) y += a.D[c] * x;
  if (a.z) {
    const float z = to_float(static_cast<const T*>(a.z)[seq * a.d.z.seq + c]);
    y *= __fdividef(z, 1.f + __expf(-z));
  }
  static_cast<T*>(a.y)[seq * a.d.y.seq + c] = from_float<T>(y);
}

}  // namespace

cudaError_t launch_selective_scan(const ScanArgs& args, int* launches, cudaStream_t s) {
  ScanArgs a = args;
  const int wide = kScanThreads / scan_lanes(a.d.N), per = a.d.C / a.d.groups;
  a.tiles = a.d.groups * ((per + wide - 1) / wide);
  const long long grid = 1LL * a.tiles * a.pieces;
  *launches = 1;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  return with_scan(a, wide_scan(a), [&](auto t, auto v, auto p) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, P = decltype(p)::value;
    if (a.piece_state) {
      launch_streaming(scan_kernel<T, V, P, true>, static_cast<unsigned>(grid), kScanThreads, 0, s, a);
      ++*launches;
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
    launch_streaming(scan_kernel<T, V, P, false>, static_cast<unsigned>(grid), kScanThreads, 0, s, a);
    return cudaGetLastError();
  });
}

cudaError_t launch_scan_step(const ScanArgs& a, cudaStream_t s) {
  const long long per = kScanThreads / scan_lanes(a.d.N), grid = (a.d.sequences * a.d.C + per - 1) / per;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  return with_scan(a, false, [&](auto t, auto v, auto p) {
    launch_streaming(scan_step_kernel<decltype(t), 1, decltype(p)::value>, static_cast<unsigned>(grid), kScanThreads, 0, s, a);
    return cudaGetLastError();
  });
}

int scan_state_slots(int N) { return 4 * scan_lanes(N); }

// Pieces of a call.  A sequence is cut where its channels alone leave SMs without work: cut, every exponential but those of the last
// pieces is taken twice.
void plan_scan_pieces(ScanArgs* a) {
  const long long longest = a->d.packed ? (a->d.longest > 0 && a->d.longest < a->d.length ? a->d.longest : a->d.length) : a->d.length;
  const int wide = kScanThreads / scan_lanes(a->d.N), per = a->d.C / a->d.groups;
  const long long tiles = 1LL * a->d.groups * ((per + wide - 1) / wide);
  const long long rows = a->d.packed ? a->d.length : a->d.sequences * a->d.length;
  long long piece = a->d.length;
  const long long even = a->d.packed ? (rows + longest - 1) / longest : a->d.sequences;     // sequences that work at the same time to the end
  if (tiles * even < 148 * 4) {
    const long long want = (148 * 8 + tiles - 1) / tiles;                                     // pieces of the whole call
    piece = (rows + want - 1) / want;
    piece = (piece + 63) / 64 * 64;
    if (piece < 128) piece = 128;
  }
  if (piece >= longest) piece = a->d.length > 0 ? a->d.length : 1;
  a->piece = static_cast<int>(piece);
  a->pieces_per_seq = static_cast<int>((a->d.length + piece - 1) / piece);
  a->pieces = static_cast<int>(a->d.packed ? a->d.sequences + a->d.length / piece : a->d.sequences * a->pieces_per_seq);
}

}  // namespace b200
