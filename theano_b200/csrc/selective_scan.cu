// The selective state space scan: prompts and single tokens.
//
//   delta = dt + dt_bias (softplus of it),  h[t] = exp(delta A) h[t - 1] + delta x B[t],  y = (sum over n of C[t] h[t] + D x) silu(z)
//
// with N states per channel and B, C shared by the channels of a group.  One exponential per token, channel and state, two where a
// sequence is cut into pieces: 16 per clock and SM, 4.6e12 a second at 1.965 GHz, which bounds prompts (at N = 16 the tensors' 8
// bytes per token and channel take a third of that time).  So a lane holds all states of a channel, which makes everything else a
// token costs (its loads, softplus, gate) as cheap per state as it gets, two states go through the polynomial instead of the special
// function unit, and the rest runs on packed pairs.  8192 tokens, 2048 channels, 16 states, bfloat16: 181 us in 37 pieces.
#include "selective_scan.cuh"

#include <algorithm>

namespace b200 {
namespace {

// A lane per channel (P lanes where there are more than 16 states): S states in registers, so that what a token costs beside the decays
// is shared by all of them; the rows of B and C, the same for all lanes, come from shared memory as float32.
constexpr int kScanBlocks = 4;                   // of an SM: 16 warps, 128 registers a thread

// ASYNC: x, dt and z of 16-bit tensors on their boundaries come by asynchronous copies, a tile ahead, in 16 bytes (181 us, by loads
// of two bytes per lane 190: no addresses per token, no registers for tokens on their way).  Float32 tiles of 16 tokens would take 52 KB
// of shared memory, more than the 48 KB that a kernel may declare; they come by loads of four bytes.
template <typename T, int S, int P, bool WIDE, bool LOCAL, bool ASYNC>
__global__ void __launch_bounds__(kScanThreads, S * P <= 32 ? kScanBlocks : 1) scan_lane_kernel(ScanArgs a) {
  constexpr int NS = S * P, kWide = kScanThreads / P, kTokens = ASYNC && NS <= 32 ? 16 : tile_tokens(NS);
  constexpr int kGroup = LOCAL ? 8 : 4;          // tokens whose x, dt and z a lane has in flight
  using Rows = StateRows<T, NS, WIDE, !LOCAL, kTokens>;
  pdl_enter();
  __shared__ __align__(16) float st[2][(LOCAL ? 1 : 2) * kTokens * NS];
  constexpr int kArrays = LOCAL ? 2 : 3;
  __shared__ __align__(16) T rows_in[ASYNC ? 2 : 1][ASYNC ? kArrays : 1][ASYNC ? kTokens : 1][ASYNC ? kWide : 8];
  const int id = blockIdx.x / a.tiles;
  const ScanTile ct = scan_tile(a, blockIdx.x - id * a.tiles, kWide);
  const Piece p = piece_of(a, id);
  if (!p.valid || (LOCAL && id == p.last)) return;
  const int q = threadIdx.x % P, ch = threadIdx.x / P, c = ct.channel + ch, N = a.d.N;
  const bool mine = ch < ct.channels;
  Pair A[S / 2], h[S / 2];
  {
    float f[S];
#pragma unroll
    for (int s = 0; s < S; ++s) f[s] = mine && q * S + s < N ? scaled_decay(a.A[1LL * c * N + q * S + s]) : 0.f;
#pragma unroll
    for (int s = 0; s < S / 2; ++s) A[s] = Pair(f[2 * s], f[2 * s + 1]);
#pragma unroll
    for (int s = 0; s < S; ++s) f[s] = !LOCAL && a.initial && mine && q * S + s < N ? a.initial[(1LL * p.seq * a.d.C + c) * N + q * S + s] : 0.f;
#pragma unroll
    for (int s = 0; s < S / 2; ++s) h[s] = Pair(f[2 * s], f[2 * s + 1]);
  }
  if (!LOCAL && mine)
#pragma unroll 4
    for (int j = p.first; j < id; ++j) {         // what the pieces before this one made of it
      const float sum = a.piece_sum[1LL * j * a.d.C + c], all = any_of(h) ? sum : 0.f;
      const float4* f = reinterpret_cast<const float4*>(a.piece_state + (1LL * j * a.d.C + c) * NS + q * S);
#pragma unroll
      for (int s = 0; s < S / 4; ++s) {
        const float4 v = f[s];
        h[2 * s] = fma2(exp2_pair(mul2(A[2 * s], Pair(all, all))), h[2 * s], Pair(v.x, v.y));
        h[2 * s + 1] = fma2(exp2_pair(mul2(A[2 * s + 1], Pair(all, all))), h[2 * s + 1], Pair(v.z, v.w));
      }
    }
  const float bias = mine && a.dt_bias ? a.dt_bias[c] : 0.f, D = mine && a.D ? a.D[c] : 0.f;
  // lanes without a channel read the block's last one and write nothing
  const int cr = mine ? c : ct.channel + ct.channels - 1;
  const long long xr = a.d.x.row, dr = a.d.dt.row, zr = a.d.z.row, yr = a.d.y.row;
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + p.from * xr + cr;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + p.from * dr + cr;
  const T* z = !LOCAL && a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + p.from * zr + cr : nullptr;
  T* y = LOCAL ? nullptr : static_cast<T*>(a.y) + p.base * a.d.y.seq + p.from * yr + cr;
  const T* B = static_cast<const T*>(a.B) + p.base * a.d.B.seq + 1LL * ct.group * N;
  const T* C = static_cast<const T*>(a.C) + p.base * a.d.Cm.seq + 1LL * ct.group * N;
  T nx[kGroup], nd[kGroup], nz[kGroup];
  auto copy_tile = [&](long long tile, int turn) {
    if constexpr (ASYNC) {
      constexpr int kVec = 16 / sizeof(T), kRow = kWide / kVec;
      const int n = p.to - tile < kTokens ? static_cast<int>(p.to - tile) : kTokens;
#pragma unroll
      for (int w = 0; w < kArrays; ++w) {
        const void* base = w == 0 ? a.x : w == 1 ? a.dt : a.z;
        const b200conv_rows& r = w == 0 ? a.d.x : w == 1 ? a.d.dt : a.d.z;
        if (!base) continue;
        const T* src = static_cast<const T*>(base) + p.base * r.seq + tile * r.row + ct.channel;
#pragma unroll
        for (int i = threadIdx.x; i < kTokens * kRow; i += kScanThreads) {
          const int t = i / kRow, cc = i % kRow * kVec;
          if (t < n && cc < ct.channels) copy_async(&rows_in[turn][w][t][cc], src + t * r.row + cc);
        }
      }
      copies_issued();
    }
  };
  auto fetch = [&](int left) {                   // the next tokens of the piece, of which there are `left`
    if (ASYNC) return;
    if (left >= kGroup) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        nx[k] = x[k * xr];
        nd[k] = dt[k * dr];
        if (z) nz[k] = z[k * zr];
      }
    } else {
#pragma unroll
      for (int k = 0; k < kGroup; ++k)
        if (k < left) {
          nx[k] = x[k * xr];
          nd[k] = dt[k * dr];
          if (z) nz[k] = z[k * zr];
        }
    }
    x += kGroup * xr;
    dt += kGroup * dr;
    if (z) z += kGroup * zr;
  };
#pragma unroll
  for (int k = 0; k < kGroup; ++k) nx[k] = nd[k] = nz[k] = from_float<T>(0.f);
  Rows rows;
  rows.load(B, a.d.B.row, C, a.d.Cm.row, p.from, p.to, N);
  int left = static_cast<int>(p.to - p.from);    // tokens that have not been fetched
  if (ASYNC) copy_tile(p.from, 0);
  fetch(left);
  left -= kGroup;
  float sum = 0.f;
  int turn = 0;
  // kGroup tokens from shared memory at `at`, the tile's from t0 on; `live`: how many of them belong to the piece
  auto group = [&](const float* at, int t0, int live, auto whole) {
    if constexpr (ASYNC) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        nx[k] = rows_in[turn][0][t0 + k][ch];
        nd[k] = rows_in[turn][1][t0 + k][ch];
        if (!LOCAL && a.z) nz[k] = rows_in[turn][kArrays - 1][t0 + k][ch];
      }
    }
    float xv[kGroup], zv[kGroup], d[kGroup], u[kGroup];
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      xv[k] = to_float(nx[k]);
      if (!LOCAL) zv[k] = to_float(nz[k]);
      d[k] = to_float(nd[k]) + bias;
    }
    if (a.d.softplus)
#pragma unroll
      for (int k = 0; k < kGroup; ++k) d[k] = softplus(d[k]);
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      if (!decltype(whole)::value && k >= live) d[k] = xv[k] = 0.f;
      u[k] = d[k] * xv[k];
      if (LOCAL) sum += d[k];
    }
    fetch(left);
    left -= kGroup;
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      const float4* bs = reinterpret_cast<const float4*>(at + k * NS);
      const float4* cs = LOCAL ? bs : bs + kTokens * NS / 4;
      const Pair dd(d[k], d[k]), uu(u[k], u[k]);
      Pair out[2];
#pragma unroll
      for (int s = 0; s < S / 4; ++s) {
        const float4 b = bs[s];
        const Pair e0 = mul2(dd, A[2 * s]), e1 = mul2(dd, A[2 * s + 1]);
        h[2 * s] = fma2(2 * s < kPolyPairs ? exp2_poly(e0) : exp2_pair(e0), h[2 * s], mul2(uu, Pair(b.x, b.y)));
        h[2 * s + 1] = fma2(2 * s + 1 < kPolyPairs ? exp2_poly(e1) : exp2_pair(e1), h[2 * s + 1], mul2(uu, Pair(b.z, b.w)));
        if (!LOCAL) {
          const float4 w = cs[s];
          out[0] = s ? fma2(h[2 * s], Pair(w.x, w.y), out[0]) : mul2(h[0], Pair(w.x, w.y));
          out[1] = s ? fma2(h[2 * s + 1], Pair(w.z, w.w), out[1]) : mul2(h[1], Pair(w.z, w.w));
        }
      }
      if (LOCAL) continue;
      const float2 o = add2(out[0], out[1]).get();
      float r = o.x + o.y;
#pragma unroll
      for (int o = 1; o < P; o <<= 1) r += __shfl_xor_sync(~0u, r, o);
      r = fmaf(D, xv[k], r);
      if (z) r *= zv[k] * sigmoid(zv[k]);
      if (q == 0 && mine && (decltype(whole)::value || k < live)) y[k * yr] = from_float<T>(r);
    }
    if (!LOCAL) y += kGroup * yr;
  };
  for (long long tile = p.from; tile < p.to; tile += kTokens, turn ^= 1) {
    rows.store(st[turn]);
    if (ASYNC) copies_landed();
    __syncthreads();                             // the tile is there, and the one before the last has been read
    if (ASYNC && tile + kTokens < p.to) copy_tile(tile + kTokens, turn ^ 1);
    rows.load(B, a.d.B.row, C, a.d.Cm.row, tile + kTokens, p.to, N);
    const int n = p.to - tile < kTokens ? static_cast<int>(p.to - tile) : kTokens;
    const float* at = st[turn] + q * S;
    int t0 = 0;
    for (; t0 + kGroup <= n; t0 += kGroup) group(at + t0 * NS, t0, kGroup, std::true_type());
    if (t0 < n) group(at + t0 * NS, t0, n - t0, std::false_type());
  }
  if (!mine) return;
  if (LOCAL) {
    float4* f = reinterpret_cast<float4*>(a.piece_state + (1LL * id * a.d.C + c) * NS + q * S);
#pragma unroll
    for (int s = 0; s < S / 4; ++s) {
      const float2 u = h[2 * s].get(), v = h[2 * s + 1].get();
      f[s] = make_float4(u.x, u.y, v.x, v.y);
    }
    if (q == 0) a.piece_sum[1LL * id * a.d.C + c] = sum;
  } else if (a.final && id == p.last) {
#pragma unroll
    for (int s = 0; s < S / 2; ++s) {
      const float2 u = h[s].get();
      const int n = q * S + 2 * s;
      float* f = a.final + (1LL * p.seq * a.d.C + c) * N;
      if (n < N) f[n] = u.x;
      if (n + 1 < N) f[n + 1] = u.y;
    }
  }
}

// One token of every sequence; the states are read, moved on and written where they lie, which is all that takes time once the work per
// channel is out of the way: P lanes share a channel, eight states each (four each: 27 us for 256 sequences of 2048 channels and 16
// states, eight 20).  QUADS: N is a multiple of four and all rows of states lie on their boundaries, so that they move in 16 bytes.
constexpr int kStepThreads = 128;
template <typename T, int P, bool QUADS>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(ScanArgs a) {
  constexpr int kWide = kStepThreads / P;
  pdl_enter();
  const int q = threadIdx.x % P, N = a.d.N, C = a.d.C, n0 = 8 * q;
  const unsigned seq = blockIdx.y;
  const int c = blockIdx.x * kWide + threadIdx.x / P;
  const bool mine = c < C;
  const int group = a.d.groups == 1 || !mine ? 0 : c / (C / a.d.groups);
  float h[8], A[8];
  Pack<T, 4> b[2], w[2];
  float d = 0.f, x = 0.f, z = 0.f;
  float* state = a.final + (1LL * seq * C + c) * N + n0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    b[j].clear();
    w[j].clear();
#pragma unroll
    for (int s = 0; s < 4; ++s) h[4 * j + s] = A[4 * j + s] = 0.f;
  }
  if (mine) {
    const float* decay = a.A + 1LL * c * N + n0;
    const T* B = static_cast<const T*>(a.B) + seq * a.d.B.seq + 1LL * group * N + n0;
    const T* Cm = static_cast<const T*>(a.C) + seq * a.d.Cm.seq + 1LL * group * N + n0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (n0 + 4 * j >= N) continue;
      if (QUADS) {
        const float4 v = reinterpret_cast<const float4*>(state)[j], u = reinterpret_cast<const float4*>(decay)[j];
        h[4 * j] = v.x; h[4 * j + 1] = v.y; h[4 * j + 2] = v.z; h[4 * j + 3] = v.w;
        A[4 * j] = u.x; A[4 * j + 1] = u.y; A[4 * j + 2] = u.z; A[4 * j + 3] = u.w;
        b[j].load(B + 4 * j);
        w[j].load(Cm + 4 * j);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (n0 + 4 * j + s < N) {
            h[4 * j + s] = state[4 * j + s];
            A[4 * j + s] = decay[4 * j + s];
            b[j].e[s] = B[4 * j + s];
            w[j].e[s] = Cm[4 * j + s];
          }
      }
    }
    d = to_float(static_cast<const T*>(a.dt)[seq * a.d.dt.seq + c]) + (a.dt_bias ? a.dt_bias[c] : 0.f);
    x = to_float(static_cast<const T*>(a.x)[seq * a.d.x.seq + c]);
    if (a.z) z = to_float(static_cast<const T*>(a.z)[seq * a.d.z.seq + c]);
  }
  if (a.d.softplus) d = softplus(d);
  const float u = d * x;
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = exp2_fast(d * scaled_decay(A[i])) * h[i] + u * b[i / 4].get(i % 4);
    if (n0 + i < N) y += h[i] * w[i / 4].get(i % 4);
  }
#pragma unroll
  for (int o = 1; o < P; o <<= 1) y += __shfl_xor_sync(~0u, y, o);
  if (!mine) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (n0 + 4 * j >= N) break;
    if (QUADS) {
      reinterpret_cast<float4*>(state)[j] = make_float4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (n0 + 4 * j + s < N) state[4 * j + s] = h[4 * j + s];
    }
  }
  if (q) return;
  if (a.D) y = fmaf(a.D[c], x, y);
  if (a.z) y *= z * sigmoid(z);
  static_cast<T*>(a.y)[seq * a.d.y.seq + c] = from_float<T>(y);
}

}  // namespace

template <typename T, int S, int P, bool WIDE, bool ASYNC>
cudaError_t run_lanes(ScanArgs a, int* launches, cudaStream_t s) {
  const int wide = kScanThreads / P, per = a.d.C / a.d.groups;
  a.tiles = a.d.groups * ((per + wide - 1) / wide);
  const long long grid = 1LL * a.tiles * a.pieces;
  if (grid >= INT32_MAX) return cudaErrorInvalidValue;
  *launches = 1;
  if (a.piece_state) {
    launch_streaming(scan_lane_kernel<T, S, P, WIDE, true, ASYNC>, static_cast<unsigned>(grid), kScanThreads, 0, s, a);
    ++*launches;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  launch_streaming(scan_lane_kernel<T, S, P, WIDE, false, ASYNC>, static_cast<unsigned>(grid), kScanThreads, 0, s, a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t run_type(const ScanArgs& a, int* launches, cudaStream_t s) {
  const int N = a.d.N;
  const bool wide = N % (16 / sizeof(T)) == 0 && rows_aligned(a.B, a.d.B, a.d.dtype) && rows_aligned(a.C, a.d.Cm, a.d.dtype);
  // channels of a block in whole 16-byte pieces
  const bool async = sizeof(T) == 2 && N <= 32 && wide && a.d.C / a.d.groups % 8 == 0 && rows_aligned(a.x, a.d.x, a.d.dtype) &&
                     rows_aligned(a.dt, a.d.dt, a.d.dtype) && rows_aligned(a.z, a.d.z, a.d.dtype);
  if constexpr (sizeof(T) == 2) {
    if (async && N <= 8) return run_lanes<T, 8, 1, true, true>(a, launches, s);
    if (async && N <= 16) return run_lanes<T, 16, 1, true, true>(a, launches, s);
    if (async) return run_lanes<T, 16, 2, true, true>(a, launches, s);
  }
#define B200_LANES(S, P) if (N <= S * P) return wide ? run_lanes<T, S, P, true, false>(a, launches, s) : run_lanes<T, S, P, false, false>(a, launches, s);
  B200_LANES(8, 1) B200_LANES(16, 1) B200_LANES(16, 2) B200_LANES(16, 4) B200_LANES(16, 8)
#undef B200_LANES
  return cudaErrorInvalidValue;
}

cudaError_t launch_selective_scan(const ScanArgs& a, int* launches, cudaStream_t s) {
  if (a.d.dtype == B200CONV_F32) return run_type<float>(a, launches, s);
  return a.d.dtype == B200CONV_F16 ? run_type<__half>(a, launches, s) : run_type<__nv_bfloat16>(a, launches, s);
}

template <typename T, int P, bool QUADS>
cudaError_t run_step(const ScanArgs& a, int* launches, cudaStream_t s) {
  const int wide = kStepThreads / P;
  const unsigned blocks = static_cast<unsigned>((a.d.C + wide - 1) / wide);
  for (int64_t first = 0; first < a.d.sequences; first += 65535) {
    ScanArgs b = a;
    const unsigned n = static_cast<unsigned>(a.d.sequences - first < 65535 ? a.d.sequences - first : 65535);
    auto on = [&](const void* p, long long stride) { return p ? static_cast<const T*>(p) + first * stride : nullptr; };
    b.x = on(a.x, a.d.x.seq); b.dt = on(a.dt, a.d.dt.seq); b.z = on(a.z, a.d.z.seq); b.B = on(a.B, a.d.B.seq); b.C = on(a.C, a.d.Cm.seq);
    b.y = const_cast<T*>(on(a.y, a.d.y.seq));
    b.final = a.final + first * a.d.C * a.d.N;
    launch_streaming(scan_step_kernel<T, P, QUADS>, dim3(blocks, n), kStepThreads, 0, s, b);
    ++*launches;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <typename T>
cudaError_t run_step_type(const ScanArgs& a, int* launches, cudaStream_t s) {
  const int N = a.d.N;
  const size_t quad = 4 * sizeof(T);
  auto whole = [&](const void* p, const b200conv_rows& r) { return reinterpret_cast<uintptr_t>(p) % quad == 0 && r.seq * sizeof(T) % quad == 0; };
  const bool quads = N % 4 == 0 && aligned16({a.final, a.A}) && whole(a.B, a.d.B) && whole(a.C, a.d.Cm);
#define B200_LANES(P) if (N <= 8 * P) return quads ? run_step<T, P, true>(a, launches, s) : run_step<T, P, false>(a, launches, s);
  B200_LANES(1) B200_LANES(2) B200_LANES(4) B200_LANES(8) B200_LANES(16)
#undef B200_LANES
  return cudaErrorInvalidValue;
}

cudaError_t launch_scan_step(const ScanArgs& a, int* launches, cudaStream_t s) {
  *launches = 0;
  if (a.d.dtype == B200CONV_F32) return run_step_type<float>(a, launches, s);
  return a.d.dtype == B200CONV_F16 ? run_step_type<__half>(a, launches, s) : run_step_type<__nv_bfloat16>(a, launches, s);
}

int scan_state_slots(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : 128; }

// The cut of a call whose pieces take `tiles` blocks each, on a device that holds `slots` of them at a time: the number of pieces that
// ends soonest, counted in tokens one after the other, rounds of blocks times a piece's tokens and some for its start.  Half-filled
// last rounds cost most: 4 sequences of 2048 tokens and 2048 channels, gradients in 4 pieces each on 256 of 296 slots 861 us, in 9
// pieces in two rounds 752 us.
void cut_pieces(ScanArgs* a, long long tiles, long long slots) {
  const long long length = a->d.length, sequences = a->d.sequences, kStart = 24;
  const long long longest = a->d.packed && a->d.longest > 0 && a->d.longest < length ? a->d.longest : length;
  long long best = -1, piece = length;
  for (long long m = 1; m <= 256; ++m) {
    const long long size = ((longest + m - 1) / m + 3) / 4 * 4;
    if (m > 1 && size < 32) break;
    // packed: windows of `size` rows, and a piece more for each sequence that begins inside of one
    const long long blocks = tiles * (a->d.packed ? length / size + sequences : sequences * ((length + size - 1) / size));
    if (m > 1 && blocks > 3 * slots) break;
    // a cut sequence is walked twice, the first time for its ends alone
    const long long cost = (blocks + slots - 1) / slots * (size + kStart) * (m > 1 ? 7 : 4);
    if (best < 0 || cost < best) {
      best = cost;
      piece = m > 1 ? size : length;
    }
  }
  piece = std::max<long long>(piece, 1);
  a->piece = static_cast<int>(piece);
  a->pieces_per_seq = static_cast<int>((length + piece - 1) / piece);
  a->pieces = static_cast<int>(a->d.packed ? sequences + length / piece : sequences * a->pieces_per_seq);
}

// Pieces of the forward call: cut, every exponential but those of the last pieces is taken twice.  Four blocks to an SM are counted in every
// form; over 32 states their registers (210 to 242) let two in.  Counted as two, some calls end sooner and some later: bfloat16, 4 x 2048
// tokens of 1024 channels and 64 states 567 -> 637 us, 8 x 1024 of 512 channels and 128 states 876 -> 686, float32 2000 of 2048 channels and 100
// states 905 -> 1003.
void plan_scan_pieces(ScanArgs* a) {
  const int lanes = a->d.N <= 16 ? 1 : scan_state_slots(a->d.N) / 16, wide = kScanThreads / lanes, per = a->d.C / a->d.groups;
  cut_pieces(a, 1LL * a->d.groups * ((per + wide - 1) / wide), 148 * kScanBlocks);
}

}  // namespace b200
