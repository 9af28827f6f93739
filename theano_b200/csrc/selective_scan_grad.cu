// Gradients of the selective state space scan.  With dy0 = dy silu(z) and lambda[t] the adjoint of h[t]:
//
//   lambda[t] = C[t] dy0[t] + a[t + 1] lambda[t + 1]   (a = exp(delta A);  the final state's gradient behind the last token)
//   through[t] = a[t] lambda[t] h[t - 1]
//   dx = delta sum_n(lambda B) + D dy0        ddelta = sum_n(through A) + x sum_n(lambda B)       ddt = ddelta softplus'
//   dB = sum over the group's channels of lambda delta x     dC = of dy0 h     dA = sum over tokens of through delta
//   dz = dy y0 silu'(z),  y0 = sum_n(C h) + D x               dinitial = a[first] lambda[first]
//
// A first kernel walks forward and leaves the states in front of every fourth token (and, where sequences are cut, what each piece makes of
// zero states and of a zero adjoint).  The second walks backward: for four tokens at a time it makes their states again, in registers, and
// runs the adjoint over them.  Both have a lane per channel with its states, so that sums over the states cost nothing; what dB and dC
// add over the channels goes through shared memory, 32 values per lane and token.  4 x 2048 tokens, 2048 channels, 16 states, bfloat16:
// 160 us the first, 419 the second, 17 the sums over blocks and pieces.  The second takes 385 instructions, 106 accesses to shared
// memory (424 clocks of an SM quarter) and 36 exponentials (288) per token and warp and is bound by neither: with 250 registers two
// blocks fit an SM (one of cut float32 sequences, whose shared memory is 118 KB), and two warps per quarter leave 60 % of the issue slots
// empty.  Four states to a lane with sums by shuffles took 525 us at 3 blocks, eight states 567; limits of 168 registers spill 180 of them.
#include "selective_scan.cuh"

namespace b200 {
namespace {

constexpr int kStep = 8;                         // tokens of the backward walk's tiles
constexpr int kKeep = 4;                         // tokens between kept states
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kGradBlocks = 2;                   // of an SM

// Place of the states kept in front of a token: pieces overlap a fourth row at most, and each has a number of its own.
__device__ __forceinline__ long long kept_at(const ScanArgs& a, const Piece& p, int id, long long tok) {
  return (a.d.packed ? tok : p.base * a.d.length + tok) / kKeep + id;
}

// Forward walk.  CUT: from zero states, with the piece's own effect on states and adjoints; else from the initial states.
template <typename T, int S, int P, bool WIDE, bool CUT>
__global__ void __launch_bounds__(kScanThreads, S * P <= 32 ? (CUT ? 3 : 4) : 1) scan_trace_kernel(ScanArgs a) {
  constexpr int NS = S * P, kWide = kScanThreads / P, kTokens = tile_tokens(NS);
  using Rows = StateRows<T, NS, WIDE, CUT>;
  pdl_enter();
  __shared__ __align__(16) float st[2][(CUT ? 2 : 1) * kTokens * NS];
  const int id = blockIdx.x / a.tiles;
  const ScanTile ct = scan_tile(a, blockIdx.x - id * a.tiles, kWide);
  const Piece p = piece_of(a, id);
  if (!p.valid) return;
  const int q = threadIdx.x % P, ch = threadIdx.x / P, c = ct.channel + ch, N = a.d.N;
  const bool mine = ch < ct.channels;
  Pair A[S / 2], h[S / 2], back[S / 2], reach[S / 2];
  {
    float f[S];
#pragma unroll
    for (int s = 0; s < S; ++s) f[s] = mine && q * S + s < N ? scaled_decay(a.A[1LL * c * N + q * S + s]) : 0.f;
#pragma unroll
    for (int s = 0; s < S / 2; ++s) A[s] = Pair(f[2 * s], f[2 * s + 1]);
#pragma unroll
    for (int s = 0; s < S; ++s) f[s] = !CUT && a.initial && mine && q * S + s < N ? a.initial[(1LL * p.seq * a.d.C + c) * N + q * S + s] : 0.f;
#pragma unroll
    for (int s = 0; s < S / 2; ++s) {
      h[s] = Pair(f[2 * s], f[2 * s + 1]);
      back[s] = Pair(0.f, 0.f);
      reach[s] = Pair(1.f, 1.f);
    }
  }
  const float bias = mine && a.dt_bias ? a.dt_bias[c] : 0.f;
  // lanes without a channel read the block's last one and write nothing
  const int cr = mine ? c : ct.channel + ct.channels - 1;
  const long long xr = a.d.x.row, dr = a.d.dt.row, zr = a.d.z.row, yr = a.d.dy.row;
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + p.from * xr + cr;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + p.from * dr + cr;
  const T* z = CUT && a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + p.from * zr + cr : nullptr;
  const T* dy = CUT ? static_cast<const T*>(a.dy) + p.base * a.d.dy.seq + p.from * yr + cr : nullptr;
  const T* B = static_cast<const T*>(a.B) + p.base * a.d.B.seq + 1LL * ct.group * N;
  const T* C = static_cast<const T*>(a.C) + p.base * a.d.Cm.seq + 1LL * ct.group * N;
  T nx[kKeep], nd[kKeep], nz[kKeep], ny[kKeep];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) nx[k] = nd[k] = nz[k] = ny[k] = from_float<T>(0.f);
  auto fetch = [&](int left) {                   // the next tokens of the piece, of which there are `left`
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (k < left) {
        nx[k] = x[k * xr];
        nd[k] = dt[k * dr];
        if (CUT) ny[k] = dy[k * yr];
        if (z) nz[k] = z[k * zr];
      }
    x += kKeep * xr;
    dt += kKeep * dr;
    if (CUT) dy += kKeep * yr;
    if (z) z += kKeep * zr;
  };
  Rows rows;
  rows.load(B, a.d.B.row, C, a.d.Cm.row, p.from, p.to, N);
  int left = static_cast<int>(p.to - p.from);    // tokens that have not been fetched
  fetch(left);
  left -= kKeep;
  float sum = 0.f;
  int turn = 0;
  float4* kept = reinterpret_cast<float4*>(a.kept) + (kept_at(a, p, id, p.from) * (NS / 4) + q * (S / 4)) * a.d.C + c;
  float* kept_sum = CUT ? a.kept_sum + kept_at(a, p, id, p.from) * a.d.C + c : nullptr;
  for (long long tile = p.from; tile < p.to; tile += kTokens, turn ^= 1) {
    rows.store(st[turn]);
    __syncthreads();                             // the tile is there, and the one before the last has been read
    rows.load(B, a.d.B.row, C, a.d.Cm.row, tile + kTokens, p.to, N);
    const int n = p.to - tile < kTokens ? static_cast<int>(p.to - tile) : kTokens;
    for (int t0 = 0; t0 < n; t0 += kKeep) {
      if (mine) {
#pragma unroll
        for (int s = 0; s < S / 4; ++s) {
          const float2 u = h[2 * s].get(), v = h[2 * s + 1].get();
          kept[1LL * s * a.d.C] = make_float4(u.x, u.y, v.x, v.y);
        }
        if (CUT && q == 0) *kept_sum = sum;
      }
      kept += 1LL * (NS / 4) * a.d.C;
      if (CUT) kept_sum += a.d.C;
      float d[kKeep], u[kKeep], g[kKeep];
#pragma unroll
      for (int k = 0; k < kKeep; ++k) {
        d[k] = to_float(nd[k]) + bias;
        if (a.d.softplus) d[k] = softplus(d[k]);
        float xv = to_float(nx[k]);
        if (t0 + k >= n) d[k] = xv = 0.f;
        u[k] = d[k] * xv;
        if (CUT) {
          const float zv = to_float(nz[k]);
          g[k] = to_float(ny[k]);
          if (z) g[k] *= zv * sigmoid(zv);
          if (t0 + k >= n) g[k] = 0.f;
        }
      }
      fetch(left);
      left -= kKeep;
#pragma unroll
      for (int k = 0; k < kKeep; ++k) {
        const float4* bs = reinterpret_cast<const float4*>(st[turn] + (t0 + k) * NS + q * S);
        const float4* cs = bs + kTokens * NS / 4;
        const Pair dd(d[k], d[k]), uu(u[k], u[k]), gg(CUT ? g[k] : 0.f, CUT ? g[k] : 0.f);
        if (CUT) sum += d[k];
#pragma unroll
        for (int s = 0; s < S / 4; ++s) {
          const float4 b = bs[s];
          const Pair e0 = mul2(dd, A[2 * s]), e1 = mul2(dd, A[2 * s + 1]);
          // the first states by polynomial as in the forward call, for its precision: the special function unit's results near 1 are 2e-8
          // too small on average, which slow states add up (dA of 9 x 969 tokens off by 8e-7, with it alone by 1.4e-6; 756 us, 748)
          const Pair a0 = 2 * s < kPolyPairs ? exp2_poly(e0) : exp2_pair(e0), a1 = 2 * s + 1 < kPolyPairs ? exp2_poly(e1) : exp2_pair(e1);
          h[2 * s] = fma2(a0, h[2 * s], mul2(uu, Pair(b.x, b.y)));
          h[2 * s + 1] = fma2(a1, h[2 * s + 1], mul2(uu, Pair(b.z, b.w)));
          if (CUT) {
            const float4 w = cs[s];
            reach[2 * s] = mul2(reach[2 * s], a0);
            reach[2 * s + 1] = mul2(reach[2 * s + 1], a1);
            back[2 * s] = fma2(reach[2 * s], mul2(Pair(w.x, w.y), gg), back[2 * s]);
            back[2 * s + 1] = fma2(reach[2 * s + 1], mul2(Pair(w.z, w.w), gg), back[2 * s + 1]);
          }
        }
      }
    }
  }
  if (!CUT || !mine) return;
  const long long at = (1LL * id * a.d.C + c) * NS + q * S;
#pragma unroll
  for (int s = 0; s < S / 4; ++s) {
    const float2 u = h[2 * s].get(), v = h[2 * s + 1].get(), w = back[2 * s].get(), y = back[2 * s + 1].get();
    reinterpret_cast<float4*>(a.piece_state + at)[s] = make_float4(u.x, u.y, v.x, v.y);
    reinterpret_cast<float4*>(a.piece_back + at)[s] = make_float4(w.x, w.y, y.x, y.y);
  }
  if (q == 0) a.piece_sum[1LL * id * a.d.C + c] = sum;
}

// Shared memory of the backward walk.
template <typename T, int P, bool CUT> struct GradShape {
  static constexpr int NS = 16 * P, kWide = kScanThreads / P, kWarps = kScanThreads / 32;
  static constexpr int kLine = 36;                                     // floats of a lane's 32 products: 8 lanes' pieces of 16 bytes meet all banks
  T rows[2][4][kStep][kWide];                                          // x, dt, dy, z of a tile
  float states[2][2][kStep][NS];                                       // its B and C
  float4 kept[2][kStep / kKeep][4][kScanThreads];                      // the states in front of its first and fifth token
  float kept_sum[2][kStep / kKeep][CUT ? kWide : 1];
  float lines[kWarps][2][32][kLine];                                   // what the lanes of a warp have for dB and dC of a token
  float sums[kWarps][kStep][32 * P];                                   // their sums
  float before[CUT ? kScanThreads : 1][CUT ? 20 : 1];                  // the states in front of the piece
};

// Sum of the lines of the 32 / P channels of a warp: 32 P values, to `out`.
template <int P, int kLine>
__device__ __forceinline__ void sum_lines(const float (*line)[kLine], float* out) {
  const int lane = threadIdx.x & 31;
  constexpr int kParts = P < 4 ? 4 / P : 1, kQuads = P > 4 ? P / 4 : 1, kRows = 32 / P / kParts;
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    const int quad = lane % (32 / kParts) + 32 * j, q = quad / 8, v = quad % 8 * 4, part = lane / (32 / kParts);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float4 f = *reinterpret_cast<const float4*>(&line[(part * kRows + r) * P + q][v]);
      s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
    }
    float* to = out + q * 32 + v;
    if (kParts == 1) {
      *reinterpret_cast<float4*>(to) = s;
    } else {
      // the parts change places: a lane keeps two of the four values, then one
      const bool hi = lane & 16;
      float a = hi ? s.z : s.x, b = hi ? s.w : s.y;
      a += __shfl_xor_sync(~0u, hi ? s.x : s.z, 16);
      b += __shfl_xor_sync(~0u, hi ? s.y : s.w, 16);
      to += hi ? 2 : 0;
      if (kParts == 2) {
        *reinterpret_cast<float2*>(to) = make_float2(a, b);
      } else {
        const bool up = lane & 8;
        const float r = (up ? b : a) + __shfl_xor_sync(~0u, up ? a : b, 8);
        to[up ? 1 : 0] = r;
      }
    }
  }
}

template <typename T, bool WIDE, int P, bool CUT>
__global__ void __launch_bounds__(kScanThreads, P == 1 ? kGradBlocks : 1) scan_grad_kernel(ScanArgs a) {
  using Shared = GradShape<T, P, CUT>;
  constexpr int NS = Shared::NS, kWide = Shared::kWide, kLine = Shared::kLine, kVec = 16 / sizeof(T);
  pdl_enter();
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int id = blockIdx.x / a.tiles, block = blockIdx.x - id * a.tiles;
  const ScanTile ct = scan_tile(a, block, kWide);
  const Piece p = piece_of(a, id);
  const int q = threadIdx.x % P, ch = threadIdx.x / P, c = ct.channel + ch, N = a.d.N, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks_per_group = a.tiles / a.d.groups;
  if (!p.valid) {
    clear_piece_sums(a, id, ct, kScanThreads);
    return;
  }
  const bool mine = ch < ct.channels;
  Pair A[8], ca[8], dA[8];                       // decays, a[t + 1] lambda[t + 1], sums of through delta
  {
    float A_[16], g[16], h[16];
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      const int n = q * 16 + s;
      const bool have = mine && n < N;
      const long long at = (1LL * p.seq * a.d.C + c) * N + n;
      A_[s] = have ? scaled_decay(a.A[1LL * c * N + n]) : 0.f;
      g[s] = have && a.dfinal ? a.dfinal[at] : 0.f;
      h[s] = CUT && have && a.initial ? a.initial[at] : 0.f;
    }
    if (CUT && mine) {
#pragma unroll 4
      for (int j = p.last; j > id; --j) {
        const long long o = 1LL * j * a.d.C + c;
        const float4* b = reinterpret_cast<const float4*>(a.piece_back + o * NS + q * 16);
        const float all = a.piece_sum[o];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float4 v = b[s];
          g[4 * s] = v.x + exp2_fast(A_[4 * s] * all) * g[4 * s];
          g[4 * s + 1] = v.y + exp2_fast(A_[4 * s + 1] * all) * g[4 * s + 1];
          g[4 * s + 2] = v.z + exp2_fast(A_[4 * s + 2] * all) * g[4 * s + 2];
          g[4 * s + 3] = v.w + exp2_fast(A_[4 * s + 3] * all) * g[4 * s + 3];
        }
      }
#pragma unroll 4
      for (int j = p.first; j < id; ++j) {
        const long long o = 1LL * j * a.d.C + c;
        const float4* b = reinterpret_cast<const float4*>(a.piece_state + o * NS + q * 16);
        const float all = a.piece_sum[o];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float4 v = b[s];
          h[4 * s] = v.x + exp2_fast(A_[4 * s] * all) * h[4 * s];
          h[4 * s + 1] = v.y + exp2_fast(A_[4 * s + 1] * all) * h[4 * s + 1];
          h[4 * s + 2] = v.z + exp2_fast(A_[4 * s + 2] * all) * h[4 * s + 2];
          h[4 * s + 3] = v.w + exp2_fast(A_[4 * s + 3] * all) * h[4 * s + 3];
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      A[s] = Pair(A_[2 * s], A_[2 * s + 1]);
      ca[s] = Pair(g[2 * s], g[2 * s + 1]);
      dA[s] = Pair(0.f, 0.f);
      if (CUT) {
        sh.before[threadIdx.x][2 * s] = h[2 * s];
        sh.before[threadIdx.x][2 * s + 1] = h[2 * s + 1];
      }
    }
  }
  const float bias = mine && a.dt_bias ? a.dt_bias[c] : 0.f, D = mine && a.D ? a.D[c] : 0.f;
  const T* x = static_cast<const T*>(a.x) + p.base * a.d.x.seq + ct.channel;
  const T* dt = static_cast<const T*>(a.dt) + p.base * a.d.dt.seq + ct.channel;
  const T* z = a.z ? static_cast<const T*>(a.z) + p.base * a.d.z.seq + ct.channel : nullptr;
  const T* dy = static_cast<const T*>(a.dy) + p.base * a.d.dy.seq + ct.channel;
  T* dx = static_cast<T*>(a.dx) + p.base * a.d.dx.seq + c;
  T* ddt = static_cast<T*>(a.ddt) + p.base * a.d.ddt.seq + c;
  T* dz = a.dz ? static_cast<T*>(a.dz) + p.base * a.d.dz.seq + c : nullptr;
  const T* B = static_cast<const T*>(a.B) + p.base * a.d.B.seq + 1LL * ct.group * N;
  const T* C = static_cast<const T*>(a.C) + p.base * a.d.Cm.seq + 1LL * ct.group * N;

  const long long steps = (p.to - p.from + kStep - 1) / kStep, last = p.from + (steps - 1) * kStep;
  // a tile's rows into shared memory, its B and C into registers
  constexpr int kMine = kStep * NS / kScanThreads * 2;
  T states[kMine];
  auto load_tile = [&](long long tok, int turn) {
    const int n = p.to - tok < kStep ? static_cast<int>(p.to - tok) : kStep;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const T* src = w == 0 ? x : w == 1 ? dt : w == 2 ? dy : z;
      const long long row = w == 0 ? a.d.x.row : w == 1 ? a.d.dt.row : w == 2 ? a.d.dy.row : a.d.z.row;
      if (!src) continue;
      if (WIDE) {
#pragma unroll
        for (int i = threadIdx.x; i < kStep * kWide / kVec; i += kScanThreads) {
          const int t = i / (kWide / kVec), cc = i % (kWide / kVec) * kVec;
          if (t < n && cc < ct.channels) copy_async(&sh.rows[turn][w][t][cc], src + (tok + t) * row + cc);
        }
      } else if (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < kStep * kWide / kScanThreads; ++k) {
          const int i = threadIdx.x + k * kScanThreads, t = i / kWide, cc = i % kWide;
          if (t < n && cc < ct.channels) copy_async_4(&sh.rows[turn][w][t][cc], src + (tok + t) * row + cc);
        }
      } else {
        T v[kStep * kWide / kScanThreads];       // all on their way before the first is needed
#pragma unroll
        for (int k = 0; k < kStep * kWide / kScanThreads; ++k) {
          const int i = threadIdx.x + k * kScanThreads, t = i / kWide, cc = i % kWide;
          v[k] = t < n && cc < ct.channels ? src[(tok + t) * row + cc] : from_float<T>(0.f);
        }
#pragma unroll
        for (int k = 0; k < kStep * kWide / kScanThreads; ++k) (&sh.rows[turn][w][0][0])[threadIdx.x + k * kScanThreads] = v[k];
      }
    }
    if (mine) {
      const long long slot = kept_at(a, p, id, tok);
      const float4* kept = reinterpret_cast<const float4*>(a.kept) + (slot * (NS / 4) + 4 * q) * a.d.C + c;
#pragma unroll
      for (int k = 0; k < kStep / kKeep; ++k)
        if (k * kKeep < n) {
#pragma unroll
          for (int s = 0; s < 4; ++s) copy_async(&sh.kept[turn][k][s][threadIdx.x], kept + (k * (NS / 4LL) + s) * a.d.C);
          if (CUT && q == 0) copy_async_4(&sh.kept_sum[turn][k][ch], a.kept_sum + (slot + k) * a.d.C + c);
        }
    }
    copies_issued();
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = threadIdx.x + k % (kMine / 2) * kScanThreads, t = i / NS, m = i % NS;
      states[k] = m < N && t < n ? k < kMine / 2 ? B[(tok + t) * a.d.B.row + m] : C[(tok + t) * a.d.Cm.row + m] : from_float<T>(0.f);
    }
  };
  if (!mine)                                     // lanes without a channel take part in the sums over channels: as zeros
#pragma unroll
    for (int k = 0; k < 2 * (kStep / kKeep); ++k) {
#pragma unroll
      for (int s = 0; s < 4; ++s) sh.kept[k / (kStep / kKeep)][k % (kStep / kKeep)][s][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (CUT) sh.kept_sum[k / (kStep / kKeep)][k % (kStep / kKeep)][ch] = 0.f;
    }
  int turn = 0;
  if (steps > 0) {
    load_tile(last, 0);
  }
  float sum_d = 0.f, sum_b = 0.f;                // dy0 x, ddt
  for (long long tok = last; tok >= p.from; tok -= kStep, turn ^= 1) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) (&sh.states[turn][0][0][0])[threadIdx.x + k * kScanThreads] = to_float(states[k]);
    copies_landed();
    __syncthreads();                             // the tile is there, and the sums of the one before have been taken
    if (tok > p.from) load_tile(tok - kStep, turn ^ 1);
#pragma unroll 1
    for (int half = kStep - kKeep; half >= 0; half -= kKeep) {
      const int live = p.to - tok - half < kKeep ? static_cast<int>(p.to - tok - half) : kKeep;
      if (live <= 0) continue;
      Pair h0[8], h[kKeep][8];
      float d[kKeep], g[kKeep];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float4 v = sh.kept[turn][half / kKeep][s][threadIdx.x];
        h0[2 * s] = Pair(v.x, v.y);
        h0[2 * s + 1] = Pair(v.z, v.w);
      }
      if (CUT) {
        const float sum = sh.kept_sum[turn][half / kKeep][ch];
        const Pair all(sum, sum);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float4 b = *reinterpret_cast<const float4*>(&sh.before[threadIdx.x][4 * s]);
          h0[2 * s] = fma2(exp2_pair(mul2(A[2 * s], all)), Pair(b.x, b.y), h0[2 * s]);
          h0[2 * s + 1] = fma2(exp2_pair(mul2(A[2 * s + 1], all)), Pair(b.z, b.w), h0[2 * s + 1]);
        }
      }
#pragma unroll
      for (int t = 0; t < kKeep; ++t) {
        const bool in = mine && t < live;
        float xv = to_float(sh.rows[turn][0][half + t][ch]);
        d[t] = to_float(sh.rows[turn][1][half + t][ch]) + bias;
        if (a.d.softplus) d[t] = softplus(d[t]);
        g[t] = to_float(sh.rows[turn][2][half + t][ch]);
        if (z) {
          const float zv = to_float(sh.rows[turn][3][half + t][ch]);
          g[t] *= zv * sigmoid(zv);
        }
        if (!in) d[t] = g[t] = xv = 0.f;
        const Pair dd(d[t], d[t]), uu(d[t] * xv, d[t] * xv);
        const float4* bs = reinterpret_cast<const float4*>(&sh.states[turn][0][half + t][q * 16]);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float4 b = bs[s];
          h[t][2 * s] = fma2(exp2_pair(mul2(dd, A[2 * s])), t ? h[t ? t - 1 : 0][2 * s] : h0[2 * s], mul2(uu, Pair(b.x, b.y)));
          h[t][2 * s + 1] = fma2(exp2_pair(mul2(dd, A[2 * s + 1])), t ? h[t ? t - 1 : 0][2 * s + 1] : h0[2 * s + 1], mul2(uu, Pair(b.z, b.w)));
        }
      }
#pragma unroll
      for (int t = kKeep - 1; t >= 0; --t) {
        const bool in = mine && t < live;
        float xv = to_float(sh.rows[turn][0][half + t][ch]);
        if (!in) xv = 0.f;
        const float u = d[t] * xv;
        asm volatile("" : "+f"(d[t]));           // the decays are taken again: kept, they would cost as many registers as the states
        const Pair dd(d[t], d[t]), uu(u, u), gg(g[t], g[t]);
        const float4* bs = reinterpret_cast<const float4*>(&sh.states[turn][0][half + t][q * 16]);
        const float4* cs = reinterpret_cast<const float4*>(&sh.states[turn][1][half + t][q * 16]);
        float4* line = reinterpret_cast<float4*>(&sh.lines[warp][t & 1][lane][0]);
        Pair lb[2], ta[2], yy[2];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float4 b4 = bs[s], c4 = cs[s];
          Pair lu[2], gh[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int i = 2 * s + j;
            const Pair b = j ? Pair(b4.z, b4.w) : Pair(b4.x, b4.y), w = j ? Pair(c4.z, c4.w) : Pair(c4.x, c4.y);
            const Pair lam = fma2(w, gg, ca[i]);
            lu[j] = mul2(lam, uu);
            gh[j] = mul2(gg, h[t][i]);
            lb[j] = s ? fma2(lam, b, lb[j]) : mul2(lam, b);
            yy[j] = s ? fma2(w, h[t][i], yy[j]) : mul2(w, h[t][i]);
            ca[i] = mul2(exp2_pair(mul2(dd, A[i])), lam);
            const Pair through = mul2(ca[i], t ? h[t ? t - 1 : 0][i] : h0[i]);
            ta[j] = s ? fma2(through, A[i], ta[j]) : mul2(through, A[i]);
            dA[i] = fma2(through, dd, dA[i]);
          }
          const float2 l0 = lu[0].get(), l1 = lu[1].get(), g0 = gh[0].get(), g1 = gh[1].get();
          line[s] = make_float4(l0.x, l0.y, l1.x, l1.y);
          line[4 + s] = make_float4(g0.x, g0.y, g1.x, g1.y);
        }
        const float2 f = add2(lb[0], lb[1]).get(), e = add2(ta[0], ta[1]).get(), o = add2(yy[0], yy[1]).get();
        float s1 = f.x + f.y, s2 = (e.x + e.y) * kLn2, s3 = o.x + o.y;
#pragma unroll
        for (int k = 1; k < P; k <<= 1) {
          s1 += __shfl_xor_sync(~0u, s1, k);
          s2 += __shfl_xor_sync(~0u, s2, k);
          s3 += __shfl_xor_sync(~0u, s3, k);
        }
        float r = s2 + xv * s1;
        if (a.d.softplus) r *= sigmoid(to_float(sh.rows[turn][1][half + t][ch]) + bias);
        if (in && q == 0) {
          const long long at = tok + half + t;
          dx[at * a.d.dx.row] = from_float<T>(d[t] * s1 + D * g[t]);
          ddt[at * a.d.ddt.row] = from_float<T>(r);
          if (dz) {
            const float zv = to_float(sh.rows[turn][3][half + t][ch]), sg = sigmoid(zv);
            dz[at * a.d.dz.row] = from_float<T>(to_float(sh.rows[turn][2][half + t][ch]) * (s3 + D * xv) * (sg * (1.f + zv * (1.f - sg))));
          }
          sum_d += g[t] * xv;
          sum_b += r;
        }
        __syncwarp();                            // the lines of this token, while those of the one after it are read no more
        sum_lines<P, kLine>(sh.lines[warp][t & 1], sh.sums[warp][half + t]);
      }
    }
    __syncthreads();
    float* out = a.partial_bc + ((static_cast<long long>(block - ct.group * blocks_per_group) * a.rows + (a.d.packed ? tok : p.base * a.d.length + tok)) *
                                     a.d.groups + ct.group) * 2 * N;
    for (int i = threadIdx.x; i < kStep * 32 * P; i += kScanThreads) {
      const int t = i / (32 * P), e = i % (32 * P), which = e >> 4 & 1, n = (e >> 5) * 16 + (e & 15);
      if (n >= N || tok + t >= p.to) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < Shared::kWarps; ++w) v += sh.sums[w][t][e];
      out[(1LL * t * a.d.groups * 2 + which) * N + n] = v;
    }
  }
  if (!mine) return;
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const float2 v = dA[s].get(), w = ca[s].get();
    const int n = q * 16 + 2 * s;
    const long long at = (1LL * p.seq * a.d.C + c) * N + n, to = (1LL * id * a.d.C + c) * N + n;
    if (n < N) a.partial_a[to] = v.x;
    if (n + 1 < N) a.partial_a[to + 1] = v.y;
    if (a.dinitial && id == p.first) {
      if (n < N) a.dinitial[at] = w.x;
      if (n + 1 < N) a.dinitial[at + 1] = w.y;
    }
  }
  if (q == 0) {
    a.partial_d[2LL * id * a.d.C + c] = sum_d;
    a.partial_d[(2LL * id + 1) * a.d.C + c] = sum_b;
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

int scan_grad_slots(int N) { return N <= 16 ? 16 : scan_state_slots(N); }
long long scan_kept(const ScanArgs& a) { return a.rows / kKeep + a.pieces + 1; }

// Pieces of the gradient's call.  Being cut costs three operations per state in the forward walk.  Counted are two blocks to an SM in every
// form, although registers and shared memory (GradShape: 118 KB for cut float32 sequences, 118 to 130 KB over 64 states) leave cut float32
// sequences and those of over 64 states one: the forward walk, which holds three, gains more from the finer cut than a second round of the
// backward walk costs.  Float32, 2048 channels, 16 states, counted as two / as they fit: 9 x 2048 tokens 1844 / 2234 us, 4 x 2048 830 / 1055,
// 1 x 8192 843 / 944; 16 x 1000 of 2560 channels 1870 / 1853; 4 x 1024 of 1024 channels and 128 states, bfloat16, 3074 / 3080.
void plan_grad_pieces(ScanArgs* a) {
  const int wide = kScanThreads * 16 / scan_grad_slots(a->d.N), per = a->d.C / a->d.groups;
  const long long tiles = 1LL * a->d.groups * ((per + wide - 1) / wide);
  a->rows = a->d.packed ? a->d.length : a->d.sequences * a->d.length;
  a->tiles = static_cast<int>(tiles);
  cut_pieces(a, tiles, 148 * kGradBlocks);
}

namespace {

template <typename T, int P, bool CUT>
cudaError_t run_grad(const ScanArgs& a, cudaStream_t s) {
  static PerDeviceOnce setup;
  constexpr int kSmem = sizeof(GradShape<T, P, CUT>);
  cudaError_t e = setup.ensure([] {
    const cudaError_t e = cudaFuncSetAttribute(scan_grad_kernel<T, true, P, CUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(scan_grad_kernel<T, false, P, CUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(a.tiles * a.pieces);
  const bool states16 = a.d.N % (16 / sizeof(T)) == 0 && rows_aligned(a.B, a.d.B, a.d.dtype) && rows_aligned(a.C, a.d.Cm, a.d.dtype);
  const int per = a.d.C / a.d.groups;
  const bool rows16 = per % (16 / static_cast<int>(sizeof(T))) == 0 && rows_aligned(a.x, a.d.x, a.d.dtype) && rows_aligned(a.dt, a.d.dt, a.d.dtype) &&
                      rows_aligned(a.z, a.d.z, a.d.dtype) && rows_aligned(a.dy, a.d.dy, a.d.dtype);
  if (states16) launch_streaming(scan_trace_kernel<T, 16, P, true, CUT>, grid, kScanThreads, 0, s, a);
  else launch_streaming(scan_trace_kernel<T, 16, P, false, CUT>, grid, kScanThreads, 0, s, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (rows16) launch_streaming(scan_grad_kernel<T, true, P, CUT>, grid, kScanThreads, kSmem, s, a);
  else launch_streaming(scan_grad_kernel<T, false, P, CUT>, grid, kScanThreads, kSmem, s, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const long long bc = a.rows * a.d.groups * 2 * a.d.N;
  if ((bc + 255) / 256 >= INT32_MAX) return cudaErrorInvalidValue;
  launch_streaming(scan_bc_kernel<T>, static_cast<unsigned>((bc + 255) / 256), 256, 0, s, a, a.tiles / a.d.groups);
  return cudaGetLastError();
}
template <typename T>
cudaError_t run_grad_type(const ScanArgs& a, cudaStream_t s) {
  const bool cut = a.piece < a.d.length;
  switch (scan_grad_slots(a.d.N) / 16) {
    case 1: return cut ? run_grad<T, 1, true>(a, s) : run_grad<T, 1, false>(a, s);
    case 2: return cut ? run_grad<T, 2, true>(a, s) : run_grad<T, 2, false>(a, s);
    case 4: return cut ? run_grad<T, 4, true>(a, s) : run_grad<T, 4, false>(a, s);
    default: return cut ? run_grad<T, 8, true>(a, s) : run_grad<T, 8, false>(a, s);
  }
}

}  // namespace

cudaError_t launch_scan_grad(const ScanArgs& args, int* launches, cudaStream_t s) {
  ScanArgs a = args;
  if (1LL * a.tiles * a.pieces >= INT32_MAX) return cudaErrorInvalidValue;
  cudaError_t e;
  if (a.d.dtype == B200CONV_F32) e = run_grad_type<float>(a, s);
  else e = a.d.dtype == B200CONV_F16 ? run_grad_type<__half>(a, s) : run_grad_type<__nv_bfloat16>(a, s);
  if (e != cudaSuccess) return e;
  *launches = 4;
  const long long all = 1LL * a.d.C * (a.d.N + 2);
  launch_streaming(scan_params_kernel, static_cast<unsigned>((all + 31) / 32), 256, 0, s, a);
  return cudaGetLastError();
}

}  // namespace b200
