// What the passes of the selective scan share: pieces of sequences, tiles of tokens in shared memory, lane sums.
//
// A channel's N states are spread over P neighbouring lanes, up to sixteen to a lane (N <= 16 P, states beyond N stay zero; steps hold eight
// to a lane), so that a warp holds 32 / P channels.  Sequences may be cut into pieces of `piece` tokens that blocks take independently; what a piece
// does to a state is h -> exp(A sum of delta) h + (its own result from zero), so pieces are joined by one exponential each.
#pragma once
#include <type_traits>

#include "internal.h"
#include "rows.cuh"

namespace b200 {

constexpr int kScanThreads = 128;

// log(1 + e^v) = max(v, 0) + log(1 + e) with e = e^-|v| in (0, 1]: no overflow, and small steps keep their relative precision.
// log(1 + e) / e is a polynomial of degree 8 whose coefficients were fitted here by iteratively reweighted least squares (Lawson),
// off by 3e-8, with float32 roundings by 2e-7: one trip through the special function unit, which the scan's decays already fill.
// The exponential adds its own 2^-22 and the rounding of |v| log2(e): below zero the whole is within (8 + 1.25 |v|) 2^-24 of the result,
// 1e-6 for the steps of 0.001 (v = -6.9) that layers start with.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_fast(-fabsf(v) * kLog2e);
  float q = 0.005232629366219044f;
  q = fmaf(q, e, -0.029504986479878426f);
  q = fmaf(q, e, 0.07822556048631668f);
  q = fmaf(q, e, -0.13663214445114136f);
  q = fmaf(q, e, 0.1910599321126938f);
  q = fmaf(q, e, -0.2484297901391983f);
  q = fmaf(q, e, 0.3331909775733948f);
  q = fmaf(q, e, -0.4999949336051941f);
  q = fmaf(q, e, 0.9999999403953552f);
  return fmaf(q, e, fmaxf(v, 0.f));
}
// v held between -127 and 128; NaN stays NaN.
__device__ __forceinline__ float clamp_exponent(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-127.f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(128.f));
  return r;
}
// 2^v of both without the special function unit: v = n + f with n the nearest integer (the low bits of v + 1.5 * 2^23), 2^f a
// polynomial of degree 5 fitted here by iteratively reweighted least squares (off by 2e-7 with float32 roundings), 2^n into the
// exponent.  The ends of the range come out of the same addition: 2^128 is the infinity's bits, 2^-127 those of zero (between 2^-127 and
// 2^-126 results are off by up to 2^-127).  The addition makes a number of a NaN's bits: v * 0 brings it back.
__device__ __forceinline__ Pair exp2_poly(Pair a) {
  const float2 v = a.get();
  const Pair x(clamp_exponent(v.x), clamp_exponent(v.y)), magic(12582912.f, 12582912.f), back(-12582912.f, -12582912.f), minus(-1.f, -1.f);
  const Pair t = add2(x, magic), f = fma2(add2(t, back), minus, x);
  Pair p = fma2(f, Pair(0.001326472731307149f, 0.001326472731307149f), Pair(0.009671512991189957f, 0.009671512991189957f));
  p = fma2(p, f, Pair(0.05550733581185341f, 0.05550733581185341f));
  p = fma2(p, f, Pair(0.24022242426872253f, 0.24022242426872253f));
  p = fma2(p, f, Pair(0.6931470036506653f, 0.6931470036506653f));
  p = fma2(p, f, Pair(1.f, 1.f));
  const float2 r = p.get(), n = t.get();
  const Pair e(__int_as_float(__float_as_int(r.x) + (__float_as_int(n.x) << 23)), __int_as_float(__float_as_int(r.y) + (__float_as_int(n.y) << 23)));
  return fma2(x, Pair(0.f, 0.f), e);
}
__device__ __forceinline__ Pair exp2_pair(Pair a) {
  const float2 f = a.get();
  return Pair(exp2_fast(f.x), exp2_fast(f.y));
}

// Whether a lane has a state that is not zero.  Where pieces are joined zeros are not multiplied by the decays of a whole piece: growing
// ones may exceed float32 together where the tokens' own, one after the other, leave the zero alone.
template <int M> __device__ __forceinline__ bool any_of(const Pair (&v)[M]) {
  unsigned long long bits = 0;
#pragma unroll
  for (int s = 0; s < M; ++s) bits |= v[s].v;
  return bits & 0x7fffffff7fffffffull;
}

// A log2(e).  A decay of minus infinity ends a state in any step of positive size and, like every other, not in one of size zero
// (as which the tokens behind a piece count).
__device__ __forceinline__ float scaled_decay(float A) {
  float v;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(A * kLog2e), "f"(-3.4e38f));
  return v;
}

// The tokens of a piece: sequence `seq`, its tokens [from, to) counted from the tensor's row `row0` of that sequence.
struct Piece {
  int seq;
  long long from, to;            // regular: tokens of the sequence; packed: rows of the tensor
  long long base;                // sequence whose `seq` stride the tensors are addressed with (packed: 0)
  int first, last;               // pieces of the same sequence, by number
  bool valid;
};
__device__ __forceinline__ Piece piece_of(const ScanArgs& a, int id) {
  Piece p;
  if (!a.d.packed) {
    p.seq = id / a.pieces_per_seq;
    const int k = id - p.seq * a.pieces_per_seq;
    p.from = 1LL * k * a.piece;
    p.to = p.from + a.piece < a.d.length ? p.from + a.piece : a.d.length;
    p.base = p.seq;
    p.first = p.seq * a.pieces_per_seq;
    p.last = p.first + a.pieces_per_seq - 1;
    p.valid = true;
    return p;
  }
  // Windows of `piece` rows cut the packed tensor; sequence i meets window k in piece i + k: the number grows by one from
  // a window to the next and from a sequence to the next, so that no two pieces share it (and some stay empty).
  const int n = static_cast<int>(a.d.sequences);
  int lo = 0, left = n;
  while (left > 0) {             // the last sequence whose first piece is not behind `id`, 32 at a time as in sequence_of
    const int step = (left + 31) >> 5, i = (threadIdx.x & 31) * step, j = lo + (i < left ? i : 0);
    const int m = __popc(__ballot_sync(~0u, i < left && start_of(a.starts, j, a.d.length) / a.piece + j <= id));
    if (m == 0) break;
    const int end = m * step < left ? m * step : left;
    left = end - (m - 1) * step - 1;
    lo += (m - 1) * step + 1;
  }
  p.seq = lo - 1;
  p.base = 0;
  p.valid = p.seq >= 0;
  p.from = p.to = 0;
  p.first = p.last = id;
  if (!p.valid) return p;
  const long long s0 = start_of(a.starts, p.seq, a.d.length), s1 = start_of(a.starts, p.seq + 1, a.d.length);
  const long long k = id - p.seq, w0 = k * a.piece, w1 = w0 + a.piece;
  p.from = s0 > w0 ? s0 : w0;
  p.to = s1 < w1 ? s1 : w1;
  p.first = p.seq + static_cast<int>(s0 / a.piece);
  p.last = s1 > s0 ? p.seq + static_cast<int>((s1 - 1) / a.piece) : p.first;
  if (p.to <= p.from) {
    p.valid = s1 <= s0 && id == p.first;         // an empty sequence: its state passes through
    p.to = p.from;
  }
  return p;
}

// The channels of a block lie in one group of B and C.
struct ScanTile { int group, channel, channels; };
__device__ __forceinline__ ScanTile scan_tile(const ScanArgs& a, int tile, int width) {
  const int per = a.d.C / a.d.groups, tiles = (per + width - 1) / width;
  ScanTile t;
  t.group = tile / tiles;
  const int c = (tile - t.group * tiles) * width;
  t.channel = t.group * per + c;
  t.channels = per - c < width ? per - c : width;
  return t;
}

// Partial sums of a piece without tokens.
__device__ __forceinline__ void clear_piece_sums(const ScanArgs& a, int id, const ScanTile& ct, int threads) {
  for (int i = threadIdx.x; i < ct.channels * a.d.N; i += threads) a.partial_a[(1LL * id * a.d.C + ct.channel) * a.d.N + i] = 0.f;
  for (int i = threadIdx.x; i < ct.channels; i += threads)
    a.partial_d[2LL * id * a.d.C + ct.channel + i] = a.partial_d[(2LL * id + 1) * a.d.C + ct.channel + i] = 0.f;
}

constexpr int kPolyPairs = 1;                    // pairs of decays that a lane takes by polynomial: none 227, one 210, two 216 us when it was brought (8192 tokens, 2048 channels), two against one 196 to 190 us since
constexpr int tile_tokens(int NS) { return NS <= 32 ? 32 : 1024 / NS; }           // of a tile of B and C

// 16 bytes from global to shared memory without a register in between.
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Rows of B (and C) of a tile on their way to shared memory: [B or C][tokens][NS], zeros beyond N and beyond the piece.
template <typename T, int NS, bool WIDE, bool BOTH, int TOKENS = tile_tokens(NS)>
struct StateRows {
  static constexpr int kTokens = TOKENS, kVec = WIDE ? 16 / sizeof(T) : 1, kRow = NS / kVec, kAll = (BOTH ? 2 : 1) * kTokens * kRow,
                       kMine = (kAll + kScanThreads - 1) / kScanThreads;
  Pack<T, kVec> v[kMine];
  __device__ __forceinline__ void load(const T* B, long long brow, const T* C, long long crow, long long tok, long long to, int N) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = threadIdx.x + k * kScanThreads, which = BOTH ? i / (kTokens * kRow) : 0, t = i / kRow % kTokens, n = i % kRow * kVec;
      if (i < kAll && tok + t < to && n < N) v[k].load(which ? C + (tok + t) * crow + n : B + (tok + t) * brow + n);
      else v[k].clear();
    }
  }
  __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = threadIdx.x + k * kScanThreads;
      if (i >= kAll) break;
#pragma unroll
      for (int e = 0; e < kVec; ++e) dst[i * kVec + e] = v[k].get(e);
    }
  }
};

}  // namespace b200
