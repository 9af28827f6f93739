// Whether tensors of rows share memory: what the sequence operators refuse for their results.  Host code, exact for any strides.
//
// Row (i, j) of a region begins at p + i * outer + j * inner.  Two regions of equal strides (the usual case of neighbours in one wider
// tensor) meet where a difference of indexes brings their starts closer than a row: a few candidates of the larger stride, each decided
// by a division.  Other strides: the rows of the region that has fewer, one after the other against the whole of the other.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "../../include/b200conv.h"

namespace b200 {

struct Region {
  const char* name;
  const char* p;                    // nullptr: nothing
  long long outer, inner;           // bytes; inner <= outer
  long long n_outer, n_inner, width;
  unsigned in_place, any;           // of a result, bits of the inputs that it may replace row by row, and that it may overlap anyhow
  long long rows[4];                // strides and extents as the caller gave them

  bool empty() const { return !p || n_outer <= 0 || n_inner <= 0 || width <= 0; }
  long long extent() const { return (n_outer - 1) * outer + (n_inner - 1) * inner + width; }
};

// sequences x length rows of `width` elements of es bytes.
inline Region region(const char* name, const void* p, const b200conv_rows& r, long long sequences, long long length, long long width, size_t es,
                     unsigned in_place = 0, unsigned any = 0) {
  const long long e = static_cast<long long>(es);
  Region a = {name, static_cast<const char*>(p), sequences > 1 ? r.seq * e : 0, length > 1 ? r.row * e : 0, sequences, length, width * e, in_place, any, {}};
  a.rows[0] = a.outer; a.rows[1] = a.inner; a.rows[2] = sequences; a.rows[3] = length;
  if (a.inner > a.outer) {
    std::swap(a.inner, a.outer);
    std::swap(a.n_inner, a.n_outer);
  }
  return a;
}
inline Region region(const char* name, const void* p, size_t bytes, unsigned in_place = 0, unsigned any = 0) {
  return region(name, p, b200conv_rows{}, 1, 1, static_cast<long long>(bytes), 1, in_place, any);
}

inline long long floor_div(long long a, long long b) { return a / b - (a % b < 0); }          // b > 0

// Whether i * outer + j * inner lies strictly between lo and hi for some i, j of the ranges; `zero`: i = j = 0 counts.
inline bool reaches(long long outer, long long inner, long long i0, long long i1, long long j0, long long j1, long long lo, long long hi, bool zero = true) {
  if (outer > 0) {                  // what j can add: [j0, j1] * inner
    i0 = std::max(i0, floor_div(lo - j1 * inner, outer));
    i1 = std::min(i1, floor_div(hi - j0 * inner, outer) + 1);
  } else {
    i0 = std::max(i0, 0LL);         // all the same: the first one (0 is in every range)
    i1 = std::min(i1, 0LL);
  }
  for (long long i = i0; i <= i1; ++i) {
    const long long l = lo - i * outer, h = hi - i * outer;
    if (inner > 0) {
      const long long first = std::max(j0, floor_div(l, inner) + 1), last = std::min(j1, floor_div(h - 1, inner));
      if (first > last) continue;
      if (zero || i || first || last) return true;
    } else if (l < 0 && 0 < h && (zero || i)) {
      return true;
    }
  }
  return false;
}

inline bool overlap(const Region& a, const Region& b) {
  if (a.empty() || b.empty()) return false;
  const long long delta = static_cast<long long>(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
  if (delta >= a.extent() || -delta >= b.extent()) return false;
  if (a.outer == b.outer && a.inner == b.inner)
    return reaches(a.outer, a.inner, 1 - b.n_outer, a.n_outer - 1, 1 - b.n_inner, a.n_inner - 1, delta - a.width, delta + b.width);
  if (a.n_outer * a.n_inner > b.n_outer * b.n_inner) return overlap(b, a);
  for (long long i = 0; i < a.n_outer; ++i)
    for (long long j = 0; j < a.n_inner; ++j) {
      const long long at = i * a.outer + j * a.inner - delta;            // this row, from b's first one
      if (reaches(b.outer, b.inner, 0, b.n_outer - 1, 0, b.n_inner - 1, at - b.width, at + a.width)) return true;
    }
  return false;
}

// Whether rows of one region share memory with each other.
inline bool folded(const Region& a) {
  if (a.empty()) return false;
  if ((a.n_inner == 1 || a.inner >= a.width) && (a.n_outer == 1 || a.outer >= (a.n_inner - 1) * a.inner + a.width)) return false;
  if ((a.n_outer > 1 && a.outer == 0) || (a.n_inner > 1 && a.inner == 0)) return true;
  return reaches(a.outer, a.inner, 0, a.n_outer - 1, 1 - a.n_inner, a.n_inner - 1, -a.width, a.width, false);
}

// Row by row the same memory (widths may differ by pad channels).
inline bool same_place(const Region& a, const Region& b) {
  return a.p == b.p && std::equal(a.rows, a.rows + 4, b.rows);
}

}  // namespace b200
