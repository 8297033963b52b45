// Whether two strided operands share a byte: exactly, since slices of one buffer (q, k and v of a fused projection) lie
// between each other without meeting. Host only, no CUDA.
#pragma once
#include <utility>

namespace lbw {

// The bytes base + i s0 + j s1 + [0, len), i < n0, j < n1.
struct ByteGrid {
  long long base, n0, s0, n1, s1, len;

  long long row_end() const { return base + (n1 - 1) * s1 + len; }  // of i = 0
  long long end() const { return row_end() + (n0 - 1) * s0; }
  ByteGrid row(long long i) const { return {base + i * s0, 1, 0, n1, s1, len}; }

  // Rows [rows, heads, dim] of elements of `size` bytes; strides in elements, of any sign.
  static ByteGrid of(const void* p, long long rows, long long row_stride, long long heads, long long head_stride, int dim,
                     int size) {
    ByteGrid g{(long long)(unsigned long long)p, rows, row_stride * size, heads, head_stride * size, (long long)dim * size};
    g.tidy();
    return g;
  }

  // Strides not negative, s0 the larger, dimensions that repeat or continue the inner ones folded into len.
  void tidy() {
    if (n0 < 1 || n1 < 1) return;  // no bytes at all
    if (s0 < 0) base += s0 * (n0 - 1), s0 = -s0;
    if (s1 < 0) base += s1 * (n1 - 1), s1 = -s1;
    if (s0 == 0) n0 = 1;
    if (s1 == 0) n1 = 1;
    if (n0 == 1) s0 = 0;
    if (n1 == 1) s1 = 0;
    if (s1 > s0) std::swap(n0, n1), std::swap(s0, s1);
    if (s1 <= len) len += s1 * (n1 - 1), n1 = 1, s1 = 0;
    if (n1 == 1) std::swap(n0, n1), std::swap(s0, s1);  // one dimension left: the inner one
    if (n1 > 1 && n0 == 1 && s1 <= len) len += s1 * (n1 - 1), n1 = 1, s1 = 0;
  }
};

// Rows of a from first to last that may meet bytes [lo, hi): those that start below hi and end above lo.
inline void rows_between(const ByteGrid& a, long long lo, long long hi, long long& first, long long& last) {
  first = a.row_end() > lo || a.s0 == 0 ? 0 : (lo - a.row_end()) / a.s0 + 1;
  last = a.s0 == 0 ? 0 : (hi - 1 - a.base) / a.s0;
  if (last > a.n0 - 1) last = a.n0 - 1;
}

inline bool overlap(ByteGrid a, ByteGrid b) {
  if (a.n0 < 1 || a.n1 < 1 || b.n0 < 1 || b.n1 < 1 || a.base >= b.end() || b.base >= a.end()) return false;
  if (a.n0 == 1 && a.n1 == 1 && b.n0 == 1 && b.n1 == 1) return true;
  // One dimension left in both: compare by that one.
  if (a.n0 == 1 && b.n0 == 1) std::swap(a.n0, a.n1), std::swap(a.s0, a.s1), std::swap(b.n0, b.n1), std::swap(b.s0, b.s1);
  if (a.n0 > 1 && b.n0 > 1 && a.s0 == b.s0) {
    // Rows i of a and i + d of b lie to each other as rows 0 and d, for few d: one row's length apart at most.
    long long first, last;
    ByteGrid all = b;  // rows -(a.n0 - 1) .. b.n0 - 1 of b
    all.base -= (a.n0 - 1) * a.s0;
    all.n0 += a.n0 - 1;
    rows_between(all, a.base, a.row_end(), first, last);
    for (long long d = first; d <= last; ++d)
      if (overlap(a.row(0), all.row(d))) return true;
    return false;
  }
  if (a.n0 == 1) std::swap(a, b);
  long long first, last;
  rows_between(a, b.base, b.end(), first, last);
  for (long long i = first; i <= last; ++i)
    if (overlap(a.row(i), b)) return true;
  return false;
}

}  // namespace lbw
