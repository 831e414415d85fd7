// Whether operands share memory (internal; plain C++).  An operand is n rows,
// `row` bytes apart, of m pieces, `col` bytes apart, of `size` bytes each.  Every
// piece counts, what lies between them does not: an operand may lie in another's gaps.
#pragma once
#include <stdint.h>

namespace ann {

struct Strided {
  const void* at;
  int64_t n, row, m, col, size;
};

// Whether one of n pieces of `size` bytes, `step` apart from p on, shares a byte with
// [lo, hi).  128 bits: strides and counts are the caller's.
inline bool pieces_meet(__int128 p, int64_t n, __int128 step, int64_t size, __int128 lo, __int128 hi) {
  if (n < 1 || size < 1 || hi <= lo) return false;
  if (step < 0) {
    p += (n - 1) * step;
    step = -step;
  }
  __int128 i = 0;   // the first piece that ends behind lo
  if (p + size <= lo) {
    if (step == 0) return false;
    i = (lo - size - p) / step + 1;
  }
  return i < n && p + i * step < hi;
}

inline bool operand_meets(const Strided& x, __int128 lo, __int128 hi) {
  const __int128 p = (intptr_t)x.at;
  // along the longer of the two counts at once
  if (x.n >= x.m) {
    for (int64_t j = 0; j < x.m; ++j)
      if (pieces_meet(p + (__int128)j * x.col, x.n, x.row, x.size, lo, hi)) return true;
  } else {
    for (int64_t i = 0; i < x.n; ++i)
      if (pieces_meet(p + (__int128)i * x.row, x.m, x.col, x.size, lo, hi)) return true;
  }
  return false;
}

// First byte and the one behind the last of what an operand spans.
inline void operand_span(const Strided& x, __int128* lo, __int128* hi) {
  const __int128 a = (__int128)(x.n - 1) * x.row, b = (__int128)(x.m - 1) * x.col;
  *lo = (__int128)(intptr_t)x.at + (a < 0 ? a : 0) + (b < 0 ? b : 0);
  *hi = (__int128)(intptr_t)x.at + (a > 0 ? a : 0) + (b > 0 ? b : 0) + x.size;
}

// Whether y, rows of one piece each (y.m 1; contiguous rows: n 1), shares a byte with x.
inline bool overlap(const Strided& x, const Strided& y) {
  if (x.n < 1 || x.m < 1 || x.size < 1 || y.n < 1 || y.size < 1) return false;
  __int128 xl, xh, yl, yh;
  operand_span(x, &xl, &xh);
  operand_span(y, &yl, &yh);
  if (xh <= yl || yh <= xl) return false;   // nearly always
  const __int128 p = (intptr_t)y.at;
  if (x.m == 1 && x.row == y.row) {   // row i of x and row j of y lie i - j strides apart from the first ones
    return pieces_meet((__int128)(intptr_t)x.at - (__int128)(y.n - 1) * y.row, x.n + y.n - 1, x.row, x.size, p,
                       p + y.size);
  }
  if (x.m == 1 && x.n < y.n) return overlap(y, x);
  for (int64_t j = 0; j < y.n; ++j) {
    const __int128 lo = p + (__int128)j * y.row;
    if (operand_meets(x, lo, lo + y.size)) return true;
  }
  return false;
}

}  // namespace ann
