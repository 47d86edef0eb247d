// Whether tensors of several dimensions share memory, for the argument checks and (compiled alone by a host compiler)
// for the tests.
#pragma once

#include "nrq_rows.h"

namespace nrq {

struct Dim {
  int64_t stride = 0;  // elements
  size_t n = 1;
};

// A tensor of up to four dimensions of rows, for the question whether two share memory. Exact where both come down to
// rows of one dimension, once dimensions that follow one another without gaps, or at one distance, are taken together; else two
// that lie between one another count as sharing.
struct Extent {
  const void* first;
  size_t len;  // elements of a row
  int size;    // bytes of one
  Dim d[4];
};

inline Rows as_rows(const Extent& e) {
  Dim d[4];
  int n = 0;
  typedef __int128 wide;
  wide low = 0, len = (wide)e.len;
  for (const Dim& x : e.d) {
    if (x.n == 0) return Rows{e.first, 0, 0, 0, e.size};
    if (x.n == 1 || x.stride == 0) continue;
    Dim y = x;
    if (y.stride < 0) {  // from its other end
      low += (wide)y.stride * (wide)(y.n - 1);
      y.stride = y.stride == INT64_MIN ? INT64_MAX : -y.stride;
    }
    int i = n++;
    for (; i > 0 && d[i - 1].stride > y.stride; i--) d[i] = d[i - 1];
    d[i] = y;
  }
  int at = 0;  // dimensions d[at] .. d[n - 1] are left
  while (at < n && (wide)d[at].stride <= len) len += (wide)d[at].stride * (wide)(d[at].n - 1), at++;
  while (n - at > 1) {
    Dim &x = d[at], &y = d[at + 1];
    if ((wide)y.stride == (wide)x.stride * (wide)x.n) {
      x.n *= y.n;
      for (int i = at + 1; i + 1 < n; i++) d[i] = d[i + 1];
      n--;
    } else {
      len += (wide)x.stride * (wide)(x.n - 1), at++;
    }
  }
  const wide past = (wide)INT64_MAX / 16;  // any memory
  if (len > past) len = past;
  Rows r{(const char*)e.first + (int64_t)(low * e.size), 1, 0, (size_t)len, e.size};
  if (at < n) r.n = d[at].n, r.stride = d[at].stride;
  return r;
}

// From the least address of a tensor to behind its greatest; what overflows reaches everywhere.
struct Range {
  uintptr_t low, high;
};
inline Range range_of(const Extent& e) {
  const uintptr_t all = ~(uintptr_t)0;
  int64_t low = 0, high = (int64_t)e.len;
  bool over = e.len > (size_t)INT64_MAX;
  for (const Dim& x : e.d) {
    if (x.n == 0) return Range{1, 0};
    int64_t span;
    over |= x.n > (size_t)INT64_MAX || __builtin_mul_overflow(x.stride, (int64_t)(x.n - 1), &span);
    if (over) return Range{0, all};
    over |= __builtin_add_overflow(span < 0 ? low : high, span, span < 0 ? &low : &high);
  }
  if (e.len == 0) return Range{1, 0};
  int64_t from, to;
  over |= __builtin_mul_overflow(low, (int64_t)e.size, &from) || __builtin_mul_overflow(high, (int64_t)e.size, &to);
  if (over || (uintptr_t)e.first < (uintptr_t)-from || (uintptr_t)e.first > all - (uintptr_t)to) return Range{0, all};
  return Range{(uintptr_t)e.first + from, (uintptr_t)e.first + to};
}

// Whether two tensors of these ranges share memory, or lie between one another as as_rows() cannot tell apart.
inline bool extents_meet(const Extent& a, const Range& x, const Extent& b, const Range& y) {
  return x.low < y.high && y.low < x.high && rows_meet(as_rows(a), as_rows(b));
}

// Whether a tensor and another of the same layout at `other` share memory, where no two rows of one overlap (each dimension steps
// over all of the smaller ones'). Exact, wherever one lies in the other: rows meet where their distance, less than a row,
// is the tensors' and some steps of each dimension. A dimension's steps leave what the smaller ones span, less than its stride,
// so that there are two numbers of them at most.
inline bool copies_meet(const Extent& e, const void* other) {
  typedef __int128 wide;
  struct Step {
    wide stride, most;  // bytes; steps either way
  } d[sizeof e.d / sizeof e.d[0]];
  int n = 0;
  wide span = (wide)e.len * e.size;  // of what is smaller, beside the row's first byte
  for (const Dim& x : e.d) {
    if (x.n == 0) return false;
    if (x.n == 1) continue;
    int i = n++;
    const Step y{(wide)(x.stride < 0 ? -(wide)x.stride : (wide)x.stride) * e.size, (wide)(x.n - 1)};
    for (; i > 0 && d[i - 1].stride > y.stride; i--) d[i] = d[i - 1];
    d[i] = y;
    span += y.stride * y.most;
  }
  if (e.len == 0) return false;
  struct Search {
    const Step* d;
    bool meet(int n, wide off, wide span) const {
      if (off >= span || -off >= span) return false;
      if (n == 0) return true;
      const Step& x = d[n - 1];
      const wide rest = span - x.stride * x.most;
      if (x.stride == 0) return meet(n - 1, off, rest);
      wide k = -(off + rest - 1) / x.stride;  // near the least with off + k stride > -rest
      k = k - 1 < -x.most ? -x.most : k - 1;
      for (; k <= x.most && off + k * x.stride < rest; k++)
        if (meet(n - 1, off + k * x.stride, rest)) return true;
      return false;
    }
  };
  return Search{d}.meet(n, (wide)(uintptr_t)other - (wide)(uintptr_t)e.first, span);
}

}  // namespace nrq
