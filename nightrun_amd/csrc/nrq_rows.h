// Whether two sets of rows in memory share a byte, for the argument checks and (compiled alone by a host compiler)
// for the tests. Exact: rows of two column ranges of one matrix lie between one another and share none.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace nrq {

struct Rows {
  const void* first;
  size_t n;
  int64_t stride;  // elements, any
  size_t len;      // elements of a row
  int size = 1;    // bytes of an element
};

inline bool rows_meet(Rows a, Rows b) {
  typedef __int128 wide;  // strides and counts may be anything
  if (!a.n || !b.n || !a.len || !b.len) return false;
  wide at[2], step[2], n[2] = {(wide)a.n, (wide)b.n}, len[2] = {(wide)a.len * a.size, (wide)b.len * b.size};
  const Rows* r[2] = {&a, &b};
  for (int i = 0; i < 2; i++) {
    at[i] = (wide)(uintptr_t)r[i]->first;
    step[i] = (wide)r[i]->stride * r[i]->size;
    if (step[i] < 0) at[i] += step[i] * (n[i] - 1), step[i] = -step[i];
    if (step[i] == 0) n[i] = 1;
    if (step[i] <= len[i] && n[i] > 1) len[i] += step[i] * (n[i] - 1), n[i] = 1;  // no gaps: one row
  }
  if (at[0] + step[0] * (n[0] - 1) + len[0] <= at[1] || at[1] + step[1] * (n[1] - 1) + len[1] <= at[0]) return false;
  if (n[0] > 1 && n[1] > 1 && step[0] == step[1]) {
    // row j of b begins d + (j - i) step behind row i of a: some j - i has to bring that above -len[1] and below len[0]
    const wide d = at[1] - at[0], s = step[0], over = d + len[1] - 1, low = -(n[0] - 1), high = n[1] - 1;
    wide k = over >= 0 ? -(over / s) : (-over + s - 1) / s;  // the least with d + k s > -len[1]
    if (k < low) k = low;
    return k <= high && d + k * s < len[0];
  }
  for (wide i = 0, j = 0; i < n[0]; i++) {  // both in order
    const wide x = at[0] + step[0] * i;
    while (j < n[1] && at[1] + step[1] * j + len[1] <= x) j++;
    if (j == n[1]) return false;
    if (at[1] + step[1] * j < x + len[0]) return true;
  }
  return false;
}

}  // namespace nrq
