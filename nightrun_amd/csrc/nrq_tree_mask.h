// What a node of a tree of drafts sees, in bits, for kernels and (compiled alone by a host compiler) for the tests.
#pragma once

#include "nrq_page.h"

namespace nrq {

// A node's parent: one of those before it, else none.
NRQ_HD int tree_parent(int parent, int node) { return parent >= 0 && parent < node ? parent : -1; }

// Bit i: whether position p0 + i is before the tree, which begins at `base`, or one of the nodes in `above`.
NRQ_HD uint32_t tree_sees(uint64_t above, int p0, int base) {
  const int64_t r = (int64_t)p0 - base;  // of bit 0 in the tree
  if (r >= 64) return 0;
  if (r >= 0) return (uint32_t)(above >> r);
  if (r <= -32) return 0xffffffffu;
  return (uint32_t)(above << -r) | ((1u << -r) - 1);
}

// Bit i: whether position p0 + i is at `lo` or behind it, or in the tree (where `above` holds the window).
NRQ_HD uint32_t tree_from(int lo, int p0, int base) {
  const int64_t r = (int64_t)(lo < base ? lo : base) - p0;  // of the first that counts
  if (r <= 0) return 0xffffffffu;
  return r >= 32 ? 0 : 0xffffffffu << r;
}

}  // namespace nrq
