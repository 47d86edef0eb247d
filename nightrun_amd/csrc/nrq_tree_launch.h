// Internal launch interface of the operators for trees of drafts (nrq_tree.hip checks the
// arguments; the kernel files launch). The public interface is include/nrq_tree.h.
#pragma once

#include "nrq_serve_launch.h"

namespace nrq {

struct NormRopeLaunch {
  RopeLaunch r;
  bool norm;
  const float *wq, *wk;  // nullptr: ones
  float eps;
  const int* at;  // cache positions; nullptr: r.pos
};
hipError_t launch_norm_rope(const NormRopeLaunch& L);

double tree_attn_line(size_t seqs, size_t n_new, size_t heads, int n_kv, int64_t held);  // tiles of all units at most
size_t tree_attn_workspace(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd);
hipError_t launch_tree_attn(const PagedAttnLaunch& L);

constexpr int kTreeMost = 64;  // nodes of a tree

struct KeepLaunch {
  int* new_lens;
  PagedKv kv;
  PageTable table;
  int64_t layer_stride;
  int layers;
  const int *lens, *path, *counts;
  int n_new;
  hipStream_t stream;
};
hipError_t launch_keep(const KeepLaunch& L);

}  // namespace nrq
