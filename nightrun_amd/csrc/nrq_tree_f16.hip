// Attention of a tree's nodes over an f16 cache, and the dispatch by the cache's type.
#include "nrq_paged.h"
#include "nrq_tree_launch.h"

namespace nrq {

hipError_t launch_tree_bf16(const PagedAttnLaunch& L);

size_t tree_attn_workspace(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd) {
  return paged_attn_workspace(seqs, n_new, heads, n_kv, hd);
}

hipError_t launch_tree_attn(const PagedAttnLaunch& L) {
  return L.kv.dtype == kF16 ? pa_launch_type<_Float16, true>(L) : launch_tree_bf16(L);
}

}  // namespace nrq
