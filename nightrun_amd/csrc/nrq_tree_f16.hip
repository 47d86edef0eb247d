// Attention of a tree's nodes over an f16 cache, and the dispatch by the cache's type.
#include "nrq_tree_attn.h"

namespace nrq {

hipError_t launch_tree_bf16(const PagedAttnLaunch& L);

double tree_attn_line(size_t seqs, size_t n_new, size_t heads, int n_kv, int64_t held) {
  return (double)(seqs * n_kv * ((n_new * (heads / n_kv) + 63) / 64)) * ((double)held / kTile + 1 + kTaSetup);
}

size_t tree_attn_workspace(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd) {
  const size_t rows = n_new * (heads / n_kv);
  // units of 64 rows at least; two parts a workgroup, of 128 rows at most where a CU has two workgroups, else of 256
  const size_t units = seqs * n_kv * ((rows + 63) / 64), slots = rows <= 128 ? 2 * rows : 256;
  return 2 * (size_t)kTaCus * slots * ((size_t)hd * sizeof(float) + sizeof(float2)) + 16 + units * sizeof(int4);
}

hipError_t launch_tree_attn(const PagedAttnLaunch& L) {
  return L.kv.dtype == kF16 ? ta_launch_type<_Float16>(L) : launch_tree_bf16(L);
}

}  // namespace nrq
