// Paged attention over an f16 cache, and the dispatch by the cache's type.
#include "nrq_paged.h"

namespace nrq {

hipError_t launch_paged_bf16(const PagedAttnLaunch& L);

size_t paged_attn_units(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd) {
  const size_t rows = n_new * (heads / n_kv), per = pa_per(hd, rows);
  return seqs * n_kv * ((rows + per - 1) / per);
}

size_t paged_attn_workspace(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd) {
  const size_t rows = n_new * (heads / n_kv), per = pa_per(hd, rows), units = paged_attn_units(seqs, n_new, heads, n_kv, hd);
  return 2 * (size_t)kPaMaxWgs * (rows < per ? rows : per) * ((size_t)hd * sizeof(float) + sizeof(float2)) + 16 +
         units * sizeof(int4);
}

hipError_t launch_paged_attn(const PagedAttnLaunch& L) {
  return L.kv.dtype == kF16 ? pa_launch_type<_Float16>(L) : launch_paged_bf16(L);
}

}  // namespace nrq
