// Attention of a tree's nodes over a bf16 cache.
#include "nrq_paged.h"
#include "nrq_tree_launch.h"

namespace nrq {
hipError_t launch_tree_bf16(const PagedAttnLaunch& L) { return pa_launch_type<__bf16, true>(L); }
}  // namespace nrq
