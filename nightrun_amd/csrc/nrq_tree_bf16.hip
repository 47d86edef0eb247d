// Attention of a tree's nodes over a bf16 cache.
#include "nrq_tree_attn.h"

namespace nrq {
hipError_t launch_tree_bf16(const PagedAttnLaunch& L) { return ta_launch_type<__bf16>(L); }
}  // namespace nrq
