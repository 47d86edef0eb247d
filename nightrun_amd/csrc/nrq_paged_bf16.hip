// Paged attention over a bf16 cache.
#include "nrq_paged.h"

namespace nrq {
hipError_t launch_paged_bf16(const PagedAttnLaunch& L) { return pa_launch_type<__bf16>(L); }
}  // namespace nrq
