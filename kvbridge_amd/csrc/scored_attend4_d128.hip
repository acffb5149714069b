// 4-bit cache, head size 128 (scored_attend.h).
#include "scored_attend.h"

namespace kvb {
hipError_t launch_attend4_d128(const ScoredArgs& a, hipStream_t stream) { return launch_attend_cache4<4>(a, stream); }
hipError_t preload_attend4_d128() { return preload_kernel(scored_attend_kernel<Cache4<4, 1>, 2, 2, true>); }
}  // namespace kvb
