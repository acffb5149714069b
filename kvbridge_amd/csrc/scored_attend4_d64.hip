// 4-bit cache, head size 64 (scored_attend.h).
#include "scored_attend.h"

namespace kvb {
hipError_t launch_attend4_d64(const ScoredArgs& a, hipStream_t stream) { return launch_attend_cache4<2>(a, stream); }
}  // namespace kvb
