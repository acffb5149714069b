// 4-bit cache, head size 128 (scored_attend.h).
#include "scored_attend.h"

namespace kvb {
hipError_t launch_attend4_d128(const ScoredArgs& a, hipStream_t stream) { return launch_attend_cache4<4>(a, stream); }
}  // namespace kvb
