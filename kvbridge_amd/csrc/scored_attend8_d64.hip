// 8-bit cache, head size 64 (scored_attend.h).
#include "scored_attend.h"

namespace kvb {
hipError_t launch_attend8_d64(const ScoredArgs& a, hipStream_t stream) {
  return launch_attend_cache<Cache8<2>>(a, stream);
}
hipError_t preload_attend8_d64() { return preload_kernel(scored_attend_kernel<Cache8<2>, 2, 2, true>); }
}  // namespace kvb
