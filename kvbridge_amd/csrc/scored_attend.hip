// Launch of the scored attention: the split kernel of the cache's format and
// head size, which merges the splits itself where counters are given; else a
// second launch does.
#include "scored_attend.h"

namespace kvb {

hipError_t launch_scored_attend(const ScoredArgs& a, hipStream_t stream) {
  hipError_t e;
  if (a.kv_bits == 4u)
    e = a.dim == 64u ? launch_attend4_d64(a, stream) : a.dim == 128u ? launch_attend4_d128(a, stream) : launch_attend4_d256(a, stream);
  else
    e = a.dim == 64u ? launch_attend8_d64(a, stream) : a.dim == 128u ? launch_attend8_d128(a, stream) : launch_attend8_d256(a, stream);
  if (e != hipSuccess || a.items == a.batch || a.counters) return e;  // an item each: nothing to merge
  const uint32_t groups = a.batch * a.kv_heads * a.head_rows;
  if (a.dim == 64u) scored_merge_kernel<64><<<groups, 256, sizeof(MergeLds) + 256u * 16u, stream>>>(a);
  else if (a.dim == 128u) scored_merge_kernel<128><<<groups, 256, sizeof(MergeLds) + 256u * 16u, stream>>>(a);
  else scored_merge_kernel<256><<<groups, 256, sizeof(MergeLds) + 256u * 16u, stream>>>(a);
  return hipGetLastError();
}

hipError_t preload_scored() {
  hipError_t (*const units[])() = {preload_attend4_d64,  preload_attend4_d128,  preload_attend4_d256, preload_attend8_d64,
                                   preload_attend8_d128, preload_attend8_d256, preload_scored_weights, preload_cache4, preload_evict};
  for (const auto unit : units)
    if (const hipError_t e = unit(); e != hipSuccess) return e;
  return preload_kernel(scored_merge_kernel<64>);
}

}  // namespace kvb
