// Launch of the scored attention: the split kernel of the cache's format and
// head size, then the merge of the splits where there are several.
#include "scored_attend.h"

namespace kvb {

hipError_t launch_scored_attend(const ScoredArgs& a, hipStream_t stream) {
  hipError_t e;
  if (a.kv_bits == 4u)
    e = a.dim == 64u ? launch_attend4_d64(a, stream) : a.dim == 128u ? launch_attend4_d128(a, stream) : launch_attend4_d256(a, stream);
  else
    e = a.dim == 64u ? launch_attend8_d64(a, stream) : a.dim == 128u ? launch_attend8_d128(a, stream) : launch_attend8_d256(a, stream);
  if (e != hipSuccess || a.splits == 1u) return e;
  const uint32_t row_heads = a.batch * a.rows * a.q_heads;
  if (a.dim == 64u) scored_merge_kernel<64><<<row_heads, 256, 0, stream>>>(a);
  else if (a.dim == 128u) scored_merge_kernel<128><<<row_heads, 256, 0, stream>>>(a);
  else scored_merge_kernel<256><<<row_heads, 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace kvb
