// Masked paged attention (masked_attention.h) over one cache format.
#include "masked_attention.h"

namespace bpt {

hipError_t launch_masked_bf16(const MaskedParams& p, bool q_split, int rt, bool many, int grid, hipStream_t stream) {
  return q_split ? launch_masked_t<kKvBf16, kScaleNone, true>(p, rt, many, grid, stream)
                 : launch_masked_t<kKvBf16, kScaleNone, false>(p, rt, many, grid, stream);
}

}  // namespace bpt
