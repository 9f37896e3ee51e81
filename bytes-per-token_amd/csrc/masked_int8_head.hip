// Masked paged attention (masked_attention.h) over one cache format.
#include "masked_attention.h"

namespace bpt {

hipError_t launch_masked_int8_head(const MaskedParams& p, bool q_split, int rt, bool many, int grid, hipStream_t stream) {
  return q_split ? launch_masked_t<kKvInt8, kScaleHead, true>(p, rt, many, grid, stream)
                 : launch_masked_t<kKvInt8, kScaleHead, false>(p, rt, many, grid, stream);
}

}  // namespace bpt
