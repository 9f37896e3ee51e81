// Masked paged attention (masked_attention.h) over one cache format.
#include "masked_attention.h"

namespace bpt {

hipError_t launch_masked_bf16(const MaskedParams& p, bool q_split, int rt, bool many, int grid, hipStream_t stream) {
  return launch_masked<kKvBf16, kScaleNone>(p, q_split, rt, many, grid, stream);
}

}  // namespace bpt
