// Masked paged attention (masked_attention.h) over one cache format.
#include "masked_attention.h"

namespace bpt {

hipError_t launch_masked_fp8_token(const MaskedParams& p, bool q_split, int rt, bool many, int grid, hipStream_t stream) {
  return launch_masked<kKvFp8, kScaleTokenHead>(p, q_split, rt, many, grid, stream);
}

}  // namespace bpt
