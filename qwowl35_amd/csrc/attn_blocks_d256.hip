// Shared-prefix attention over a block-scaled cache, head dimension 256: see prefix_attention.h.
#include "prefix_attention.h"

namespace qw35 {

hipError_t launch_attn_blocks_d256(const AttnArgs& a, bool bf16, bool i8, hipStream_t stream) {
    return attn::launch_blocks<256>(a, bf16, i8, stream);
}

}  // namespace qw35
