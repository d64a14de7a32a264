// Shared-prefix attention, head dimension 256: see prefix_attention.h.
#include "prefix_attention.h"

namespace qw35 {

hipError_t launch_attn_d256(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream) {
    return attn::launch_dim<256>(a, bf16, f8, stream);
}

}  // namespace qw35
