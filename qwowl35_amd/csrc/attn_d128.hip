// Shared-prefix attention, head dimension 128: see prefix_attention.h.
#include "prefix_attention.h"

namespace qw35 {

hipError_t launch_attn_d128(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream) {
    return attn::launch_dim<128>(a, bf16, f8, stream);
}

}  // namespace qw35
