// Shared-prefix attention (attn_prefix.hpp): bfloat16.
#include "attn_prefix.hpp"

namespace pf {

hipError_t launch_prefix_bf16(const PrefixParams& p, int D, hipStream_t stream) {
  return prefix::launch_dim<bf16_t>(p, D, stream);
}

}  // namespace pf
