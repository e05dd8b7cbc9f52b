// Shared-prefix attention (attn_prefix.hpp): float16.
#include "attn_prefix.hpp"

namespace pf {

hipError_t launch_prefix_f16(const PrefixParams& p, int D, hipStream_t stream) {
  return prefix::launch_dim<f16_t>(p, D, stream);
}

}  // namespace pf
