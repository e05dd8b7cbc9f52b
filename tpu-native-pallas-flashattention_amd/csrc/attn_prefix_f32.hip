// Shared-prefix attention (attn_prefix.hpp): float32.
#include "attn_prefix.hpp"

namespace pf {

hipError_t launch_prefix_f32(const PrefixParams& p, int D, hipStream_t stream) {
  return prefix::launch_dim<float>(p, D, stream);
}

}  // namespace pf
