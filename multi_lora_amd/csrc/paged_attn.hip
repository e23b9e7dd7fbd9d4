// Attention over pages of 16-bit numbers: the kernels of paged_attn.h.
#include "paged_attn.h"

namespace mlora {

hipError_t launch_paged_attention(const PagedAttnArgs& a, int max_new, int dtype, int head_dim, hipStream_t stream) {
  return launch_of<false>(a, max_new, dtype, head_dim, stream);
}

}  // namespace mlora
