// Attention over pages of 8-bit codes with block exponents: the kernels of paged_attn.h.
#include "paged_attn.h"

namespace mlora {

hipError_t launch_paged_attention8(const PagedAttnArgs& a, int max_new, int dtype, int head_dim, hipStream_t stream) {
  return launch_of<true>(a, max_new, dtype, head_dim, stream);
}

}  // namespace mlora
