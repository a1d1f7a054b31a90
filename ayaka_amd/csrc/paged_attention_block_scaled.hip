// Instantiations of the matrix-core decode kernel (paged_attention_mfma_kernel.h) for block-scaled
// fp8 caches (codec "fp8_e4m3_block"), for decode rows and for windows.
#include "paged_attention_mfma_kernel.h"

namespace ayk {

template <int D>
static hipError_t launch_d(const AttnParams& p, int gc, bool bf16, bool split, hipStream_t stream) {
  return bf16 ? launch_mfma_gc<D, true, true, true>(p, gc, split, stream)
              : launch_mfma_gc<D, false, true, true>(p, gc, split, stream);
}

template <int D>
static hipError_t launch_window_d(const AttnParams& p, bool bf16, bool split, hipStream_t stream) {
  return bf16 ? launch_window_typed<D, true, true, true>(p, split, stream)
              : launch_window_typed<D, false, true, true>(p, split, stream);
}

hipError_t launch_attention_block_scaled(const AttnParams& p, int head_dim, int gc, bool bf16, bool split,
                                         hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_d<64>(p, gc, bf16, split, stream);
    case 128: return launch_d<128>(p, gc, bf16, split, stream);
    case 256: return launch_d<256>(p, gc, bf16, split, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_window_block_scaled(const AttnParams& p, int head_dim, bool bf16, bool split, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_window_d<64>(p, bf16, split, stream);
    case 128: return launch_window_d<128>(p, bf16, split, stream);
    case 256: return launch_window_d<256>(p, bf16, split, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ayk
