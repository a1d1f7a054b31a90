// Instantiations of the matrix-core decode kernel (paged_attention_mfma_kernel.h) for 16-bit caches
// and fp8 caches of the "fp8_e4m3" codec, for decode rows and for windows.
#include "paged_attention_mfma_kernel.h"

namespace ayk {

template <int D>
static hipError_t launch_mfma_d(const AttnParams& p, int gc, bool bf16, bool split, bool kv8, hipStream_t stream) {
  if (kv8) return bf16 ? launch_mfma_gc<D, true, true>(p, gc, split, stream)
                       : launch_mfma_gc<D, false, true>(p, gc, split, stream);
  return bf16 ? launch_mfma_gc<D, true, false>(p, gc, split, stream)
              : launch_mfma_gc<D, false, false>(p, gc, split, stream);
}

hipError_t launch_window_mfma(const AttnParams& p, int head_dim, bool bf16, bool split, bool kv8, hipStream_t stream) {
  switch (head_dim) {
    case 64:
      if (kv8) return bf16 ? launch_window_typed<64, true, true>(p, split, stream)
                           : launch_window_typed<64, false, true>(p, split, stream);
      return bf16 ? launch_window_typed<64, true, false>(p, split, stream)
                  : launch_window_typed<64, false, false>(p, split, stream);
    case 128:
      if (kv8) return bf16 ? launch_window_typed<128, true, true>(p, split, stream)
                           : launch_window_typed<128, false, true>(p, split, stream);
      return bf16 ? launch_window_typed<128, true, false>(p, split, stream)
                  : launch_window_typed<128, false, false>(p, split, stream);
    case 256:
      if (kv8) return bf16 ? launch_window_typed<256, true, true>(p, split, stream)
                           : launch_window_typed<256, false, true>(p, split, stream);
      return bf16 ? launch_window_typed<256, true, false>(p, split, stream)
                  : launch_window_typed<256, false, false>(p, split, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attention_mfma(const AttnParams& p, int head_dim, int gc, bool bf16, bool split, bool kv8,
                                 int waves, hipStream_t stream) {
  (void)waves;
  switch (head_dim) {
    case 64: return launch_mfma_d<64>(p, gc, bf16, split, kv8, stream);
    case 128: return launch_mfma_d<128>(p, gc, bf16, split, kv8, stream);
    case 256: return launch_mfma_d<256>(p, gc, bf16, split, kv8, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ayk
