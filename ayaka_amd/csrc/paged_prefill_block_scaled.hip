// Instantiations of the multi-row kernel (paged_prefill_kernel.h) for block-scaled fp8 caches (codec
// "fp8_e4m3_block"); waves_per_group as for launch_prefill.
#include "paged_prefill_kernel.h"

namespace ayk {

template <int D>
static hipError_t launch_d(const AttnParams& p, const int32_t* tiles, dim3 grid, bool bf16, int waves_per_group,
                           hipStream_t stream) {
  switch (waves_per_group) {
    case 0:
      if constexpr (D != 64) return launch_prefill_ps_block_scaled<D, 1, 8>(p, tiles, grid, bf16, stream);
      return hipErrorInvalidValue;
    case 1: return launch_prefill_ps_block_scaled<D, 1>(p, tiles, grid, bf16, stream);
    case 2: return launch_prefill_ps_block_scaled<D, 2>(p, tiles, grid, bf16, stream);
    case 4: return launch_prefill_ps_block_scaled<D, 4>(p, tiles, grid, bf16, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_prefill_block_scaled(const AttnParams& p, const int32_t* tiles, int n_tiles, int head_dim, bool bf16,
                                       int waves_per_group, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)n_tiles * (p.num_heads / p.group)));
  switch (head_dim) {
    case 64: return launch_d<64>(p, tiles, grid, bf16, waves_per_group, stream);
    case 128: return launch_d<128>(p, tiles, grid, bf16, waves_per_group, stream);
    case 256: return launch_d<256>(p, tiles, grid, bf16, waves_per_group, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ayk
