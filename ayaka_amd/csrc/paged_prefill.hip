// Instantiations of the multi-row kernel (paged_prefill_kernel.h) for 16-bit caches and fp8 caches
// of the "fp8_e4m3" codec.
#include "paged_prefill_kernel.h"

namespace ayk {

// waves_per_group 1, 2, 4: tiles of the full capacity, a half, a quarter (4-wave workgroups);
// 0: the double tile (8-wave workgroups, head_dim 128 and 256).
template <int D>
static hipError_t launch_prefill_d(const AttnParams& p, const int32_t* tiles, dim3 grid, bool bf16, bool kv8,
                                   int waves_per_group, hipStream_t stream) {
  switch (waves_per_group) {
    case 0:
      if constexpr (D != 64) return launch_prefill_ps<D, 1, 8>(p, tiles, grid, bf16, kv8, stream);
      return hipErrorInvalidValue;
    case 1: return launch_prefill_ps<D, 1>(p, tiles, grid, bf16, kv8, stream);
    case 2: return launch_prefill_ps<D, 2>(p, tiles, grid, bf16, kv8, stream);
    case 4: return launch_prefill_ps<D, 4>(p, tiles, grid, bf16, kv8, stream);
    default: return hipErrorInvalidValue;
  }
}

int prefill_tile_pairs_for(int head_dim) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) ? prefill_tile_pairs(head_dim) : 0;
}

hipError_t launch_prefill(const AttnParams& p, const int32_t* tiles, int n_tiles, int head_dim, bool bf16, bool kv8,
                          int waves_per_group, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)n_tiles * (p.num_heads / p.group)));
  switch (head_dim) {
    case 64: return launch_prefill_d<64>(p, tiles, grid, bf16, kv8, waves_per_group, stream);
    case 128: return launch_prefill_d<128>(p, tiles, grid, bf16, kv8, waves_per_group, stream);
    case 256: return launch_prefill_d<256>(p, tiles, grid, bf16, kv8, waves_per_group, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ayk
