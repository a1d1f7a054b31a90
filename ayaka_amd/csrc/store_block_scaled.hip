// KV write into block-scaled fp8 caches (gfx950): encode a step's rows, raising their blocks'
// scales where they need it.
//
// Per block, key/value head and tensor (see ayaka_hip_block_scaled.h for the whole rule):
//   s' = max(s, 2^ceil(log2(max |x| / 448))),  new codes e4m3(x / s'),  held codes e4m3(c s / s').
//
// The rows of one block are one run of adjacent rows, and a wave owns a (run, head, tensor): it
// reads the run's slice of the rows, takes the largest magnitude over the wave, settles the scale,
// re-encodes the tokens held before the run if the scale grew, and encodes the rows. Nothing is
// shared between waves, so there is no atomic and no order to depend on.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ayaka_hip_internal.h"
#include "block_scale.h"
#include "kv_address.h"

namespace ayk {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// fp32 of magnitude 448 at most, or NaN, to an e4m3 code, to nearest even.
__device__ __forceinline__ uint32_t code_of(float f) {
  const uint32_t u = __float_as_uint(f);
  const uint32_t sign = (u >> 24) & 0x80u;
  const uint32_t mag = u & 0x7fffffffu;
  uint32_t code;
  if (mag > 0x7f800000u) code = 0x7fu;
  else if (mag < 0x3c800000u) code = (uint32_t)__builtin_rintf(__uint_as_float(mag) * 512.0f);  // below 2^-6
  else code = ((mag + 0x7ffffu + ((mag >> 20) & 1u)) >> 20) - (120u << 3);
  return code | sign;
}

template <bool BF16>
__device__ __forceinline__ float widen(uint32_t h) {
  if constexpr (BF16) return __uint_as_float(h << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// x / scale for the encoder: magnitudes above 448 saturate, what is not finite is NaN.
template <bool BF16>
__device__ __forceinline__ float scaled(uint32_t h, float inv) {
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  const float x = fminf(fmaxf(widen<BF16>(h) * inv, -448.f), 448.f);
  return (h & 0x7fffu) >= kInf ? __uint_as_float(0x7fc00000u) : x;
}

struct StoreParams {
  const uint16_t* rows[2];  // k, v
  uint8_t* cache[2];
  float* scales;
  const int64_t* slots;
  int64_t n_rows;
  int64_t num_slots;
  int64_t block_stride, token_stride, head_stride;  // bytes
  int32_t num_kv_heads, block_size;
  uint32_t bs_magic;
  int32_t bs_shift;
};

// Block of row i's slot, or 0 (padding) for a row that is dropped; and the offset in it.
__device__ __forceinline__ int slot_block(const StoreParams& p, int64_t i, int& offset) {
  const int64_t slot = p.slots[i];
  if (slot < p.block_size || slot >= p.num_slots) return 0;
  const uint32_t t = (uint32_t)slot;
  const int block = (int)((__umulhi(t, p.bs_magic) + t) >> p.bs_shift);
  offset = (int)(t - (uint32_t)block * (uint32_t)p.block_size);
  return block;
}

template <int D, bool BF16>
__global__ __launch_bounds__(256) void store_block_scaled_kernel(const StoreParams p) {
  constexpr int LPR = D / 8;     // lanes per row: 8 elements each
  constexpr int RPP = 64 / LPR;  // rows per pass of the wave
  const int lane = threadIdx.x & 63;
  const int unit = blockIdx.y * 4 + (threadIdx.x >> 6);  // (head, tensor)
  if (unit >= 2 * p.num_kv_heads) return;
  const int head = unit >> 1, which = unit & 1;
  const int64_t row0 = blockIdx.x;
  int offset = 0;
  const int block = slot_block(p, row0, offset);
  if (block == 0) return;
  int other = 0;
  if (row0 > 0 && slot_block(p, row0 - 1, other) == block) return;  // not the first row of its run
  // the run's length and its first offset
  int64_t count = 0;
  int first = p.block_size;
  for (bool more = true; more;) {
    const int64_t i = row0 + count + lane;
    int at = 0;
    const bool same = i < p.n_rows && slot_block(p, i, at) == block;
    const uint64_t mask = __builtin_amdgcn_ballot_w64(same);
    const int n = mask == ~0ull ? 64 : __builtin_ctzll(~mask);
    first = min(first, lane < n ? at : first);
    count += n;
    more = n == 64;
  }
#pragma unroll
  for (int st = 1; st < 64; st <<= 1) first = min(first, __shfl_xor(first, st));

  const int r = lane / LPR, c = lane % LPR;
  const int64_t row_elems = (int64_t)p.num_kv_heads * D;
  const uint16_t* src = p.rows[which] + row0 * row_elems + head * D + c * 8;
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0;
  for (int64_t i = r; i < count; i += RPP) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(src + i * row_elems);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = w[e] & 0x7fffu, hi = (w[e] >> 16) & 0x7fffu;
      top = max(top, lo < kInf ? lo : 0u);
      top = max(top, hi < kInf ? hi : 0u);
    }
  }
#pragma unroll
  for (int st = 1; st < 64; st <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, st));

  float* scale_at = p.scales + ((int64_t)block * p.num_kv_heads + head) * 2 + which;
  const float need = scale_for(widen<BF16>(top));
  const float old = first > 0 ? canonical_scale(*scale_at) : 0.f;
  const float now = fmaxf(old, need);
  uint8_t* dst = p.cache[which] + (int64_t)block * p.block_stride + head * p.head_stride + c * 8;
  if (now > old && old > 0.f) {
    const float ratio = old / now;  // a power of two: exact
    for (int t = r; t < first; t += RPP) {
      u32x2* at = reinterpret_cast<u32x2*>(dst + (int64_t)t * p.token_stride);
      u32x2 w = *at;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t out = 0;
        out |= code_of(__builtin_amdgcn_cvt_f32_fp8((int)w[e], 0) * ratio);
        out |= code_of(__builtin_amdgcn_cvt_f32_fp8((int)w[e], 1) * ratio) << 8;
        out |= code_of(__builtin_amdgcn_cvt_f32_fp8((int)w[e], 2) * ratio) << 16;
        out |= code_of(__builtin_amdgcn_cvt_f32_fp8((int)w[e], 3) * ratio) << 24;
        w[e] = out;
      }
      *at = w;
    }
  }
  const float inv = now > 0.f ? 1.0f / now : 1.0f;
  for (int64_t i = r; i < count; i += RPP) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(src + i * row_elems);
    int at = 0;
    slot_block(p, row0 + i, at);
    u32x2 out = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t pair = code_of(scaled<BF16>(w[e] & 0xffffu, inv)) | code_of(scaled<BF16>(w[e] >> 16, inv)) << 8;
      out[e >> 1] |= pair << (16 * (e & 1));
    }
    *reinterpret_cast<u32x2*>(dst + (int64_t)at * p.token_stride) = out;
  }
  if (lane == 0) *scale_at = now;
}

}  // namespace

hipError_t launch_store_block_scaled(const void* k, const void* v, void* k_cache, void* v_cache, float* scales,
                                     const int64_t* slot_mapping, int64_t n_rows, int32_t num_kv_heads,
                                     int32_t head_dim, int32_t num_blocks, int32_t block_size, uint32_t bs_magic,
                                     int32_t bs_shift, bool hnd, bool bf16, hipStream_t stream) {
  StoreParams p;
  p.rows[0] = static_cast<const uint16_t*>(k);
  p.rows[1] = static_cast<const uint16_t*>(v);
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.scales = scales;
  p.slots = slot_mapping;
  p.n_rows = n_rows;
  p.num_slots = (int64_t)num_blocks * block_size;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.bs_magic = bs_magic;
  p.bs_shift = bs_shift;
  const int64_t H = num_kv_heads, D = head_dim, B = block_size;
  p.block_stride = B * H * D;
  p.token_stride = hnd ? D : H * D;
  p.head_stride = hnd ? B * D : D;
  const dim3 grid((unsigned)n_rows, (unsigned)((2 * num_kv_heads + 3) / 4)), block(256);
#define AYK_STORE(W)                                                                                   \
  do {                                                                                                 \
    if (bf16) hipLaunchKernelGGL((store_block_scaled_kernel<W, true>), grid, block, 0, stream, p);     \
    else hipLaunchKernelGGL((store_block_scaled_kernel<W, false>), grid, block, 0, stream, p);         \
  } while (0)
  switch (head_dim) {
    case 64: AYK_STORE(64); break;
    case 128: AYK_STORE(128); break;
    case 256: AYK_STORE(256); break;
    default: return hipErrorInvalidValue;
  }
#undef AYK_STORE
  return hipGetLastError();
}

}  // namespace ayk
