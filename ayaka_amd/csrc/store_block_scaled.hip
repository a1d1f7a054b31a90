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
//
// Rows of a run of up to 16 positions stay in registers between the maximum and the encoding, one
// v_cvt_scalef32_pk_fp8 per two elements: it divides by the scale, rounds to nearest even and gives
// NaN for what is not finite, exactly as the codec says. A wave looks for the runs that begin among
// `range` rows. Blocks of up to 16 positions: a workgroup's waves are four heads, each on its own.
// Larger blocks (COOP): its waves are of one head and tensor; they share the runs of up to 16 rows
// out and take longer ones together, 16 rows each at a time, their maxima meeting in LDS.
//
// Bound by memory once a step is large: 16.4K rows of 8 heads of 128 move 101 MB in 21 us (4.8
// TB/s; a large copy makes 5.0). Small ones are one chain of loads: 4 us from 4 to 256 rows.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ayaka_hip_internal.h"
#include "block_scale.h"
#include "kv_address.h"

namespace ayk {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two elements, divided by the scale, to e4m3 codes in the low (HIGH: high) half of `to`.
template <bool BF16, bool HIGH>
__device__ __forceinline__ i16x2 encode_pair(i16x2 to, uint32_t w, float scale) {
  if constexpr (BF16)
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(to, __builtin_bit_cast(bf16x2, w), scale, HIGH);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(to, __builtin_bit_cast(f16x2, w), scale, HIGH);
}

// Four codes times a power of two below 1, to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t lower_codes(uint32_t codes, float ratio) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  int out = __builtin_amdgcn_cvt_pk_fp8_f32(a.x * ratio, a.y * ratio, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b.x * ratio, b.y * ratio, out, true);
}

// A 16-bit magnitude's value.
template <bool BF16>
__device__ __forceinline__ float widen(uint32_t h) {
  if constexpr (BF16) return __uint_as_float(h << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

template <int CTRL>
__device__ __forceinline__ uint32_t lane_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}

// The largest x of the wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, lane_dpp<0xB1>(x));   // quad_perm [1,0,3,2]: lane ^ 1
  x = max(x, lane_dpp<0x4E>(x));   // quad_perm [2,3,0,1]: lane ^ 2
  x = max(x, lane_dpp<0x141>(x));  // row_half_mirror: the other quad of the 8
  x = max(x, lane_dpp<0x140>(x));  // row_mirror: the other 8 of the 16
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(r[0], r[1]);
  const auto t = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(t[0], t[1]);
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

template <int D, bool BF16, bool COOP>
__global__ __launch_bounds__(256) void store_block_scaled_kernel(const StoreParams p, int range) {
  constexpr int LPR = D / 8;     // lanes per row: 8 elements each
  constexpr int RPP = 64 / LPR;  // rows per load of the wave
  constexpr int U = 16 / RPP;    // loads of 16 rows
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  __shared__ uint32_t s_top[2][4];  // COOP: the waves' maxima of a long run
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int unit = COOP ? blockIdx.y : blockIdx.y * 4 + wave;
  if (unit >= 2 * p.num_kv_heads) return;
  const int which = unit >= p.num_kv_heads ? 1 : 0, head = unit - which * p.num_kv_heads;
  // lane l looks at row row0 - 1 + l: the row before the range, the range, and what its last run may need
  const int64_t row0 = (int64_t)blockIdx.x * range;
  const int64_t mine = row0 - 1 + lane;
  int offset = 0;
  const int block = mine >= 0 && mine < p.n_rows ? slot_block(p, mine, offset) : 0;
  const int before = __shfl_up(block, 1);
  uint64_t runs = __builtin_amdgcn_ballot_w64(lane > 0 && lane <= range && block != 0 && block != before);

  const int r = lane / LPR, c = lane % LPR;
  const int64_t row_elems = (int64_t)p.num_kv_heads * D;
  int shared_out = 0, together = 0;  // COOP: runs of either kind so far (the same in every wave)
  for (; runs; runs &= runs - 1) {
    const int at = __builtin_ctzll(runs);
    const int blk = __builtin_amdgcn_readlane(block, at);
    const uint64_t same = __builtin_amdgcn_ballot_w64(block == blk) >> at;  // bits past lane 63 read as 0
    int64_t count = __builtin_ctzll(~same);
    uint32_t first = ~wave_max(lane >= at && lane < at + (int)count ? ~(uint32_t)offset : 0u);  // the least
    for (bool more = at + count == 64; more;) {  // a run longer than the wave sees
      const int64_t i = row0 - 1 + at + count + lane;
      int o = 0;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(i < p.n_rows && slot_block(p, i, o) == blk);
      const int n = mask == ~0ull ? 64 : __builtin_ctzll(~mask);
      first = min(first, ~wave_max(lane < n ? ~(uint32_t)o : 0u));
      count += n;
      more = n == 64;
    }
    // this wave's rows of the run: 16 from `begin` on, and `step` further on the next 16
    const bool split = COOP && count > 16;
    if (COOP && !split && (shared_out++ & 3) != wave) continue;
    const int64_t begin = split ? 16 * wave : 0, step = split ? 64 : 16;
    float* scale_at = p.scales + ((int64_t)blk * p.num_kv_heads + head) * 2 + which;
    const float stored = *scale_at;  // read beside the rows
    const uint16_t* src = p.rows[which] + (row0 - 1 + at) * row_elems + head * D + c * 8;
    uint8_t* dst = p.cache[which] + (int64_t)blk * p.block_stride + head * p.head_stride + c * 8;

    u32x4 w[U];
    auto load = [&](int64_t base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {  // past the run's end its last row again
        const int64_t i = base + u * RPP + r;
        w[u] = *reinterpret_cast<const u32x4*>(src + (i < count ? i : count - 1) * row_elems);
      }
    };
    auto largest = [&](bool finite) {
      u16x2 top = {0, 0};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u16x2 m = __builtin_bit_cast(u16x2, w[u][e] & 0x7fff7fffu);
          if (finite) {
            m.x = m.x < kInf ? m.x : 0;
            m.y = m.y < kInf ? m.y : 0;
          }
          top = __builtin_elementwise_max(top, m);
        }
      return (uint32_t)max(top.x, top.y);
    };
    // of the whole run, in every wave that has a part in it
    auto run_max = [&](uint32_t top) {
      top = wave_max(top);
      if (split) {
        uint32_t* all = s_top[together++ & 1];
        if (lane == 0) all[wave] = top;
        __syncthreads();
        top = max(max(all[0], all[1]), max(all[2], all[3]));
      }
      return top;
    };
    load(begin);
    uint32_t top = largest(false);
    for (int64_t base = begin + step; base < count; base += step) {
      load(base);
      top = max(top, largest(false));
    }
    top = run_max(top);
    const bool odd = top >= kInf;
    if (odd) {  // something is not finite: the finite values alone settle the scale
      top = 0;
      for (int64_t base = begin; base < count; base += step) {
        load(base);
        top = max(top, largest(true));
      }
      top = run_max(top);
    }
    const float old = first > 0 ? canonical_scale(stored) : 0.f;
    const float now = fmaxf(old, scale_for(widen<BF16>(top)));
    if (now > old && old > 0.f) {
      const float ratio = old / now;  // a power of two: exact
      for (int t = r + (split ? wave * RPP : 0); t < (int)first; t += split ? 4 * RPP : RPP) {
        u32x2* cell = reinterpret_cast<u32x2*>(dst + (int64_t)t * p.token_stride);
        const u32x2 codes = *cell;
        *cell = u32x2{lower_codes(codes.x, ratio), lower_codes(codes.y, ratio)};
      }
    }
    const float by = now > 0.f ? now : 1.f;
    // the largest scale: magnitudes past 448 of it saturate (bf16 values above 2^88 alone)
    const bool saturate = BF16 && now == power_of_two(kScaleMost);
    auto encode = [&](int64_t base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = base + u * RPP + r;
        int o = __shfl(offset, (at + (int)i) & 63);  // its lane's, where the wave saw the row
        if (i >= count) continue;
        if (at + i > 63) slot_block(p, row0 - 1 + at + i, o);
        u32x4 x = w[u];
        if (saturate) {
          constexpr uint32_t kMost = (uint32_t)(127 + 8 + kScaleMost) << 7 | 0x60u;  // 448 * 2^80 in bf16
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t lo = x[e] & 0x7fffu, hi = (x[e] >> 16) & 0x7fffu;
            lo = lo > kMost && lo < kInf ? kMost : lo;
            hi = hi > kMost && hi < kInf ? kMost : hi;
            x[e] = (x[e] & 0x80008000u) | lo | hi << 16;
          }
        }
        i16x2 lo = {0, 0}, hi = {0, 0};
        lo = encode_pair<BF16, false>(lo, x.x, by);
        lo = encode_pair<BF16, true>(lo, x.y, by);
        hi = encode_pair<BF16, false>(hi, x.z, by);
        hi = encode_pair<BF16, true>(hi, x.w, by);
        *reinterpret_cast<u32x2*>(dst + (int64_t)o * p.token_stride) =
            u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
      }
    };
    if (begin + step >= count && !odd) {  // the rows are still in registers
      encode(begin);
    } else {
      for (int64_t base = begin; base < count; base += step) {
        load(base);
        encode(base);
      }
    }
    if (lane == 0 && (!split || wave == 0)) *scale_at = now;
  }
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
  // Rows to a range. Few rows (a decode step): every run on a wave of its own, beside the others.
  // Many: as many as keep the waves that find no run to do few, for starting them is what such a step
  // then costs (16.4K rows of 8 heads of 128 that follow each other, us: blocks of 16, a wave to each
  // row 127, 4 rows 49, 16 rows 21; blocks of 64 and ranges of 16 47, of 32 27). Where each row
  // begins a run a long range does them one after the other (1024 such rows: 9.4, 8.7, 16.8), so
  // between the two a middle one. By the waves that one row each would take:
  const int64_t waves = n_rows * 2 * num_kv_heads;
  const bool coop = block_size > 16;
  const int range = coop ? (waves <= 8192 ? 4 : waves <= 32768 ? 16 : block_size <= 32 ? 32 : 63)
                         : (waves <= 8192 ? 1 : waves <= 32768 ? 4 : 16);
  const dim3 grid((unsigned)((n_rows + range - 1) / range),
                  (unsigned)(coop ? 2 * num_kv_heads : (2 * num_kv_heads + 3) / 4));
  const dim3 block(256);
#define AYK_STORE(W, C)                                                                                    \
  do {                                                                                                     \
    if (bf16) hipLaunchKernelGGL((store_block_scaled_kernel<W, true, C>), grid, block, 0, stream, p, range); \
    else hipLaunchKernelGGL((store_block_scaled_kernel<W, false, C>), grid, block, 0, stream, p, range);     \
  } while (0)
#define AYK_STORE_WIDTH(W)             \
  do {                                 \
    if (coop) AYK_STORE(W, true);      \
    else AYK_STORE(W, false);          \
  } while (0)
  switch (head_dim) {
    case 64: AYK_STORE_WIDTH(64); break;
    case 128: AYK_STORE_WIDTH(128); break;
    case 256: AYK_STORE_WIDTH(256); break;
    default: return hipErrorInvalidValue;
  }
#undef AYK_STORE_WIDTH
#undef AYK_STORE
  return hipGetLastError();
}

}  // namespace ayk
