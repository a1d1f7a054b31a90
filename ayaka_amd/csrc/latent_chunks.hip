// Attention of chunks of new tokens over a latent cache, expanded form (gfx950).
//
//   k[h, t] = [keys[h] latent_t | rotary part_t],  v[h, t] = values[h] latent_t,
//   out[row, h] = softmax(scale * q[row, h] . k[h, .]) v[h, .]   over positions 0 .. position(row).
// A (row, head, position) takes 2 (192 + 128) operations so, against 2 (2 DC + 64) on the latents
// themselves (a third at DC 512); expanding takes 2 * 256 * DC per (head, position), once for all rows.
//
// Two kernels, for as many heads at a time as the workspace holds:
//
// latent_expand_kernel: a product of 128 tokens by one head's 256 outputs (its keys, then its values),
// 8 waves of 64 x 64 on v_mfma_f32_16x16x32, operands through LDS in steps of 32 of DC, three steps in
// flight (global_load_lds, 74 KB). Two workgroups share a compute unit, so that one's first loads and
// stores run beside the other's products: with one of twice the step 16384 tokens for 16 heads at DC 512
// took 95 us at their best, so 80 (0.86 PFLOP/s, and 134 MB written; 92 at the median of 20 launches from rest, as
// the card lowers its clock). Tokens are gathered from their pages here; what follows reads straight lines.
//
// Keys and values are kept as fp16 whatever the model's type, with a power of two for every 128 tokens,
// head and of both kinds, chosen from the largest finite value there, so nothing overflows and each
// element is within 2^-11 of itself (or 2^-38 of its tile's largest): bf16 keys and values would each
// cost the outputs as much as their own rounding does. The key's scale joins the factor that scores take
// anyway. The value's, 2^e of a tile, meets a reference of each row's own: beside a reference m for its scores
// (kWeightLift under a running maximum) a row keeps a level E, about the largest score + e so far less that maximum, and
//   O = sum_t 2^(score_t - m + e_t - E) code_t,   l = sum_t 2^(score_t - m),   out = 2^E O / l.
// Weights are at most 2^15 with the scale and without it, tiles that weigh nothing cost nothing however
// loud they are, and the sum never sees a scale. E and e are whole, so where they agree, as they do for most
// tiles, a weight is one exponential, and elsewhere it is multiplied by a power of two.
//
// latent_chunk_kernel: a workgroup (8 waves) per 128 rows of a request and head. Four waves of 32 rows
// work on every other 32 positions and four on those between (two waves to a SIMD); joined at the end in
// LDS. S^T = K Q^T, weights stay in the lane that scored them, O^T += V^T P^T with values read
// transposed, as the other attention kernels. Rounds of 64 positions (40 KB) in a ring of three.
// Where row tiles and heads are fewer than the compute units the caller has each tile's context cut into parts,
// a workgroup each, which latent_join_kernel joins: chunks of 600 rows of 4 heads over 3.6K positions take 42 us
// so, 85 whole.
// Bound by issue, not by memory: the loads alone take 34 us where 4 requests of 512 rows over 4096
// positions, 16 heads, take 112 at their best and 131 at the median (0.72 and 0.61 PFLOP/s in the causal part). Of
// about 3100 cycles a round 1280 are matrix instructions and as many vector ones, and exponentials do not run beside matrix
// instructions of the same SIMD (alone 8.7 cycles each; beside a wave of products they wait for its
// end). Measured and left: the waves of a SIMD half a round apart, keys read a round ahead, both
// within 3% of this and longer.
#include <type_traits>

#include "attention_common.h"

namespace ayk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr int kRope = 64;
constexpr int kNope = 128;
constexpr int kValue = 128;
constexpr int kTokens = kLatentChunkTokens;  // of an expanded tile, with one scale
constexpr int kRows = kLatentChunkRows;      // of a workgroup
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;

template <bool BF16>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 acc) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
}

__device__ __forceinline__ uint32_t quotient(uint32_t n, Divisor d) {
  return (uint32_t)(((uint64_t)__umulhi(n, d.magic) + n) >> d.shift);
}

// Rounded by itself, never part of an fma.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// 16 bytes a lane to LDS at `to` + 16 * lane (`to` uniform).
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint8_t* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint8_t* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <class T>
__device__ __forceinline__ uint32_t lds_offset(T* p) {
  return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) T*)p);
}

// Where piece c (16 bytes) of row r stands in LDS, for rows of 64, 128 and 256 bytes: any 16 rows that
// one cycle's reads touch are spread over all 64 banks.
__device__ __forceinline__ int swizzle64(int r) { return (r >> 1) & 3; }
__device__ __forceinline__ int swizzle128(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swizzle256(int r) { return r & 15; }

// The even power of two that brings a largest magnitude into [2^13, 2^15). (Even: tiles alike in magnitude share theirs
// more often, and the attention multiplies weights where a tile's is not the row's: 16 heads of 4 chunks over 4096
// positions take 176 us where all tiles share one and 185 where two are mixed, and latents drawn alike are mixed at a
// quarter of their magnitudes so, at half of them with powers of any kind.)
__device__ __forceinline__ int exponent_for(float largest) {
  if (largest == 0.f) return -100;
  return max(-100, min(114, ((int)((__float_as_uint(largest) >> 23) & 255) - 126 - 14) & ~1));
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// 2^x for x up to 0 as part * 2^whole: past fp32's least too, and times another power of two as exact as by itself.
struct Power {
  float part;
  int whole;
};
__device__ __forceinline__ Power power_of(float x) {
  const float whole = __builtin_rintf(fmaxf(x, -1000.f));
  return Power{fast_exp2(x - whole), (int)whole};
}
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = __builtin_fabsf(x);
  return a < INFINITY ? a : 0.f;  // (also where it is NaN)
}
__device__ __forceinline__ uint32_t two_halves(float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// --- expansion

constexpr int kStep = 32;        // of DC in LDS at a time
constexpr int kSteps = 3;        // in flight
constexpr int kOutputs = kNope + kValue;

template <int DC, bool BF16>
__global__ __launch_bounds__(kThreads, 4) void latent_expand_kernel(const LatentChunkParams p) {
  struct Shared {
    uint16_t token[kSteps][kTokens * kStep];
    uint16_t weight[kSteps][kOutputs * kStep];
    float largest[kWaves];
    int32_t infinite[kWaves];  // not 0: among a wave's elements is one that is not finite
  };
  __shared__ __align__(16) Shared lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mt = lane & 15, mq = lane >> 4;
  const int head = blockIdx.x % p.group_heads, tile = blockIdx.x / p.group_heads;
  const int request = p.token_tiles[4 * tile], first = p.token_tiles[4 * tile + 1], length = p.token_tiles[4 * tile + 2];
  const int64_t ws_row = p.token_tiles[4 * tile + 3];
  const int real_head = p.first_head + head;

  auto slot_of = [&](int row) {
    const uint32_t pos = (uint32_t)min(first + row, length - 1);
    const uint32_t block = quotient(pos, p.by_block);
    const uint32_t id = (uint32_t)p.block_table[request * p.table_stride + block];
    return reinterpret_cast<const uint8_t*>(p.cache) +
           ((uint64_t)(id < (uint32_t)p.num_blocks ? id : 0u) * (uint32_t)p.block_size + (pos - block * (uint32_t)p.block_size)) * ((DC + kRope) * 2);
  };
  // What this wave fetches of each step, 16 rows a load: 16 tokens and 32 outputs.
  const uint8_t* from[3];
  const int row16 = lane >> 2, piece16 = ((lane & 3) ^ swizzle64(row16)) * 16;
  from[0] = slot_of(wave * 16 + row16) + piece16;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = wave * 32 + i * 16 + row16;
    const uint16_t* w = row < kNope ? p.keys + ((int64_t)real_head * kNope + row) * DC
                                    : p.values + ((int64_t)real_head * kValue + row - kNope) * DC;
    from[1 + i] = reinterpret_cast<const uint8_t*>(w) + piece16;
  }
  const uint32_t token_lds = lds_offset(&lds.token[0][0]), weight_lds = lds_offset(&lds.weight[0][0]);
  auto get = [&](int step) {
    const uint32_t s = (uint32_t)(step % kSteps);
    load_to_lds(token_lds + s * (kTokens * kStep * 2) + wave * 16 * (kStep * 2), from[0] + step * (kStep * 2));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      load_to_lds(weight_lds + s * (kOutputs * kStep * 2) + (wave * 32 + i * 16) * (kStep * 2), from[1 + i] + step * (kStep * 2));
  };
  // the rotary parts go along once, from the first head's workgroups
  if (real_head == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = wave * 16 + i * 8 + (lane >> 3);
      *reinterpret_cast<u32x4*>(p.ws_rope + (ws_row + row) * kRope + (lane & 7) * 8) =
          *reinterpret_cast<const u32x4*>(slot_of(row) + DC * 2 + (lane & 7) * 16);
    }
  }

  // Outputs are the product's rows and tokens its columns, so that a lane holds 4 outputs of a token.
  const int m = wave & 1, n = wave >> 1;  // 64 tokens, 64 outputs
  f32x4 acc[4][4];  // [outputs][tokens]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int STEPS = DC / kStep;
  get(0);
  get(1);
#pragma unroll
  for (int step = 0; step < STEPS; ++step) {
    if (step + 1 < STEPS) wait_loads<3>();
    else wait_loads<0>();
    lds_barrier();
    if (step + 2 < STEPS) get(step + 2);
    const uint8_t* token = reinterpret_cast<const uint8_t*>(lds.token[step % kSteps]) + m * 64 * kStep * 2;
    const uint8_t* weight = reinterpret_cast<const uint8_t*>(lds.weight[step % kSteps]) + n * 64 * kStep * 2;
    u32x4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (i * 16 + mt) * (kStep * 2) + (mq ^ swizzle64(mt)) * 16;
      a[i] = *reinterpret_cast<const u32x4*>(weight + at);
      b[i] = *reinterpret_cast<const u32x4*>(token + at);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma32<BF16>(a[i], b[j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }

  // The scale of the tile's keys (waves 0-3) and of its values (4-7).
  float largest = 0.f;
  bool infinite = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        largest = fmaxf(largest, finite_magnitude(acc[i][j][e]));
        infinite |= !(__builtin_fabsf(acc[i][j][e]) < INFINITY);
      }
  infinite = __builtin_amdgcn_ballot_w64(infinite) != 0;
  largest = column_max(largest);
#pragma unroll
  for (int d = 8; d >= 1; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
  if (lane == 0) lds.largest[wave] = largest, lds.infinite[wave] = infinite;
  lds_barrier();
  const int half = n >> 1;  // keys, values
  largest = fmaxf(fmaxf(lds.largest[4 * half], lds.largest[4 * half + 1]), fmaxf(lds.largest[4 * half + 2], lds.largest[4 * half + 3]));
  const int exponent = exponent_for(largest);
  infinite = lds.infinite[4 * half] | lds.infinite[4 * half + 1] | lds.infinite[4 * half + 2] | lds.infinite[4 * half + 3];
  const float by = power(-exponent);
  // Through LDS (rows of 512 bytes, as tokens; every wave is past its last read), then whole rows out.
  uint8_t* rows = reinterpret_cast<uint8_t*>(&lds.token[0][0]);
  static_assert(offsetof(Shared, largest) >= kTokens * kOutputs * 2, "the tile fits where the operands were");
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int token = m * 64 + j * 16 + mt, output = n * 64 + i * 16 + 4 * mq;
      const u32x2 x = {two_halves(acc[i][j][0] * by, acc[i][j][1] * by), two_halves(acc[i][j][2] * by, acc[i][j][3] * by)};
      *reinterpret_cast<u32x2*>(rows + token * (kOutputs * 2) + (((output >> 3) ^ swizzle256(token)) * 16) + (output & 4) * 2) = x;
    }
  lds_barrier();
  const int64_t ws = (int64_t)head * p.ws_rows + ws_row;
#pragma unroll
  for (int i = 0; i < kTokens * kOutputs / 8 / kThreads; ++i) {
    const int at = i * kThreads + tid, token = at >> 5, piece = at & 31;
    const u32x4 x = *reinterpret_cast<const u32x4*>(rows + token * (kOutputs * 2) + ((piece ^ swizzle256(token)) * 16));
    uint16_t* to = piece < 16 ? p.ws_keys : p.ws_values;
    *reinterpret_cast<u32x4*>(to + (ws + token) * kNope + (piece & 15) * 8) = x;
  }
  if (tid == 0 || tid == 4 * kWave) p.ws_exponents[(head * (p.ws_rows / kTokens) + ws_row / kTokens) * 2 + half] = 2 * exponent + infinite;
}

// --- attention

constexpr int kPositions = 32;            // of a wave's step
constexpr int kRound = 2 * kPositions;    // of both halves of the workgroup
constexpr int kRing = 3;
constexpr int kWindow = 256;  // tiles whose exponents wait in LDS
constexpr float kPasses = kWeightLift + kRescaleSlack;  // from a row's reference to where a score moves it

struct Round {
  uint16_t keys[kRound * kNope];
  uint16_t values[kRound * kValue];
  uint16_t rope[kRound * kRope];
};

template <bool BF16>
__global__ __launch_bounds__(kThreads, 1) void latent_chunk_kernel(const LatentChunkParams p) {
  struct Shared {
    Round round[kRing];
    float state[4][2][3][16];  // (m, l, level) of the later half's rows
    int32_t exponent[kWindow][2];  // of the tiles being read: twice that, and 1 where an element is not finite
  };
  __shared__ __align__(16) Shared lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mt = lane & 15, mq = lane >> 4;
  const int rg = wave & 3, kg = wave >> 2;  // 32 rows, every other 32 positions
  const int head = blockIdx.x % p.group_heads, tile = blockIdx.x / p.group_heads;
  const int first_row = p.row_tiles[4 * tile], n_rows = p.row_tiles[4 * tile + 1], first_pos = p.row_tiles[4 * tile + 3];
  const int64_t ws_row = p.row_tiles[4 * tile + 2];
  const int real_head = p.first_head + head;
  const int context = first_pos + n_rows;  // positions that the last row sees
  // this workgroup's part of the context
  const int all_rounds = (context + kRound - 1) / kRound;
  const int first_round = (int)((int64_t)blockIdx.y * all_rounds / p.splits);
  const int rounds = (int)((int64_t)(blockIdx.y + 1) * all_rounds / p.splits);

  const uint8_t* keys = reinterpret_cast<const uint8_t*>(p.ws_keys + ((int64_t)head * p.ws_rows + ws_row) * kNope);
  const uint8_t* values = reinterpret_cast<const uint8_t*>(p.ws_values + ((int64_t)head * p.ws_rows + ws_row) * kValue);
  const uint8_t* rope = reinterpret_cast<const uint8_t*>(p.ws_rope + ws_row * kRope);
  const int32_t* exponents = p.ws_exponents + (head * (p.ws_rows / kTokens) + ws_row / kTokens) * 2;
  const uint32_t ring = lds_offset(&lds.round[0]);
  // a wave's loads of a round: 8 rows of keys, of values (4 a load) and of rotary parts (8 a load)
  uint32_t at[3];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = wave * 8 + i * 4 + (lane >> 4);
    at[i] = row * 256 + ((lane & 15) ^ swizzle256(row)) * 16;
  }
  at[2] = (wave * 8 + (lane >> 3)) * 128 + ((lane & 7) ^ swizzle128(wave * 8 + (lane >> 3))) * 16;
  auto get = [&](int round) {
    const uint32_t to = ring + (uint32_t)(round % kRing) * sizeof(Round) + wave * 8 * 256;
    const int64_t from = (int64_t)round * kRound * 256;
#pragma unroll
    for (int i = 0; i < 2; ++i) load_to_lds(to + i * 1024, keys + from, at[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) load_to_lds(to + kRound * 256 + i * 1024, values + from, at[i]);
    load_to_lds(ring + (uint32_t)(round % kRing) * sizeof(Round) + 2 * kRound * 256 + wave * 8 * 128, rope + from / 2, at[2]);
  };
  constexpr int LOADS = 5;

  // The queries: 16 rows a tile, their first part as fp16 under a power of two of each row's own.
  u32x4 q[2][4], qr[2][2];
  int unit[2];  // the power of two that a raw score of the first part is worth, but for the keys'
  int my_pos[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = rg * 32 + j * 16 + mt;
    my_pos[j] = row < n_rows ? first_pos + row : -1;
    const u32x4* from =
        reinterpret_cast<const u32x4*>(p.q + ((int64_t)(first_row + (row < n_rows ? row : 0)) * p.heads + real_head) * (kNope + kRope)) + mq;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[j][k] = from[4 * k];
#pragma unroll
    for (int k = 0; k < 2; ++k) qr[j][k] = from[16 + 4 * k];
  }
  if (first_round < rounds) get(first_round);
  if (first_round + 1 < rounds) get(first_round + 1);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float largest = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        largest = fmaxf(largest, fmaxf(finite_magnitude(Elem<BF16>::lo(q[j][k][e])), finite_magnitude(Elem<BF16>::hi(q[j][k][e]))));
    const int exponent = exponent_for(column_max(largest));
    const float by = power(-exponent);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[j][k][e] = two_halves(Elem<BF16>::lo(q[j][k][e]) * by, Elem<BF16>::hi(q[j][k][e]) * by);
    unit[j] = exponent;
  }
  const bool loud = __builtin_amdgcn_ballot_w64(unit[0] > 127 - 114 || unit[1] > 127 - 114) != 0;  // (keys: up to 114)
  f32x4 o[8][2];
  float m[2], l[2], level[2];  // (level: whole; of O, where m is a number)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.f;
    level[j] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int k_at[4], r_at[2], v_at[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) k_at[i] = mt * 256 + ((4 * i + mq) ^ swizzle256(mt)) * 16;
#pragma unroll
  for (int i = 0; i < 2; ++i) r_at[i] = 2 * kRound * 256 + mt * 128 + ((4 * i + mq) ^ swizzle128(mt)) * 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = 4 * mq + (mt >> 2);
    v_at[i] = kRound * 256 + t * 256 + ((2 * i + ((mt & 3) >> 1)) ^ swizzle256(t)) * 16 + (mt & 1) * 8;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt 0, said to the compiler: its waits for the queries end here
  // Scores stay as the products give them, to be scaled inside the exponent, but for rows whose maximum
  // is so large that one scaled and rounded by itself and one scaled in an fma could be whole powers of
  // two apart, and for a negative scale.
  bool far[2] = {p.scale_log2 < 0.f, p.scale_log2 < 0.f};
  bool any_far = p.scale_log2 < 0.f;

  const int first_masked = first_pos + rg * 32;  // rows of this wave see up to there, all of them
  for (int round = first_round; round < rounds; ++round) {
    if (round + 1 < rounds) wait_loads<LOADS>();
    else wait_loads<0>();
    lds_barrier();
    if (round == first_round || round % (kWindow * kTokens / kRound) == 0) {
      // The exponents come by way of LDS: a load of the compiler's own in every round would make it wait
      // there for all the loads to LDS that are on their way.
      const int first = round / (kTokens / kRound) / kWindow * kWindow, n = min(kWindow, (context + kTokens - 1) / kTokens - first);
      for (int i = tid; i < 2 * n; i += kThreads) lds.exponent[i >> 1][i & 1] = exponents[2 * first + i];
      lds_barrier();
    }
    if (round + 2 < rounds) get(round + 2);
    const int t0 = round * kRound + kg * kPositions;
    if (t0 >= context || t0 > first_masked + 31) continue;  // nothing for these rows
    const uint8_t* here = reinterpret_cast<const uint8_t*>(&lds.round[round % kRing]);
    const uint8_t* k_here = here + kg * kPositions * 256;
    const uint8_t* r_here = here + kg * kPositions * 128;
    const int key_exponent = __builtin_amdgcn_readfirstlane(lds.exponent[t0 / kTokens % kWindow][0]) >> 1;
    const int value_word = __builtin_amdgcn_readfirstlane(lds.exponent[t0 / kTokens % kWindow][1]);
    const float exponent = (float)(value_word >> 1);

    f32x4 s[2][2], r[2][2];  // [16 positions][16 rows], of the first part and of the rotary part
    u32x4 a[2][6];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 4; ++k) a[h][k] = *reinterpret_cast<const u32x4*>(k_here + h * 16 * 256 + k_at[k]);
#pragma unroll
      for (int k = 0; k < 2; ++k) a[h][4 + k] = *reinterpret_cast<const u32x4*>(r_here + h * 16 * 128 + r_at[k]);
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 v[8];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        r[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) s[h][j] = mfma32<false>(a[h][k], q[j][k], s[h][j]);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) r[h][j] = mfma32<BF16>(a[h][4 + k], qr[j][k], r[h][j]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint16_t* from = reinterpret_cast<const uint16_t*>(k_here + v_at[d]);
      const u32x2 x = lds_read_transposed(from), y = lds_read_transposed(from + 16 * kValue);
      v[d] = u32x4{x.x, x.y, y.x, y.y};
    }
    __builtin_amdgcn_sched_barrier(0);

    const bool masked = t0 + kPositions - 1 > first_masked;
    float by[2] = {p.scale_log2, p.scale_log2};  // of what s holds from here on
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      int up = unit[j] + key_exponent;
      if (loud) {  // past the largest power of two the factor comes in two, so that products of 0 stay 0
        const int first = max(0, up - 127);
        up -= first;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][j][i] = __builtin_ldexpf(s[h][j][i], first);
      }
      const float ratio = __builtin_ldexpf(1.f, up);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][j][i] = __builtin_fmaf(s[h][j][i], ratio, r[h][j][i]);
    }
    if (masked || any_far) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int seen = my_pos[j] - t0 - 4 * mq;
        const bool whole = masked || far[j];
        by[j] = whole ? 1.f : p.scale_log2;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[h][j][i] = 16 * h + i <= seen ? (whole ? product(s[h][j][i], p.scale_log2) : s[h][j][i]) : -INFINITY;
      }
    }
    if (masked && (value_word & 1)) {
      // Values that are not finite become zeros, behind NaN for the rows that see them. (What says so are the values
      // themselves: a finite latent may take one past the range of fp32 and leave its key and every score alone.)
      const uint8_t* mine = here + kRound * 256 + kg * kPositions * 256;
#pragma unroll 1
      for (int t = 0; t < kPositions; ++t) {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(mine + t * 256 + ((2 * d + (mq >> 1)) ^ swizzle256(t)) * 16 + (mq & 1) * 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool off = ((i & 2 ? x.y : x.x) >> (16 * (i & 1)) & 0x7c00u) == 0x7c00u;
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (off && t0 + t <= my_pos[j]) o[d][j][i] = NAN;
          }
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((v[d][i] & 0x7c00u) == 0x7c00u) v[d][i] &= 0xffff0000u;
          if ((v[d][i] & 0x7c000000u) == 0x7c000000u) v[d][i] &= 0xffffu;
        }
    }
    float top[2];
    bool passes = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[j] = fmaxf(fmaxf(fmaxf(s[0][j][0], s[0][j][1]), fmaxf(s[0][j][2], s[0][j][3])),
                     fmaxf(fmaxf(s[1][j][0], s[1][j][1]), fmaxf(s[1][j][2], s[1][j][3]))) * by[j];
      // (a difference: beside a maximum whose neighbours are 16 away a sum could round up to what passes it)
      passes |= top[j] - m[j] + fmaxf(exponent - level[j], 0.f) > kPasses;
    }
    if (__builtin_amdgcn_ballot_w64(passes)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float highest = column_max(top[j]);
        // (a row by its own scores alone, and by scales only in whole powers of two: what others see must not change
        // its roundings)
        const bool moves = highest - m[j] > kPasses;
        const float now = moves ? highest - kWeightLift : m[j];
        const Power down = power_of(moves ? m[j] - now : 0.f);
        const float by_l = __builtin_ldexpf(down.part, down.whole);
        float by_o = by_l, next = exponent;
        if (__builtin_amdgcn_ballot_w64(level[j] != exponent && m[j] != -INFINITY)) {
          const float kept = moves ? ceilf(level[j] + (m[j] - now)) : level[j];
          // (to the nearest: of a row that moves the difference is 0 but for its rounding, and the level the tile's exponent)
          const float wanted = exponent + __builtin_rintf(highest - now - kWeightLift);
          next = moves || highest - now + (exponent - kept) > kPasses ? fmaxf(kept, wanted) : kept;
          by_o = __builtin_ldexpf(down.part, down.whole + (int)fmaxf(level[j] - next, -2000.f));
        }
        m[j] = now;
        level[j] = next;
        l[j] *= by_l;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d][j] *= by_o;
        far[j] |= __builtin_fabsf(now) > 16777216.f && now != -INFINITY;
        if (far[j] && by[j] != 1.f) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][j][i] = product(s[h][j][i], p.scale_log2);
          by[j] = 1.f;
        }
      }
      any_far = __builtin_amdgcn_ballot_w64(far[0] | far[1]) != 0;
    }
    u32x4 w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float from = m[j] == -INFINITY ? 0.f : -m[j];
      float e[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[4 * h + i] = fast_exp2(__builtin_fmaf(s[h][j][i], by[j], from));
      w[j] = u32x4{two_halves(e[0], e[1]), two_halves(e[2], e[3]), two_halves(e[4], e[5]), two_halves(e[6], e[7])};
      float sum;
      if constexpr (BF16) sum = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      else  // the sum of the weights as rounded: where one outweighs the others its rounding cancels
        sum = ((Elem<false>::lo(w[j][0]) + Elem<false>::hi(w[j][0])) + (Elem<false>::lo(w[j][1]) + Elem<false>::hi(w[j][1]))) +
              ((Elem<false>::lo(w[j][2]) + Elem<false>::hi(w[j][2])) + (Elem<false>::lo(w[j][3]) + Elem<false>::hi(w[j][3])));
      l[j] += sum;
      const float scale = m[j] == -INFINITY ? 0.f : exponent - level[j];
      if (__builtin_amdgcn_ballot_w64(scale != 0.f)) {
        // (a scale past 2^100: its weights may be below fp32's least while it is not in them)
        if (__builtin_amdgcn_ballot_w64(scale > 100.f)) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (scale > 100.f) e[4 * h + i] = fast_exp2(__builtin_fmaf(s[h][j][i], by[j], from) + (scale - 100.f));
        }
        const float times = power((int)fminf(fmaxf(scale, -126.f), 100.f));
        w[j] = u32x4{two_halves(e[0] * times, e[1] * times), two_halves(e[2] * times, e[3] * times),
                     two_halves(e[4] * times, e[5] * times), two_halves(e[6] * times, e[7] * times)};
      }
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int j = 0; j < 2; ++j) o[d][j] = mfma32<false>(v[d], w[j], o[d][j]);
    __builtin_amdgcn_s_setprio(0);
  }

  // --- the two halves joined: the later one's state through LDS
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    l[j] += __shfl_xor(l[j], 16);
    l[j] += __shfl_xor(l[j], 32);
  }
  lds_barrier();
  f32x4* hand = reinterpret_cast<f32x4*>(&lds.round[0]);
  static_assert(sizeof(lds.round) >= 4 * 16 * kWave * 16, "four waves' O");
  if (kg == 1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (mq == 0) {
        lds.state[rg][j][0][mt] = m[j];
        lds.state[rg][j][1][mt] = l[j];
        lds.state[rg][j][2][mt] = level[j];
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) hand[((rg * 2 + j) * 8 + d) * kWave + lane] = o[d][j];
    }
  }
  lds_barrier();
  if (kg == 1) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float pm = lds.state[rg][j][0][mt], pl = lds.state[rg][j][1][mt], p_level = lds.state[rg][j][2][mt];
    const float now = fmaxf(m[j], pm);
    const float mine = now == m[j] ? 0.f : m[j] - now, other = now == pm ? 0.f : pm - now;
    const Power by_mine = power_of(mine), by_other = power_of(other);
    const float sum = __builtin_ldexpf(l[j] * by_mine.part, by_mine.whole) + __builtin_ldexpf(pl * by_other.part, by_other.whole);
    const float total = sum == 0.f ? 0.f : 1.f / sum;
    // a half without scores has no level
    const float high = fmaxf(fmaxf(ceilf(level[j] + mine), ceilf(p_level + other)), -200.f);
    const float a = __builtin_ldexpf(by_mine.part, by_mine.whole + (int)fmaxf(level[j] - high, -2000.f));
    const float b = __builtin_ldexpf(by_other.part, by_other.whole + (int)fmaxf(p_level - high, -2000.f));
    const int row = rg * 32 + j * 16 + mt;
    if (row >= n_rows) continue;
    if (p.splits > 1) {  // a part's output and what it weighs, for the merge
      const int64_t at = ((int64_t)blockIdx.x * p.splits + blockIdx.y) * kRows + row;
      if (mq == 0) {
        p.part_ml[at * 2] = now;
        p.part_ml[at * 2 + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const f32x4 x = hand[((rg * 2 + j) * 8 + d) * kWave + lane];
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_ldexpf((o[d][j][i] * a + x[i] * b) * total, (int)high);
        *reinterpret_cast<f32x4*>(p.part_o + at * kValue + d * 16 + 4 * mq) = y;
      }
      continue;
    }
    uint16_t* out = static_cast<uint16_t*>(p.out) + ((int64_t)(first_row + row) * p.heads + real_head) * kValue + 4 * mq;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const f32x4 x = hand[((rg * 2 + j) * 8 + d) * kWave + lane];
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = __builtin_ldexpf((o[d][j][i] * a + x[i] * b) * total, (int)high);
      *reinterpret_cast<u32x2*>(out + d * 16) = u32x2{round_two<BF16>(y[0], y[1]), round_two<BF16>(y[2], y[3])};
    }
  }
}

// Joins the parts of a context: block (tile and head, y) takes 8 rows, a lane 4 elements.
template <bool BF16>
__global__ __launch_bounds__(256) void latent_join_kernel(const LatentChunkParams p) {
  const int head = blockIdx.x % p.group_heads, tile = blockIdx.x / p.group_heads;
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5), e0 = (threadIdx.x & 31) * 4;
  if (row >= p.row_tiles[4 * tile + 1]) return;
  const int64_t first = (int64_t)blockIdx.x * p.splits * kRows + row;
  float top = -INFINITY;
  for (int i = 0; i < p.splits; ++i) top = fmaxf(top, p.part_ml[(first + i * kRows) * 2]);
  float sum = 0.f;
  for (int i = 0; i < p.splits; ++i) {
    const float m = p.part_ml[(first + i * kRows) * 2];
    const Power by = power_of(m == top ? 0.f : m - top);
    sum += __builtin_ldexpf(p.part_ml[(first + i * kRows) * 2 + 1] * by.part, by.whole);
  }
  const float total = sum == 0.f ? 0.f : 1.f / sum;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < p.splits; ++i) {
    const int64_t at = first + i * kRows;
    const float m = p.part_ml[at * 2];
    const Power by = power_of(m == top ? 0.f : m - top);
    const float weight = p.part_ml[at * 2 + 1] * by.part * total;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + at * kValue + e0);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] += __builtin_ldexpf(x[k] * weight, by.whole);
  }
  uint16_t* out = static_cast<uint16_t*>(p.out) + ((int64_t)(p.row_tiles[4 * tile] + row) * p.heads + p.first_head + head) * kValue + e0;
  *reinterpret_cast<u32x2*>(out) = u32x2{round_two<BF16>(o[0], o[1]), round_two<BF16>(o[2], o[3])};
}

template <bool BF16>
hipError_t launch_type(LatentChunkParams p, int32_t latent_dim, hipStream_t stream) {
  const int group = p.group_heads;
  for (p.first_head = 0; p.first_head < p.heads; p.first_head += group) {
    p.group_heads = p.heads - p.first_head < group ? p.heads - p.first_head : group;
    const dim3 expand((unsigned)(p.n_token_tiles * p.group_heads)), attend((unsigned)(p.n_row_tiles * p.group_heads), (unsigned)p.splits);
    if (p.n_token_tiles == 0) {
      // nothing but rows without a context
    } else if (latent_dim == 512) hipLaunchKernelGGL((latent_expand_kernel<512, BF16>), expand, dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((latent_expand_kernel<256, BF16>), expand, dim3(kThreads), 0, stream, p);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL((latent_chunk_kernel<BF16>), attend, dim3(kThreads), 0, stream, p);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (p.splits > 1) {
      hipLaunchKernelGGL((latent_join_kernel<BF16>), dim3(attend.x, kRows / 8), dim3(256), 0, stream, p);
      err = hipGetLastError();
      if (err != hipSuccess) return err;
    }
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_latent_chunks(const LatentChunkParams& p, int32_t latent_dim, bool bf16, hipStream_t stream) {
  if (p.n_row_tiles == 0) return hipSuccess;
  return bf16 ? launch_type<true>(p, latent_dim, stream) : launch_type<false>(p, latent_dim, stream);
}

}  // namespace ayk
