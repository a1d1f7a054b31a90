// Attention over a paged cache of latent vectors, absorbed form (gfx950).
//
// A position's row is [latent (DC) | rotated key part (64)], shared by all heads:
//   score(row, head, t) = scale * q[row, head] . row_t,   out[row, head] = sum_t p_t latent_t,
// softmax over the positions 0 .. position(row), everything past the score in fp32, rounded once.
// A request of length 0 gives zeros.
//
// The rows of a request's queries, [rows x heads, DC + 64], are one contiguous matrix, so any number
// of rows and heads is cut into tiles of NC consecutive (row, head) pairs; every pair of a tile reads
// the same context, which a workgroup streams once for all of them. With NC pairs a position of
// 2 (DC + 64) bytes takes 2 NC (2 DC + 64) operations: at NC 64, DC 512 the matrix cores need a
// quarter of the time that memory does, so what counts is that loads never pause.
//
//  * A workgroup (4 waves, one per compute unit) holds 4 chunks of 32 positions in LDS (147 KB):
//    one being worked on, three on their way, fetched straight into LDS (global_load_lds_dwordx4,
//    no registers). 110 KB in flight per compute unit cover the latency at the full rate.
//  * 16-byte pieces of a row are stored in an order that depends on the position (swizzle), which
//    keeps both the row-wise reads (q.k) and the transposing ones (P.V) spread over the banks.
//  * q.k: S^T = K Q^T, v_mfma_f32_16x16x32, keys from LDS, q in registers for the whole tile: a wave
//    takes 16 of the chunk's positions and half of the pairs.
//  * P.V: O^T += V^T P^T; the values are the latents already in LDS, read transposed
//    (ds_read_b64_tr_b16); each wave takes a quarter of DC for all pairs. P goes through LDS, bf16 in
//    two parts (high and remainder by truncation: one bf16 would lose 2^-9 of each weight, as much as
//    the output's own rounding), fp16 rounded to nearest (2^-12).
//  * The running maximum moves only when a score passes it by kRescaleSlack; until then weights up to
//    2^kRescaleSlack keep their accuracy, and the waves need no word from each other. When one does,
//    a flag read after the barrier sends all of them through the exchange of maxima.
//
// Work is split without the host: positions, cut into chunks, of all tiles form one line, and of G
// workgroups the g-th takes [g T / G, (g + 1) T / G). The lengths are read on the device, so eager
// steps and replays of a captured one run the same code. A workgroup that begins or ends inside a
// tile leaves a partial (m, l, O), at most two of them, and latent_merge_kernel joins each cut tile.
//
// Visible and masked: a masked position's weight is an exact 0, and what it multiplies must be
// finite. Slots behind the context are never read (the last position stands in for them). Rows of one
// request see different ends; if a raw score in their last chunks is not finite, the chunk's
// non-finite elements are taken out of the values before P.V: rows that see that position get NaN
// from its score, the others must not notice.
#include "attention_common.h"

namespace ayk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr int kRope = 64;
constexpr int kChunk = 32;       // positions
constexpr int kStages = 4;       // chunks in LDS
constexpr int kLatentWaves = 4;
constexpr int kTableWindow = 1024;  // block-table entries in LDS
constexpr int kPlaceWords = 8;
// Fewest chunks of one workgroup: a partial's write and merge cost about as much as two chunks.
constexpr int kLeastChunks = 4;

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

// Rounded by itself, never part of an fma: scores are compared and subtracted as rounded values.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// 16 bytes a lane from base + offset to LDS at `to` + 16 * lane (`to` uniform).
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

// Where in a row's 128-byte groups of 8 pieces piece c of position t is: c ^ swizzle(t). Any 8
// consecutive positions differ, and 4 consecutive ones differ in pairs of pieces.
__host__ __device__ constexpr int swizzle(int t) { return ((t & 3) << 1) | ((t >> 2) & 1); }

template <int DC, int NT>
struct __align__(16) LatentShared {
  struct Stage {
    uint16_t latent[kChunk * DC];
    uint16_t rope[kChunk * kRope];
  };
  Stage stage[kStages];
  // weights [pair][position], 8 bytes of padding a row against bank conflicts
  uint16_t weight[2][NT * 16 * (kChunk + 8)];
  int32_t table[kTableWindow];
  float exchange[2][NT * 16];
  int32_t flag[2];
  int32_t sums[kLatentWaves][2];
  int32_t place[kPlaceWords];
};

// A workgroup's place in the line of chunks.
struct Place {
  int request, tile, chunk, first_row, chunks, rows, total, active;
};

// Chunks of the whole step and where workgroup `group` of `groups` begins. Every thread takes a run
// of requests; two sums over the workgroup's threads find the request that holds the beginning.
template <int NC, class Shared>
__device__ __forceinline__ Place find_place(const LatentParams& p, Shared& lds, int group, int groups) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int threads = kLatentWaves * kWave;
  const int each = (p.n_requests + threads - 1) / threads;
  const int from = min(p.n_requests, tid * each), to = min(p.n_requests, from + each);
  auto chunks_of = [&](int b) { return max(1, (max(0, min(p.kv_lengths[b], p.max_len)) + kChunk - 1) / kChunk); };
  auto items_of = [&](int b, int rows) { return (rows * p.heads + NC - 1) / NC * chunks_of(b); };
  int items = 0, rows = 0;
  for (int b = from; b < to; ++b) {
    const int r = max(0, p.rows[b]);
    rows += r;
    items += items_of(b, r);
  }
  int items_upto = items, rows_upto = rows;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(items_upto, d), c = __shfl_up(rows_upto, d);
    if (lane >= d) items_upto += a, rows_upto += c;
  }
  if (lane == 63) lds.sums[wave][0] = items_upto, lds.sums[wave][1] = rows_upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kLatentWaves; ++w) {
    if (w < wave) items_upto += lds.sums[w][0], rows_upto += lds.sums[w][1];
    total += lds.sums[w][0];
  }
  const int active = max(1, min(groups, total / kLeastChunks));
  const int begin = (int)((int64_t)min(group, active) * total / active);
  int before = items_upto - items;
  if (begin >= before && begin < items_upto) {
    int row = rows_upto - rows;
    for (int b = from; b < to; ++b) {
      const int r = max(0, p.rows[b]), n = items_of(b, r);
      if (begin < before + n) {
        const int c = chunks_of(b);
        lds.place[0] = b;
        lds.place[1] = (begin - before) / c;
        lds.place[2] = (begin - before) % c;
        lds.place[3] = row;
        lds.place[4] = c;
        lds.place[5] = r;
        break;
      }
      before += n;
      row += r;
    }
  }
  __syncthreads();
  auto uniform = [&](int i) { return __builtin_amdgcn_readfirstlane(lds.place[i]); };
  return Place{uniform(0), uniform(1), uniform(2), uniform(3), uniform(4), uniform(5), total, active};
}

template <int DC, bool BF16, int NT>
__global__ __launch_bounds__(kLatentWaves* kWave, 1) void latent_attention_kernel(const LatentParams p) {
  constexpr int NC = NT * 16;
  constexpr int ROW = DC + kRope;
  constexpr int KS = DC / 32;          // steps of q.k over the latent; two more over the rotary part
  constexpr int NQ = NT == 4 ? 2 : 1;  // 16-pair tiles of a wave's q.k
  constexpr int DT = DC / kLatentWaves / 16;  // 16-element slices of a wave's P.V
  constexpr int ROWS_PER_LOAD = 1024 / (DC * 2);
  constexpr int LOADS = 8 / ROWS_PER_LOAD + 1;  // a wave's per chunk
  typedef LatentShared<DC, NT> Shared;
  __shared__ Shared lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mt = lane & 15, mq = lane >> 4;
  const int kg = wave & 1, half = wave >> 1;  // q.k: positions 16 kg .., tiles NQ half ..
  const bool scores = NT > 1 || half == 0;
  const int groups = gridDim.x, group = blockIdx.x;

  Place at = find_place<NC>(p, lds, group, groups);
  if (group < at.active && tid < kPlaceWords) {
    const int words[kPlaceWords] = {at.request, at.tile, at.chunk, at.first_row, at.chunks, at.rows, at.total, at.active};
    int w = words[0];
#pragma unroll
    for (int i = 1; i < kPlaceWords; ++i) w = tid == i ? words[i] : w;
    p.places[group * kPlaceWords + tid] = w;
  }
  if (group >= at.active || at.total == 0) return;
  const int begin = (int)((int64_t)group * at.total / at.active);
  int left = (int)((int64_t)(group + 1) * at.total / at.active) - begin;

  const uint32_t lds_base = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) Shared*)&lds);
  // a lane's offsets into a stage (bytes)
  const int key = kg * 16 + mt;
  int k_at[2], v_at[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) k_at[i] = ((4 * i + mq) ^ swizzle(key)) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * mq + (mt >> 2);
    v_at[i] = t * DC * 2 + wave * (DC / kLatentWaves) * 2 + ((2 * i + ((mt & 3) >> 1)) ^ swizzle(t)) * 16 + (mt & 1) * 8;
  }
  // what this wave fetches: positions 8 wave .. 8 wave + 7 of each chunk
  const uint32_t rope_from = DC * 2 + ((lane & 7) ^ swizzle(lane >> 3)) * 16;

  while (left > 0) {
    // --- one tile, chunks [at.chunk, end) of it
    const int end = min(at.chunks, at.chunk + left);
    const bool whole = at.chunk == 0 && end == at.chunks;
    const int pairs = min(at.rows * p.heads - at.tile * NC, NC);
    const int length = max(0, min(p.kv_lengths[at.request], p.max_len));
    const int first_pos = length - at.rows;
    // the last row of the tile sees the most
    const int context = length == 0 ? 0 : max(0, min(length, first_pos + (at.tile * NC + pairs - 1) / p.heads + 1));
    const int from = at.chunk, to = min(end, (context + kChunk - 1) / kChunk);
    // rows from here on are not seen by every pair
    const int least_pos = first_pos + at.tile * NC / p.heads;
    const int64_t pair0 = (int64_t)at.first_row * p.heads + at.tile * NC;
    const int64_t pairs_left = (int64_t)p.n_rows * p.heads - pair0;  // (row counts that disagree stay in bounds)

    int my_pos[NQ];
    u32x4 q[NQ][KS + 2];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int c = (half * NQ + j) * 16 + mt;
      const bool real = scores && c < pairs && c < pairs_left;
      my_pos[j] = real ? first_pos + (at.tile * NC + c) / p.heads : -1;
      const u32x4* from_q = reinterpret_cast<const u32x4*>(p.q + (pair0 + (real ? c : 0)) * ROW) + mq;
#pragma unroll
      for (int s = 0; s < KS + 2; ++s) q[j][s] = real ? from_q[4 * s] : u32x4{0, 0, 0, 0};
    }
    f32x4 o[DT][NT];
    float m[NT], l[NQ];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      m[c] = -INFINITY;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) l[j] = 0.f;

    const int32_t* table = p.block_table + at.request * p.table_stride;
    for (int w0 = from; w0 < to;) {
      // --- a window of the block table
      const int b0 = (int)quotient((uint32_t)(w0 * kChunk), p.by_block);
      const int last_block = (int)quotient((uint32_t)(min(to * kChunk, context) - 1), p.by_block);
      const int blocks = min(kTableWindow, last_block - b0 + 1);
      // whole chunks that its blocks cover
      const int w1 = b0 + blocks > last_block ? to : (b0 + blocks) * p.block_size / kChunk;
      __syncthreads();
      for (int i = tid; i < blocks; i += kLatentWaves * kWave) {
        const uint32_t id = (uint32_t)table[b0 + i];
        lds.table[i] = id < (uint32_t)p.num_blocks ? (int)id : 0;
      }
      if (tid < 2) lds.flag[tid] = 0;
      __syncthreads();

      auto fetch = [&](int chunk) {
        const int pos = min(chunk * kChunk + wave * 8 + (lane & 7), context - 1);
        const uint32_t block = quotient((uint32_t)pos, p.by_block);
        const uint32_t slot = (uint32_t)lds.table[block - b0] * (uint32_t)p.block_size + ((uint32_t)pos - block * (uint32_t)p.block_size);
        const uint32_t stage = lds_base + (uint32_t)((chunk & (kStages - 1)) * sizeof(typename Shared::Stage));
        const uint8_t* cache = reinterpret_cast<const uint8_t*>(p.cache);
#pragma unroll
        for (int j = 0; j < 8 / ROWS_PER_LOAD; ++j) {
          const uint32_t lds_to = stage + (uint32_t)((wave * 8 + j * ROWS_PER_LOAD) * DC * 2);
          if constexpr (ROWS_PER_LOAD == 1) {
            const uint32_t s = __builtin_amdgcn_readlane(slot, j);
            load_to_lds(lds_to, cache + (uint64_t)s * (ROW * 2), (uint32_t)((lane ^ swizzle(j)) * 16));
          } else {
            const uint32_t s0 = __builtin_amdgcn_readlane(slot, 2 * j), s1 = __builtin_amdgcn_readlane(slot, 2 * j + 1);
            const uint32_t s = lane < 32 ? s0 : s1;
            const int piece = (lane & 31) ^ (lane < 32 ? swizzle(2 * j) : swizzle(2 * j + 1));
            load_to_lds(lds_to, cache + (uint64_t)s * (ROW * 2) + piece * 16);
          }
        }
        const uint32_t s = (uint32_t)__shfl((int)slot, lane >> 3);
        load_to_lds(stage + (uint32_t)(kChunk * DC * 2 + wave * 8 * kRope * 2), cache + (uint64_t)s * (ROW * 2) + rope_from);
      };

#pragma unroll
      for (int i = 0; i < kStages - 1; ++i)
        if (w0 + i < w1) fetch(w0 + i);

      for (int chunk = w0; chunk < w1; ++chunk) {
        const uint8_t* stage = reinterpret_cast<const uint8_t*>(&lds.stage[chunk & (kStages - 1)]);
        if (chunk + 2 < w1) wait_loads<2 * LOADS>();
        else if (chunk + 1 < w1) wait_loads<LOADS>();
        else wait_loads<0>();
        lds_barrier();  // the chunk is here, and nobody works on the one before it
        if (chunk + kStages - 1 < w1) fetch(chunk + kStages - 1);
        if (tid == 0) lds.flag[(chunk + 1) & 1] = 0;

        const int t0 = chunk * kChunk;
        const bool masked = t0 + kChunk > context || t0 + kChunk - 1 > least_pos;
        f32x4 s[NQ];
        float before[NQ];  // the sums without this chunk
        // weights of this wave's scores under the maximum m
        auto put_weights = [&] {
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            const float mj = NT == 4 ? (half ? m[(NT == 4 ? 2 : 0) + j] : m[j]) : NT == 2 ? (half ? m[NT - 1] : m[0]) : m[0];
            const float base = mj == -INFINITY ? 0.f : mj;
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = fast_exp2(s[j][i] - base);
            l[j] = before[j] + ((w[0] + w[1]) + (w[2] + w[3]));
            u32x2 hi, lo;
            split_weights4<BF16>(w, hi, lo);
            const int row = ((half * NQ + j) * 16 + mt) * (kChunk + 8) + 8 * mq + 4 * kg;
            *reinterpret_cast<u32x2*>(&lds.weight[0][row]) = hi;
            if constexpr (split_p(BF16)) *reinterpret_cast<u32x2*>(&lds.weight[1][row]) = lo;
          }
        };
        if (scores) {
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            before[j] = l[j];
          }
          const uint8_t* row = stage + key * DC * 2;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(row + (k >> 1) * 128 + k_at[k & 1]);
#pragma unroll
            for (int j = 0; j < NQ; ++j) s[j] = mfma32<BF16>(a, q[j][k], s[j]);
          }
          const uint8_t* tail = stage + kChunk * DC * 2 + key * kRope * 2;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(tail + k_at[k]);
#pragma unroll
            for (int j = 0; j < NQ; ++j) s[j] = mfma32<BF16>(a, q[j][KS + k], s[j]);
          }
          bool passes = false, odd = false;
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            const float mj = NT == 4 ? (half ? m[(NT == 4 ? 2 : 0) + j] : m[j]) : NT == 2 ? (half ? m[NT - 1] : m[0]) : m[0];
            const int seen = min(my_pos[j], context - 1) - t0 - kg * 16 - 4 * mq;  // position i of the lane's 4: i <= seen
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (masked) odd |= !(__builtin_fabsf(s[j][i]) < INFINITY);
              const float t = product(s[j][i], p.scale_log2);
              s[j][i] = !masked || i <= seen ? t : -INFINITY;
              passes |= s[j][i] > mj + kRescaleSlack;
            }
          }
          const int word = (__builtin_amdgcn_ballot_w64(passes) ? 1 : 0) | (__builtin_amdgcn_ballot_w64(odd) ? 2 : 0);
          if (word && lane == 0) atomicOr(&lds.flag[chunk & 1], word);
          put_weights();
        }
        lds_barrier();
        const int word = __builtin_amdgcn_readfirstlane(lds.flag[chunk & 1]);
        if (word) {
          if (word & 2) {
            // this wave's slice of the values: 32 positions x DC / 4 elements, in 16-byte pieces
            uint8_t* mine = const_cast<uint8_t*>(stage) + wave * (DC / kLatentWaves) * 2;
            constexpr int PIECES = DC / kLatentWaves / 8;
            for (int i = lane; i < kChunk * PIECES; i += kWave) {
              uint32_t* x = reinterpret_cast<uint32_t*>(mine + (i / PIECES) * DC * 2 + (i % PIECES) * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                constexpr uint32_t EXP = BF16 ? 0x7f80u : 0x7c00u;
                uint32_t w = x[e];
                if ((w & EXP) == EXP) w &= 0xffff0000u;
                if (((w >> 16) & EXP) == EXP) w &= 0xffffu;
                x[e] = w;
              }
            }
          }
          // every pair's maximum over the chunk, then the state and the weights under the new one
          if (scores) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              const float top = column_max(fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])));
              if (mq == 0) lds.exchange[kg][(half * NQ + j) * 16 + mt] = top;
            }
          }
          lds_barrier();
          float by[NT];
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            const float top = fmaxf(m[c], fmaxf(lds.exchange[0][c * 16 + mt], lds.exchange[1][c * 16 + mt]));
            by[c] = top == m[c] ? 1.f : fast_exp2(m[c] - top);
            m[c] = top;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][c] *= by[c];
          }
          if (scores) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              const float b = NT == 4 ? (half ? by[(NT == 4 ? 2 : 0) + j] : by[j]) : NT == 2 ? (half ? by[NT - 1] : by[0]) : by[0];
              before[j] *= b;
            }
            put_weights();
          }
          lds_barrier();
        }
        // O^T += V^T P^T
        u32x4 w[2][NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const int row = (c * 16 + mt) * (kChunk + 8) + 8 * mq;
          w[0][c] = *reinterpret_cast<const u32x4*>(&lds.weight[0][row]);
          if constexpr (split_p(BF16)) w[1][c] = *reinterpret_cast<const u32x4*>(&lds.weight[1][row]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint16_t* v = reinterpret_cast<const uint16_t*>(stage + v_at[d & 3] + (d >> 2) * 128);
          const u32x2 a = lds_read_transposed(v), b = lds_read_transposed(v + 16 * DC);
          const u32x4 va = u32x4{a.x, a.y, b.x, b.y};
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            o[d][c] = mfma32<BF16>(va, w[0][c], o[d][c]);
            if constexpr (split_p(BF16)) o[d][c] = mfma32<BF16>(va, w[1][c], o[d][c]);
          }
        }
      }
      w0 = w1;
    }

    // --- the tile's sums, and its output or this workgroup's part of it
    if (scores) {
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float sum = l[j];
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        l[j] = sum;
      }
    }
    lds_barrier();  // the exchange may still be read
    if (scores && mq == 0) {
#pragma unroll
      for (int j = 0; j < NQ; ++j) lds.exchange[kg][(half * NQ + j) * 16 + mt] = l[j];
    }
    lds_barrier();
    const int slot = 2 * group + (at.chunk == 0 ? 1 : 0);
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const int pair = c * 16 + mt;
      const float sum = lds.exchange[0][pair] + lds.exchange[1][pair];
      if (pair < pairs && pair < pairs_left) {
        const int e0 = wave * (DC / kLatentWaves) + 4 * mq;
        if (whole) {
          const float by = sum == 0.f ? 0.f : 1.f / sum;
          uint16_t* out = static_cast<uint16_t*>(p.out) + (pair0 + pair) * DC + e0;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            u32x2 two;
            two.x = Elem<BF16>::round(o[d][c][0] * by) | Elem<BF16>::round(o[d][c][1] * by) << 16;
            two.y = Elem<BF16>::round(o[d][c][2] * by) | Elem<BF16>::round(o[d][c][3] * by) << 16;
            *reinterpret_cast<u32x2*>(out + d * 16) = two;
          }
        } else {
          if (wave == 0 && mq == 0) {
            p.part_ml[(slot * NC + pair) * 2] = m[c];
            p.part_ml[(slot * NC + pair) * 2 + 1] = sum;
          }
          float* out = p.part_o + ((int64_t)slot * NC + pair) * DC + e0;
#pragma unroll
          for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(out + d * 16) = o[d][c];
        }
      }
    }

    // --- on to the next tile
    left -= end - at.chunk;
    at.chunk = 0;
    if (left > 0 && (at.tile + 1) * NC >= at.rows * p.heads) {
      at.tile = -1;
      do {
        at.first_row += at.rows;
        if (++at.request >= p.n_requests) return;  // (lengths changed under the launch)
        at.rows = max(0, p.rows[at.request]);
      } while (at.rows == 0);
      at.chunks = max(1, (max(0, min(p.kv_lengths[at.request], p.max_len)) + kChunk - 1) / kChunk);
    }
    ++at.tile;
  }
}

// Joins the parts of a tile that workgroups share. Block (g, y): the tile that workgroup g begins
// inside, unless an earlier one does too; a wave takes a pair, lanes DC / 64 elements each.
template <int DC, bool BF16, int NC>
__global__ __launch_bounds__(256) void latent_merge_kernel(const LatentParams p, int groups) {
  constexpr int EPL = DC / 64;
  const int g = blockIdx.x + 1, lane = threadIdx.x & 63;
  const int32_t* place = p.places + g * kPlaceWords;
  const int total = p.places[6], active = p.places[7];
  if (g >= active) return;
  const int chunk = place[2], chunks = place[4];
  if (chunk == 0) return;
  auto begin_of = [&](int i) { return (int)((int64_t)i * total / active); };
  const int start = begin_of(g) - chunk;  // of the tile
  if (begin_of(g - 1) > start) return;
  int last = g;  // the last workgroup with chunks of this tile
  while (last + 1 < active && begin_of(last + 1) < start + chunks) ++last;
  const int pair = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int tile = place[1], rows = place[5];
  const int64_t at = (int64_t)place[3] * p.heads + tile * NC + pair;
  if (tile * NC + pair >= rows * p.heads || at >= (int64_t)p.n_rows * p.heads) return;
  // part i of the tile: workgroup g - 1's began the tile, the others' continued it
  auto slot_of = [&](int i) { return (int64_t)(2 * i + (i == g - 1 ? 1 : 0)) * NC + pair; };
  float top = -INFINITY;
  for (int i = g - 1 + lane; i <= last; i += 64) top = fmaxf(top, p.part_ml[slot_of(i) * 2]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  float sum = 0.f;
  float o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = g - 1; i <= last; ++i) {
    const int64_t slot = slot_of(i);
    const float m = p.part_ml[slot * 2], l = p.part_ml[slot * 2 + 1];
    // (a part without visible positions has l 0; one whose scores were NaN has a NaN l)
    const float by = m == top ? 1.f : fast_exp2(m - top);
    sum += l * by;
    const float* from = p.part_o + slot * DC + lane * 4;
#pragma unroll
    for (int e = 0; e < EPL; e += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(from + e * 64);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[e + k] += x[k] * by;
    }
  }
  const float by = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* out = static_cast<uint16_t*>(p.out) + at * DC + lane * 4;
#pragma unroll
  for (int e = 0; e < EPL; e += 4) {
    u32x2 two;
    two.x = Elem<BF16>::round(o[e] * by) | Elem<BF16>::round(o[e + 1] * by) << 16;
    two.y = Elem<BF16>::round(o[e + 2] * by) | Elem<BF16>::round(o[e + 3] * by) << 16;
    *reinterpret_cast<u32x2*>(out + e * 64) = two;
  }
}

template <int DC, bool BF16, int NT>
hipError_t launch_pairs(const LatentParams& p, int compute_units, hipStream_t stream) {
  hipLaunchKernelGGL((latent_attention_kernel<DC, BF16, NT>), dim3(compute_units), dim3(kLatentWaves * kWave), 0, stream, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || compute_units < 2) return err;
  hipLaunchKernelGGL((latent_merge_kernel<DC, BF16, NT * 16>), dim3(compute_units - 1, NT * 4), dim3(256), 0, stream, p,
                     compute_units);
  return hipGetLastError();
}

template <int DC, bool BF16>
hipError_t launch_type(const LatentParams& p, int pairs, int compute_units, hipStream_t stream) {
  if (pairs == 16) return launch_pairs<DC, BF16, 1>(p, compute_units, stream);
  if (pairs == 32) return launch_pairs<DC, BF16, 2>(p, compute_units, stream);
  return launch_pairs<DC, BF16, 4>(p, compute_units, stream);
}

}  // namespace

int latent_tile_pairs(int64_t n_rows, int32_t n_requests, int32_t heads) {
  const int64_t each = n_requests > 0 ? n_rows * heads / n_requests : 0;
  return each <= 16 ? 16 : each <= 32 ? 32 : 64;
}

size_t latent_workspace_bytes(int32_t latent_dim, int pairs, int compute_units) {
  return (size_t)compute_units * (kPlaceWords * 4 + 2 * (size_t)pairs * (2 + latent_dim) * 4);
}

hipError_t launch_latent_attention(const LatentParams& p, int32_t latent_dim, bool bf16, int pairs, int compute_units,
                                   hipStream_t stream) {
  if (latent_dim == 512)
    return bf16 ? launch_type<512, true>(p, pairs, compute_units, stream)
                : launch_type<512, false>(p, pairs, compute_units, stream);
  return bf16 ? launch_type<256, true>(p, pairs, compute_units, stream)
              : launch_type<256, false>(p, pairs, compute_units, stream);
}

}  // namespace ayk
