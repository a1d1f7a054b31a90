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
// 2 (DC + 64) bytes takes 2 NC (2 DC + 64) operations: at DC 512 memory and matrix cores take the
// same time at about 140 pairs, at the rates that a copy and a library product reach (5.0 TB/s and 1.25
// PFLOP/s); a bf16 P doubles the operations of its product.
//
//  * A workgroup (8 waves, one workgroup per compute unit) holds 4 chunks of 32 positions in LDS
//    (147 KB), fetched straight into it (global_load_lds_dwordx4, no registers), up to three on their
//    way while one is worked on: 110 KB in flight per compute unit cover the latency at the full rate.
//  * 16-byte pieces of a row are stored in an order that depends on the position (swizzle), which
//    keeps both the row-wise reads (q.k) and the transposing ones (P.V) spread over the banks.
//  * S^T = K Q^T: two waves for each 16 pairs, 16 positions each, q in registers. The weights go through
//    LDS, and O^T += V^T P^T by all 8 waves, an eighth of DC each for all pairs (so a wave's q and O fit
//    its 256 registers); the values are the latents already in LDS, read transposed
//    (ds_read_b64_tr_b16). v_mfma_f32_16x16x32. A bf16 P is taken in two parts (high and remainder by
//    truncation: one bf16 would lose 2^-9 of each weight, as much as the output's own rounding), an fp16
//    P rounded to nearest (2^-11, from 2^-21 of the maximum on 2^-32 of it: kWeightLift).
//  * The running maximum moves only when a score passes it by kRescaleSlack; until then weights up to
//    2^kRescaleSlack times what they were keep their accuracy and nothing is rescaled.
//  * Up to 32 pairs memory is the bound: two barriers a chunk, and the four waves without scores fetch.
//    With 64 pairs the products are, so a chunk is scored while the last one is weighed, one barrier a
//    chunk: of the two waves of a SIMD one weighs first and one scores first.
//
// Work is split without the host: the chunks of all tiles, and tile_cost(NC) for each tile's own start and
// end, form one line, and of G workgroups the g-th takes [g T / G, (g + 1) T / G). The lengths are read
// on the device, so eager steps and replays of a captured one run the same code. A workgroup that
// begins or ends inside a tile leaves a partial (m, l, O), at most two of them, and
// latent_merge_kernel joins each cut tile.
//
// Measured at DC 512 (this kernel + the merge): 64 requests of 4096 positions, 16 heads, bf16: 54 + 5 us,
// 302 MB at 5.6 TB/s in the first; 61 requests of 16 to 16384 positions, 128 heads, bf16: 79 + 10 us; 32
// requests of 4096 with 4 rows each, 32 heads, fp16: 72 + 9 us, 510 TFLOP/s in the first, where 3000 cycles a
// chunk of 64 pairs go to 1150 of matrix instructions (1600 for bf16) and the reads of LDS and exponentials
// that they do not cover; 4 requests of 128 to 1000, 16 heads: 15 + 4 us, which is the chain of
// lengths, table, first rows (8 us) and a few chunks.
//
// Visible and masked: a masked position's weight is an exact 0, and what it multiplies must be
// finite. Slots behind the context are never read (the last position stands in for them). Rows of one
// request see different ends; if a raw score in their last chunks is not finite, the non-finite
// elements are taken out of the values there, and rows that see them get NaN in their place: the
// others must not notice.
#include <type_traits>

#include "attention_common.h"

namespace ayk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr int kRope = 64;
constexpr int kChunk = 32;   // positions
constexpr int kStages = 4;   // chunks in LDS
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kTableWindow = 768;       // block-table entries in LDS
constexpr int kPlaceWords = 8;
// What a tile of NC pairs costs beside its chunks (queries, first loads, output), in chunks. Measured with
// 3, 5, 8 and 12: 64 pairs of the uneven requests above 102, 85, 80, 80 us, of the rows of four 68, 70, 69, 72;
// 16 pairs of the 4 short requests 14, 15, 18, 21, of the 64 long ones 53, 55, 55, 55.
constexpr int tile_cost(int nc) { return nc == 64 ? 8 : 5; }
// Fewest chunks, beside a tile's cost, for one workgroup: as many as a partial's write and merge are worth
// (the 4 short requests: 15 us with 2, 20 with 6; the others do not care).
constexpr int kLeastChunks = 2;

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

// 16 bytes a lane from base + offset (or from `at`) to LDS at `to` + 16 * lane (`to` uniform).
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

// Where 16-byte pieces stand in LDS. Its 64 banks serve 16 pieces a cycle, in a 16-byte read those of
// lanes 0-3, 12-15 and 20-27, and so on (measured: 4.0 cycles a read where these 16 differ
// modulo 256 bytes, 8.0 where two meet). Piece c of a latent of position t is at c ^ (t % 16) of its
// row, piece c of a rotary part (rows of 128 bytes) at c ^ (t / 2 % 8), piece c of a pair's weights
// (rows of 64 bytes) at c ^ (pair / 4 % 4): there two meet in a read, and yet the fp16 verify windows above take
// 71 us so and 73 with c ^ (pair / 2 % 4), where none do; steps of 128 bf16 heads 78 either way, and calls on inputs
// that change the same within half a percent.
__host__ __device__ constexpr int latent_swizzle(int t) { return t & 15; }
__host__ __device__ constexpr int rope_swizzle(int t) { return (t >> 1) & 7; }
__host__ __device__ constexpr int weight_swizzle(int pair) { return (pair >> 2) & 3; }

// How far a pair's reference lies under the maximum that set it, and from there to where a score moves it. (A bf16 P
// has fp32's range.)
constexpr float lift(bool bf16) { return bf16 ? 0.f : kWeightLift; }
constexpr float reach(bool bf16) { return lift(bf16) + kRescaleSlack; }
// The largest score that does not move a reference m. Where m's neighbours are far apart (`far`: at least 2 at 2^24) the
// sum may round up to a score whose weight an fp16 P cannot hold: past half a unit over (2^15.5 of 65504) it is m itself.
template <bool BF16>
__device__ __forceinline__ float limit_of(float m, bool far) {
  const float limit = m + reach(BF16);
  return !BF16 && far && limit - m > reach(BF16) + 0.5f ? m : limit;
}

// Tiles of 64 pairs score a chunk while they weigh the one before it.
constexpr bool ahead(int nt) { return nt == 4; }

template <int DC, int NT>
struct __align__(16) LatentShared {
  uint16_t latent[kStages][kChunk * DC];
  uint16_t rope[ahead(NT) ? 3 : kStages][kChunk * kRope];
  uint16_t weight[ahead(NT) ? 2 : 1][2][NT * 16 * kChunk];  // [chunk][high, low][pair][position]
  int32_t table[kTableWindow];
  float exchange[2][NT * 16];
  int32_t flag[3];
  int32_t sums[kWaves][2];
  int32_t place[8];
};

__device__ __forceinline__ int length_of(const LatentParams& p, int request) {
  return max(0, min(p.kv_lengths[request], p.max_len));
}
__device__ __forceinline__ int chunks_of(int length) { return max(1, (length + kChunk - 1) / kChunk); }

// Chunks [from, to) of a tile, to be worked on by one workgroup.
struct Piece {
  int request, tile, first_row, rows, length;
  int from, to;
  bool whole;
};

// A workgroup's walk along the line of tiles.
template <int NC>
struct Walk {
  int request, tile, unit, first_row, chunks, rows, length;  // the next tile, from its `unit` on
  int left;                                                   // units

  __device__ __forceinline__ bool next(const LatentParams& p, Piece& piece) {
    while (left > 0) {
      const int take = min(chunks + tile_cost(NC) - unit, left);
      piece.request = request;
      piece.tile = tile;
      piece.first_row = first_row;
      piece.rows = rows;
      piece.length = length;
      piece.from = max(0, unit - tile_cost(NC));
      piece.to = unit + take - tile_cost(NC);
      piece.whole = piece.from == 0 && piece.to == chunks;
      left -= take;
      unit = 0;
      ++tile;
      if (left > 0 && tile * NC >= rows * p.heads) {
        tile = 0;
        do {
          first_row += rows;
          if (++request >= p.n_requests) {  // (the step's numbers changed under the launch)
            left = 0;
            break;
          }
          rows = max(0, p.rows[request]);
        } while (rows == 0);
        if (left > 0) {
          length = length_of(p, request);
          chunks = chunks_of(length);
        }
      }
      if (piece.to > piece.from) return true;
    }
    return false;
  }
};

// Where workgroup `group` of `groups` begins. Every thread takes a run of requests; two sums over the
// workgroup's threads find the request that holds the beginning. False: no work.
template <int NC, class Shared>
__device__ __forceinline__ bool find_place(const LatentParams& p, Shared& lds, int group, int groups, Walk<NC>& walk) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (p.n_requests + kThreads - 1) / kThreads;
  const int from = min(p.n_requests, tid * each), to = min(p.n_requests, from + each);
  auto units_of = [&](int length, int rows) { return (rows * p.heads + NC - 1) / NC * (chunks_of(length) + tile_cost(NC)); };
  int units = 0, rows = 0, first_rows = 0, first_length = 0;
  for (int b = from; b < to; ++b) {
    const int r = max(0, p.rows[b]), length = length_of(p, b);
    if (b == from) first_rows = r, first_length = length;
    rows += r;
    units += units_of(length, r);
  }
  int units_upto = units, rows_upto = rows;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(units_upto, d), c = __shfl_up(rows_upto, d);
    if (lane >= d) units_upto += a, rows_upto += c;
  }
  if (lane == 63) lds.sums[wave][0] = units_upto, lds.sums[wave][1] = rows_upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) units_upto += lds.sums[w][0], rows_upto += lds.sums[w][1];
    total += lds.sums[w][0];
  }
  const int active = max(1, min(groups, total / (tile_cost(NC) + kLeastChunks)));
  auto begin_of = [&](int i) { return (int)((int64_t)i * total / active); };
  const int begin = begin_of(min(group, active));
  int before = units_upto - units;
  if (begin >= before && begin < units_upto) {
    int row = rows_upto - rows;
    for (int b = from; b < to; ++b) {
      const int r = b == from ? first_rows : max(0, p.rows[b]);
      const int length = b == from ? first_length : length_of(p, b);
      const int n = units_of(length, r), tile = chunks_of(length) + tile_cost(NC);
      if (begin < before + n) {
        lds.place[0] = b;
        lds.place[1] = (begin - before) / tile;
        lds.place[2] = (begin - before) % tile;
        lds.place[3] = row;
        lds.place[4] = chunks_of(length);
        lds.place[5] = r;
        lds.place[6] = length;
        break;
      }
      before += n;
      row += r;
    }
  }
  __syncthreads();
  auto uniform = [&](int i) { return __builtin_amdgcn_readfirstlane(lds.place[i]); };
  walk.request = uniform(0);
  walk.tile = uniform(1);
  walk.unit = uniform(2);
  walk.first_row = uniform(3);
  walk.chunks = uniform(4);
  walk.rows = uniform(5);
  walk.length = uniform(6);
  walk.left = begin_of(group + 1) - begin;
  const bool some = group < active && total > 0;
  if (group < active && tid == 0) {  // for the merge
    int32_t* place = p.places + group * kPlaceWords;
    place[0] = walk.tile;
    place[1] = max(0, walk.unit - tile_cost(NC));
    place[2] = walk.first_row;
    place[3] = walk.chunks;
    place[4] = walk.rows;
    place[5] = total;
    place[6] = active;
  }
  return some;
}

// A piece's geometry.
struct Tile {
  int first_pos;   // of the request's first row
  int context;     // positions that some pair sees
  int least_pos;   // what every pair sees: up to and with this position
  int to;          // chunks from piece.from to here hold any of them
  int pairs;       // of this tile, as far as there are rows
  int64_t pair0;
};

template <int NC>
__device__ __forceinline__ Tile tile_of(const LatentParams& p, const Piece& piece) {
  Tile t;
  const int pair = piece.tile * NC;
  t.first_pos = piece.length - piece.rows;
  t.pair0 = (int64_t)piece.first_row * p.heads + pair;
  const int pairs = min(piece.rows * p.heads - pair, NC);
  t.pairs = (int)max((int64_t)0, min((int64_t)pairs, (int64_t)p.n_rows * p.heads - t.pair0));
  t.context = piece.length == 0 ? 0 : max(0, min(piece.length, t.first_pos + (pair + pairs - 1) / p.heads + 1));
  t.least_pos = t.first_pos + pair / p.heads;
  t.to = min(piece.to, (t.context + kChunk - 1) / kChunk);
  return t;
}

// The chunks [w0, w1) whose blocks fit the table window, and the first of those blocks.
struct Window {
  int b0, blocks, w1;
};
__device__ __forceinline__ Window window_of(const LatentParams& p, const Tile& t, int w0) {
  Window w;
  w.b0 = (int)quotient((uint32_t)(w0 * kChunk), p.by_block);
  const int last = (int)quotient((uint32_t)(min(t.to * kChunk, t.context) - 1), p.by_block);
  w.blocks = min(kTableWindow, last - w.b0 + 1);
  w.w1 = w.b0 + w.blocks > last ? t.to : (w.b0 + w.blocks) * p.block_size / kChunk;
  return w;
}

__device__ __forceinline__ void stage_table(const LatentParams& p, int request, const Window& w, int32_t* s_table) {
  const int32_t* table = p.block_table + request * p.table_stride + w.b0;
  for (int i = threadIdx.x; i < w.blocks; i += kThreads) {
    const uint32_t id = (uint32_t)table[i];
    s_table[i] = id < (uint32_t)p.num_blocks ? (int)id : 0;
  }
}

// The slot of position first + lane % MINE; positions past `last` are replaced by it.
template <int MINE>
__device__ __forceinline__ uint32_t slot_of(const LatentParams& p, const int32_t* s_table, int b0, int first, int last) {
  const int pos = min(first + (int)(threadIdx.x & (MINE - 1)), last);
  const uint32_t block = quotient((uint32_t)pos, p.by_block);
  return (uint32_t)s_table[block - b0] * (uint32_t)p.block_size + ((uint32_t)pos - block * (uint32_t)p.block_size);
}

// Ask for a share of a chunk (of several waves `wave`): MINE rows of latents, 1024 bytes a load, and one load of their
// rotary parts, 8 lanes a position.
template <int DC, int MINE>
__device__ __forceinline__ void fetch(const LatentParams& p, uint32_t slot, int wave, uint32_t latent, uint32_t rope) {
  static_assert(MINE <= 8, "a load of rotary parts covers 8 positions");
  constexpr int ROW = (DC + kRope) * 2;
  constexpr int PER_LOAD = 1024 / (DC * 2);
  const int lane = threadIdx.x & 63, first = wave * MINE;
  const uint8_t* cache = reinterpret_cast<const uint8_t*>(p.cache);
#pragma unroll
  for (int j = 0; j < MINE / PER_LOAD; ++j) {
    const uint32_t to = latent + (uint32_t)((first + j * PER_LOAD) * DC * 2);
    if constexpr (PER_LOAD == 1) {
      const uint32_t s = __builtin_amdgcn_readlane(slot, j);
      load_to_lds(to, cache + (uint64_t)s * ROW, (uint32_t)((lane ^ latent_swizzle(first + j)) * 16));
    } else {
      const uint32_t s0 = __builtin_amdgcn_readlane(slot, 2 * j), s1 = __builtin_amdgcn_readlane(slot, 2 * j + 1);
      const int piece = (lane & 31) ^ latent_swizzle(first + 2 * j + (lane >> 5));
      load_to_lds(to, cache + (uint64_t)(lane < 32 ? s0 : s1) * ROW + piece * 16);
    }
  }
  const uint32_t s = (uint32_t)__shfl((int)slot, lane >> 3);
  if (MINE == 8 || lane < MINE * 8)
    load_to_lds(rope + (uint32_t)(first * kRope * 2),
                cache + (uint64_t)s * ROW + (DC * 2 + ((lane & 7) ^ rope_swizzle(first + (lane >> 3))) * 16));
}

// The queries of pair `pair` of a tile as MFMA operands (zeros where there is none): 8 elements of
// each 32 for every lane of the pair's column.
template <int DC, int N>
__device__ __forceinline__ void load_query(const LatentParams& p, const Tile& t, int pair, u32x4 (&q)[N]) {
  const int mq = (threadIdx.x >> 4) & 3;
  const u32x4* from = reinterpret_cast<const u32x4*>(p.q + (pair < t.pairs ? t.pair0 + pair : 0) * (DC + kRope)) + mq;
#pragma unroll
  for (int s = 0; s < N; ++s) q[s] = from[4 * s];
}
template <int N>
__device__ __forceinline__ void drop_query(bool real, u32x4 (&q)[N]) {
  if (!real) {
#pragma unroll
    for (int s = 0; s < N; ++s) q[s] = u32x4{0, 0, 0, 0};
  }
}
// Said to the compiler, not only to the hardware: it would otherwise wait for the queries, and with
// them for every chunk on its way, at each of their uses.
__device__ __forceinline__ void queries_are_here() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt 0

// N operands from LDS, each used by products: read in groups of G, one group ahead of the products.
// (Left alone, the compiler reads one operand, waits for it and multiplies, and with one wave on a
// SIMD nothing else fills the wait: a chunk of 32 positions and 16 pairs took 1.5 us so.)
template <int N, int G, class Read, class Use>
__device__ __forceinline__ void read_ahead(Read read, Use use) {
  static_assert(N % G == 0, "whole groups");
  u32x4 a[2][G];
#pragma unroll
  for (int i = 0; i < G; ++i) a[0][i] = read(i);
#pragma unroll
  for (int g = 0; g < N / G; ++g) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < G; ++i)
      if ((g + 1) * G + i < N) a[(g + 1) & 1][i] = read((g + 1) * G + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < G; ++i) use(g * G + i, a[g & 1][i]);
  }
  __builtin_amdgcn_sched_barrier(0);
}

template <bool BF16>
__device__ __forceinline__ bool is_finite(uint32_t bits) {
  constexpr uint32_t EXP = BF16 ? 0x7f80u : 0x7c00u;
  return (bits & EXP) != EXP;
}
// Non-finite elements of a word of two, replaced by zeros.
template <bool BF16>
__device__ __forceinline__ uint32_t finite_word(uint32_t w) {
  if (!is_finite<BF16>(w)) w &= 0xffff0000u;
  if (!is_finite<BF16>(w >> 16)) w &= 0xffffu;
  return w;
}

// Four elements of an output, or of a partial output.
template <bool BF16>
__device__ __forceinline__ void put_output(uint16_t* out, f32x4 o, float by) {
  *reinterpret_cast<u32x2*>(out) = u32x2{round_two<BF16>(o[0] * by, o[1] * by), round_two<BF16>(o[2] * by, o[3] * by)};
}

template <int DC, bool BF16, int NT>
__global__ __launch_bounds__(kThreads, 1) void latent_attention_kernel(const LatentParams p) {
  constexpr int NC = NT * 16;
  constexpr int KS = DC / 32;       // steps of q.k over the latent; two more over the rotary part
  constexpr int SLICE = DC / kWaves;     // elements of a wave's P.V
  constexpr int DT = SLICE / 16;
  // Waves that score (2 for each 16 pairs) and waves that fetch: the last four, which have no scores
  // up to 32 pairs, or all.
  constexpr int SCORING = 2 * NT;
  constexpr bool AHEAD = ahead(NT);
  constexpr int DEPTH = AHEAD ? 2 : kStages - 1;  // chunks on their way or here, beside those worked on
  constexpr int FETCHING = NT == 4 ? kWaves : 4;
  constexpr int MINE = kChunk / FETCHING;  // positions of a chunk that a wave fetches
  constexpr int LOADS = MINE * DC * 2 / 1024 + 1;
  typedef LatentShared<DC, NT> Shared;
  __shared__ Shared lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mt = lane & 15, mq = lane >> 4;
  const int kg = wave & 1, ct = wave >> 1;  // scores: positions 16 kg .. of the chunk, pairs 16 ct ..
  const bool scores = wave < SCORING;
  const int fetching = wave - (kWaves - FETCHING);  // which of those waves, below 0: none

  Walk<NC> walk;
  if (!find_place<NC>(p, lds, blockIdx.x, gridDim.x, walk)) return;

  const uint32_t lds_base = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) Shared*)&lds);
  auto rope_of = [](int chunk) { return AHEAD ? chunk % 3 : chunk & (kStages - 1); };
  // a lane's offsets into a stage (bytes)
  const int key = kg * 16 + mt;
  // (the others of its places differ from the first in a few bits, which costs an instruction each and no register)
  int k_first = key * DC * 2 + (mq ^ latent_swizzle(key)) * 16;
  int r_first = key * kRope * 2 + (mq ^ rope_swizzle(key)) * 16;
  int v_at[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    const int t = 4 * mq + (mt >> 2), piece = wave * (SLICE / 8) + 2 * i + ((mt & 3) >> 1);
    v_at[i] = t * DC * 2 + (piece >> 4) * 256 + ((piece & 15) ^ latent_swizzle(t)) * 16 + (mt & 1) * 8;
  }

  Piece piece;
  while (walk.next(p, piece)) {
    const Tile tile = tile_of<NC>(p, piece);
    const int my_pair = ct * 16 + mt;
    const bool real = scores && my_pair < tile.pairs;
    const int my_pos = real ? tile.first_pos + (piece.tile * NC + my_pair) / p.heads : -1;
    bool emptied = false;  // values lost non-finite elements
    bool far = false;      // of some pair's reference
    u32x4 q[KS + 2];
    f32x4 o[DT][NT];
    float m[NT], my_m = -INFINITY, l = 0.f;  // references of every pair; of my_pair, with its sum over this wave's positions
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      m[c] = -INFINITY;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    for (int w0 = piece.from; w0 < tile.to;) {
      const Window win = window_of(p, tile, w0);
      __syncthreads();
      stage_table(p, piece.request, win, lds.table);
      if (tid < 3) lds.flag[tid] = 0;
      __syncthreads();
      uint32_t slot = 0;  // of the next chunk to ask for, looked up ahead
      auto look_up = [&](int chunk) {
        if (chunk < win.w1)
          slot = slot_of<MINE>(p, lds.table, win.b0, chunk * kChunk + fetching * MINE, tile.context - 1);
      };
      auto get = [&](int chunk) {
        fetch<DC, MINE>(p, slot, fetching, lds_base + (uint32_t)((chunk & (kStages - 1)) * sizeof(lds.latent[0])),
                        lds_base + (uint32_t)(offsetof(Shared, rope) + rope_of(chunk) * sizeof(lds.rope[0])));
        look_up(chunk + 1);
      };
      if (fetching >= 0) {
        look_up(w0);
#pragma unroll
        for (int i = 0; i < DEPTH; ++i)
          if (w0 + i < win.w1) get(w0 + i);
      }
      if (scores && w0 == piece.from) load_query<DC>(p, tile, real ? my_pair : NC, q);
      if (scores) queries_are_here();
      drop_query(real, q);

      f32x4 s;       // the scores of a chunk
      float before;  // and the sum without it
      bool masked;
      auto flag_of = [&](int chunk) -> int32_t& { return lds.flag[AHEAD ? chunk % 3 : chunk & 1]; };
      // weights of this wave's scores under the reference my_m, on top of the sum `so_far`
      auto put_weights = [&](int chunk, float so_far) {
        const float base = my_m == -INFINITY ? 0.f : my_m;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fast_exp2(s[i] - base);
        u32x2 hi, lo;
        split_weights4<BF16>(w, hi, lo);
        if constexpr (!BF16) {  // the sum of the weights as rounded: where one outweighs the others its rounding cancels
          w[0] = Elem<false>::lo(hi.x), w[1] = Elem<false>::hi(hi.x);
          w[2] = Elem<false>::lo(hi.y), w[3] = Elem<false>::hi(hi.y);
        }
        l = so_far + ((w[0] + w[1]) + (w[2] + w[3]));
        const int row = my_pair * kChunk + (mq ^ weight_swizzle(my_pair)) * 8 + 4 * kg;
        auto& weight = lds.weight[AHEAD ? chunk & 1 : 0];
        *reinterpret_cast<u32x2*>(&weight[0][row]) = hi;
        if constexpr (split_p(BF16)) *reinterpret_cast<u32x2*>(&weight[1][row]) = lo;
      };
      auto score = [&](int chunk) {
        const int t0 = chunk * kChunk;
        const uint8_t* latent = reinterpret_cast<const uint8_t*>(lds.latent[chunk & (kStages - 1)]);
        const uint8_t* rope = reinterpret_cast<const uint8_t*>(lds.rope[rope_of(chunk)]);
        before = l;
        asm volatile("" : "+v"(k_first), "+v"(r_first));
        masked = t0 + kChunk > tile.context || t0 + kChunk - 1 > tile.least_pos;
        s = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 t{0.f, 0.f, 0.f, 0.f};  // (two sums: one would be a chain of products that wait for each other)
        read_ahead<KS + 2, KS != 16 ? 5 : NT == 4 ? 2 : 6>(
            [&](int k) { return *reinterpret_cast<const u32x4*>(k < KS ? latent + (k_first ^ (k & 3) << 6) + (k >> 2) * 256 : rope + (r_first ^ (k & 1) << 6)); },
            [&](int k, u32x4 a) {
              if (k & 1) t = mfma32<BF16>(a, q[k], t);
              else s = mfma32<BF16>(a, q[k], s);
            });
        s += t;
        bool passes = false, odd = false;
        const float limit = limit_of<BF16>(my_m, far);
        const int seen = min(my_pos, tile.context - 1) - t0 - kg * 16 - 4 * mq;  // of the lane's 4 positions: i <= seen
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (masked) odd |= !(__builtin_fabsf(s[i]) < INFINITY);
          const float t = product(s[i], p.scale_log2);
          s[i] = !masked || i <= seen ? t : -INFINITY;
          passes |= s[i] > limit;
        }
        const int word = (__builtin_amdgcn_ballot_w64(passes) ? 1 : 0) | (__builtin_amdgcn_ballot_w64(odd) ? 2 : 0);
        if (word && lane == 0) atomicOr(&flag_of(chunk), word);
        put_weights(chunk, before);
      };
      u32x4 v[DT];  // this wave's values of a chunk
      auto read_values = [&](int chunk) {
        const uint8_t* latent = reinterpret_cast<const uint8_t*>(lds.latent[chunk & (kStages - 1)]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint16_t* at = reinterpret_cast<const uint16_t*>(latent + v_at[d]);
          const u32x2 a = lds_read_transposed(at), b = lds_read_transposed(at + 16 * DC);
          v[d] = u32x4{a.x, a.y, b.x, b.y};
        }
      };
      // Where a score passed what its pair's reference reaches, or one is not finite; true: values changed.
      auto settle = [&](int chunk) {
        const int word = __builtin_amdgcn_readfirstlane(flag_of(chunk));
        if (!word) return false;
        if (word & 2) {  // (what they stand for comes after the loop)
          emptied = true;
          constexpr int PIECES = SLICE / 8;  // of this wave's values, which it alone reads from here on
          for (int i = lane; i < kChunk * PIECES; i += kWave) {
            const int t = i / PIECES, piece = wave * PIECES + i % PIECES;
            uint32_t* x = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(lds.latent[chunk & (kStages - 1)]) + t * DC * 2 +
                                                      (piece ^ latent_swizzle(t)) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = finite_word<BF16>(x[e]);
          }
        }
        // every pair's maximum over the chunk, then the state and the weights under the new one
        if (scores) {
          const float top = column_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
          if (mq == 0) lds.exchange[kg][my_pair] = top;
        }
        lds_barrier();
        float by = 1.f;  // of my_pair
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const float top = fmaxf(lds.exchange[0][c * 16 + mt], lds.exchange[1][c * 16 + mt]);
          // (a pair by its own scores alone: what others see must not change its roundings)
          const float now = top > limit_of<BF16>(m[c], true) ? top - lift(BF16) : m[c];
          const float b = now == m[c] ? 1.f : fast_exp2(m[c] - now);
          m[c] = now;
          if (c == ct) my_m = now, by = b;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][c] *= b;
        }
        if constexpr (!BF16) far |= __builtin_amdgcn_ballot_w64(__builtin_fabsf(my_m) >= 16777216.f && my_m != -INFINITY) != 0;
        if (scores) put_weights(chunk, before * by);
        lds_barrier();
        return (word & 2) != 0;
      };
      auto weigh = [&](int chunk) {  // O^T += V^T P^T
        const auto& weight = lds.weight[AHEAD ? chunk & 1 : 0];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const int row = (c * 16 + mt) * kChunk + (mq ^ weight_swizzle(mt)) * 8;
          const u32x4 hi = *reinterpret_cast<const u32x4*>(&weight[0][row]);
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][c] = mfma32<BF16>(v[d], hi, o[d][c]);
          if constexpr (split_p(BF16)) {
            const u32x4 lo = *reinterpret_cast<const u32x4*>(&weight[1][row]);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][c] = mfma32<BF16>(v[d], lo, o[d][c]);
          }
        }
      };

      if constexpr (AHEAD) {
        // One barrier a chunk. Of the two waves of a SIMD one weighs the last chunk and then scores this
        // one, the other the other way round: the products of one run beside the exponentials of the other.
        if (w0 + 1 < win.w1) wait_loads<LOADS>();
        else wait_loads<0>();
        lds_barrier();
        for (int chunk = w0; chunk <= win.w1; ++chunk) {
          if (tid == 0) lds.flag[(chunk + 1) % 3] = 0;
          const bool more = chunk + 2 < win.w1;
          if (wave < 4) {
            if (more) get(chunk + 2);
            if (chunk > w0) {
              read_values(chunk - 1);
              weigh(chunk - 1);
            }
          }
          if (chunk < win.w1) score(chunk);
          if (wave >= 4) {
            if (more) get(chunk + 2);
            if (chunk > w0) {
              read_values(chunk - 1);
              weigh(chunk - 1);
            }
          }
          if (more) wait_loads<LOADS>();
          else wait_loads<0>();
          lds_barrier();  // the next chunk is here, and this one's weights
          if (chunk < win.w1) settle(chunk);
        }
      } else {
        for (int chunk = w0; chunk < win.w1; ++chunk) {
          if (fetching >= 0) {
            if (chunk + 2 < win.w1) wait_loads<2 * LOADS>();
            else if (chunk + 1 < win.w1) wait_loads<LOADS>();
            else wait_loads<0>();
          }
          lds_barrier();  // the chunk is here, and nobody works on the one before it
          if (fetching >= 0 && chunk + DEPTH < win.w1) get(chunk + DEPTH);
          if (tid == 0) lds.flag[(chunk + 1) & 1] = 0;
          if (scores) score(chunk);
          read_values(chunk);  // on their way while the wave waits for the weights
          lds_barrier();
          if (settle(chunk)) read_values(chunk);
          weigh(chunk);
        }
      }
      w0 = win.w1;
    }

    if (emptied) {
      // NaN for the pairs that see such an element (0 times infinity where its score is -inf, and what the
      // score made of it elsewhere), in the chunks that some pair does not see whole
      const int first_chunk = max(piece.from, max(0, tile.least_pos + 1) / kChunk);
#pragma unroll 1
      for (int t = first_chunk * kChunk; t < min(tile.to * kChunk, tile.context); ++t) {
        const uint32_t block = quotient((uint32_t)t, p.by_block);
        const uint32_t id = (uint32_t)p.block_table[piece.request * p.table_stride + block];
        const uint64_t slot = (uint64_t)(id < (uint32_t)p.num_blocks ? id : 0u) * (uint32_t)p.block_size + ((uint32_t)t - block * (uint32_t)p.block_size);
        const uint16_t* from = p.cache + slot * (DC + kRope) + wave * SLICE + 4 * mq;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(from + d * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool off = !is_finite<BF16>((i & 2 ? x.y : x.x) >> (16 * (i & 1)) & 0xffffu);
#pragma unroll
            for (int c = 0; c < NT; ++c)
              if (off && tile.first_pos + (piece.tile * NC + c * 16 + mt) / p.heads >= t) o[d][c][i] = NAN;
          }
        }
      }
    }

    // --- the tile's sums, and its output or this workgroup's part of it
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    lds_barrier();  // the exchange may still be read
    if (scores && mq == 0) lds.exchange[kg][my_pair] = l;
    lds_barrier();
    const int slot = 2 * blockIdx.x + (piece.from == 0 ? 1 : 0);
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const int pair = c * 16 + mt;
      const float sum = lds.exchange[0][pair] + lds.exchange[1][pair];
      if (pair >= tile.pairs) continue;
      const int e0 = wave * SLICE + 4 * mq;
      if (piece.whole) {
        const float by = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t* out = static_cast<uint16_t*>(p.out) + (tile.pair0 + pair) * DC + e0;
#pragma unroll
        for (int d = 0; d < DT; ++d) put_output<BF16>(out + d * 16, o[d][c], by);
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
}

// Joins the parts of a tile that workgroups share. Block (g, y): the tile that workgroup g begins
// inside, unless an earlier one does too; a wave takes a pair, lanes DC / 64 elements each.
template <int DC, bool BF16, int NC>
__global__ __launch_bounds__(256) void latent_merge_kernel(const LatentParams p, int groups) {
  constexpr int EPL = DC / 64;
  const int g = blockIdx.x + 1, lane = threadIdx.x & 63;
  const int32_t* place = p.places + g * kPlaceWords;
  const int total = p.places[5], active = p.places[6];
  if (g >= active) return;
  const int chunk = place[1], chunks = place[3];
  if (chunk == 0) return;
  auto begin_of = [&](int i) { return (int)((int64_t)i * total / active); };
  const int start = begin_of(g) - chunk;  // of the tile's chunks
  if (begin_of(g - 1) > start) return;
  int last = g;  // the last workgroup with chunks of this tile
  while (last + 1 < active && begin_of(last + 1) < start + chunks) ++last;
  const int pair = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int tile = place[0], rows = place[4];
  const int64_t at = (int64_t)place[2] * p.heads + tile * NC + pair;
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
  for (int e = 0; e < EPL; e += 4) put_output<BF16>(out + e * 64, f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]}, by);
}

template <int DC, bool BF16>
hipError_t launch_type(const LatentParams& p, int pairs, int compute_units, hipStream_t stream) {
  const dim3 grid(compute_units), merge_grid(compute_units - 1, pairs / 4);
  if (pairs == 16) hipLaunchKernelGGL((latent_attention_kernel<DC, BF16, 1>), grid, dim3(kThreads), 0, stream, p);
  else if (pairs == 32) hipLaunchKernelGGL((latent_attention_kernel<DC, BF16, 2>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((latent_attention_kernel<DC, BF16, 4>), grid, dim3(kThreads), 0, stream, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || compute_units < 2) return err;
  if (pairs == 16) hipLaunchKernelGGL((latent_merge_kernel<DC, BF16, 16>), merge_grid, dim3(256), 0, stream, p, compute_units);
  else if (pairs == 32) hipLaunchKernelGGL((latent_merge_kernel<DC, BF16, 32>), merge_grid, dim3(256), 0, stream, p, compute_units);
  else hipLaunchKernelGGL((latent_merge_kernel<DC, BF16, 64>), merge_grid, dim3(256), 0, stream, p, compute_units);
  return hipGetLastError();
}

}  // namespace

int64_t latent_tile_units(int pairs, int64_t length) {
  return (length < kChunk ? 1 : (length + kChunk - 1) / kChunk) + tile_cost(pairs);
}

// Pairs of a tile. Larger tiles read a context less often and take fewer products of few rows; smaller ones
// make more work to share while there is not enough for every compute unit, and start and end sooner. With u
// units a workgroup (as they are dealt out above) a launch takes about 13 + 1.15 u us with 16 pairs, 14 + 1.45 u
// with 32 and 20 + 1.7 u with 64, fitted to 40 drawn steps and these (measured with 16, 32 and 64 pairs, main
// kernel): 16 heads over 64 requests of 4096 positions 54, 55, 74 us, over 4 short ones 15, 17, 27; 128 heads over
// 61 uneven requests 158, 95, 79; 4 rows of 32 heads over 4096 positions 175, 100, 69. Whole calls: 8 rows of 16
// heads for 2 requests of 321 at most 17, 21, 32; 40 to 64 rows of 32 heads for 4 of 918 38, 35, 39.
struct TileChoice {
  int64_t units[3] = {0, 0, 0};
  void add(int64_t requests, int64_t pairs, int64_t length) {
    for (int i = 0; i < 3; ++i) units[i] += requests * ((pairs + (16 << i) - 1) / (16 << i)) * latent_tile_units(16 << i, length);
  }
  int best(int compute_units) const {
    constexpr double START[3] = {13, 14, 20}, EACH[3] = {1.15, 1.45, 1.7};
    int found = 16;
    double least = 0;
    for (int i = 0; i < 3; ++i) {
      const int64_t most = units[i] / (tile_cost(16 << i) + kLeastChunks);
      const int64_t workgroups = most < 1 ? 1 : most < compute_units ? most : compute_units;
      const double us = START[i] + EACH[i] * (double)units[i] / (double)workgroups;
      if (i == 0 || us < least) found = 16 << i, least = us;
    }
    return found;
  }
};

int latent_tile_pairs(const int32_t* rows, const int32_t* kv_lengths, int32_t n_requests, int32_t heads, int compute_units) {
  TileChoice choice;
  for (int32_t b = 0; b < n_requests; ++b)
    if (rows[b] > 0) choice.add(1, (int64_t)rows[b] * heads, kv_lengths[b]);
  return choice.best(compute_units);
}

// Where the lengths are not known: requests of as many rows each, over 2048 positions.
int latent_tile_pairs(int64_t n_rows, int32_t n_requests, int32_t heads, int compute_units) {
  TileChoice choice;
  if (n_requests > 0) choice.add(n_requests, (n_rows + n_requests - 1) / n_requests * heads, 2048);
  return choice.best(compute_units);
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
