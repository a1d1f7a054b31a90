// Step tables built on the GPU (gfx950): blocks for the requests that lack them, every row's
// request, position and slot, and a decode bucket's v2 split (see ayaka_hip_tables.h).
//
// Two sums over the requests say everything: the rows before a request, and the new blocks handed
// out before it. A workgroup makes both in LDS -- a few thousand requests at most, so each makes
// them for itself rather than waiting for another to -- and then every row, and every new block,
// finds its request by bisection and computes its own numbers, independent of all the others.
//
// Nothing here is bound by bytes or operations: what counts is the chain of dependent steps. So what
// a later step reads from memory is fetched with the requests (the entry where a request's last
// token lies, and for a decode bucket the free blocks its rows could at most be given), the sums
// are wave scans on DPP in saturating 32-bit integers, and the split's candidate sizes are all
// summed at once, 32 sizes by as many slices of the requests as the workgroup has threads for.
// Steps of many rows spread over workgroups of 256 rows; the last of them to finish (by a
// counter) writes the words that the others read, so the pool's state and the lengths may be
// updated in place.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "ayaka_hip_internal.h"
#include "kv_address.h"

namespace ayk {

namespace {

constexpr int kBins = 256;
constexpr int kMaxWaves = 16;
// Free blocks a decode bucket fetches ahead (its rows need one each at most).
constexpr int kAhead = 1024;

struct Scratch {
  uint32_t wave_sum[3][kMaxWaves];
  uint32_t given, left_out, longest, partial_at, empty_at, last;
  unsigned long long total;
  uint32_t items[AYK_TABLES_SIZES];
  uint32_t bins[kBins];
};

// x + y, or UINT32_MAX: the sums only ever meet limits below that.
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// x of the lane the control names, 0 where it names none (or its rows are masked off).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}

// The sum of x over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = add_sat(x, dpp<0x111>(x));  // row_shr: within 16 lanes
  x = add_sat(x, dpp<0x112>(x));
  x = add_sat(x, dpp<0x114>(x));
  x = add_sat(x, dpp<0x118>(x));
  x = add_sat(x, dpp<0x142, 0xA>(x));  // row_bcast15 into rows 1 and 3
  x = add_sat(x, dpp<0x143, 0xC>(x));  // row_bcast31 into rows 2 and 3
  return x;
}

// Sum of x over the workgroup's threads before this one, and over all of them. One barrier: a
// workgroup's successive scans use different `k`.
__device__ __forceinline__ uint32_t scan_exclusive(uint32_t x, Scratch& s, int k, uint32_t* all = nullptr) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const uint32_t upto = wave_scan(x);
  if (lane == 63) s.wave_sum[k][wave] = upto;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kMaxWaves; ++w) {
    const uint32_t v = w < waves ? s.wave_sum[k][w] : 0u;
    before = add_sat(before, w < wave ? v : 0u);
    total = add_sat(total, v);
  }
  if (all) *all = total;
  const uint32_t previous = (uint32_t)__shfl_up((int)upto, 1);
  return add_sat(before, lane ? previous : 0u);
}

// The first request whose running sum passes i, or n.
__device__ __forceinline__ int find(const uint32_t* sums, int n, uint32_t i) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ uint32_t divide(uint32_t t, uint32_t magic, int32_t shift) {  // t < 2^31
  return (__umulhi(t, magic) + t) >> shift;
}
__device__ __forceinline__ int block_at(const TablesParams& p, int t) {
  return (int)divide((uint32_t)t, p.bs_magic, p.bs_shift);
}
__device__ __forceinline__ int blocks_for(const TablesParams& p, int tokens) {
  return tokens > 0 ? block_at(p, tokens - 1) + 1 : 0;
}

// The v2 split of the rows' lengths, s_len[b] - 1 each, into p.staged. s_end is free to use; the
// scratch's longest and total are those of the lengths.
__device__ void stage_split(const TablesParams& p, const int32_t* s_len, uint32_t* s_end, Scratch& s) {
  uint32_t* s_items = s.items;  // both cleared by the caller
  uint32_t* s_bins = s.bins;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.n_requests, per = (n + threads - 1) / threads;
  const int lo = min(tid * per, n), hi = min(n, lo + per);
  {
    // Work items of every size: thread t sums size t % 32 over every (threads / 32)-th request. A
    // request counts 2^18 partitions at most (more than any list holds), so no sum overflows.
    const int c = tid % AYK_TABLES_SIZES;
    uint32_t items = 0;
    if (c < p.n_sizes) {
      const uint32_t magic = p.size_magic[c];
      const int32_t shift = p.size_shift[c];
      for (int b = tid / AYK_TABLES_SIZES; b < n; b += threads / AYK_TABLES_SIZES) {
        const int len = s_len[b] + 1;
        items += len > 0 ? min(divide((uint32_t)(len - 1), magic, shift) + 1, 1u << 18) : 0u;
      }
      if (items) atomicAdd(&s_items[c], items);
    }
  }
  __syncthreads();
  const int longest = (int)s.longest;
  const uint32_t empties = s.empty_at;  // rows without context
  // A size's time, in positions: its work spread over the compute units plus 0.3 of its longest
  // item (what the last to finish trails by); a launch of one round takes its longest item. Over
  // 600 drawn batches this picks sizes 2.6% behind the scheduled model's on average. Every wave
  // decides for itself, a size per lane: the least of {time's upper bits, size's place}.
  uint32_t key = 0xffffffffu;
  if (lane < p.n_sizes) {
    const int size = p.sizes[lane];
    const uint32_t items = s_items[lane];
    const float item = (float)(min(size, longest) + p.cost);
    const float groups = (float)p.groups, units = (float)p.compute_units;
    float time = ((float)s.total + (float)p.cost * (float)items) * groups / units + 0.3f * item;
    if ((float)items * groups <= units) time = item;
    // sizes up to the first that covers the longest row; of those whose lists are so long that
    // start-up costs decide (8 rounds of the GPU), the largest
    const bool offered = lane == 0 || p.sizes[lane - 1] < longest;
    if ((float)items * groups > 8.f * units) time = 1e30f * (float)(1 + AYK_TABLES_SIZES - lane);
    if (offered && items + empties <= (uint32_t)p.capacity) key = (__float_as_uint(time) & ~31u) | (uint32_t)lane;
  }
#pragma unroll
  for (int st = 1; st < 64; st <<= 1) key = min(key, (uint32_t)__shfl_xor((int)key, st));
  const bool fits = key != 0xffffffffu;
  const int pick = fits ? (int)(key & 31u) : 0;
  const uint32_t size = fits ? (uint32_t)p.sizes[pick] : (uint32_t)max(p.sizes[0], (longest + 63) / 64 * 64);

  // Full partitions and partial ones before each row in one sum (13 bits hold every request's
  // partial one, the API holds the list to 2^18 items).
  uint32_t mine = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)(s_len[b] + 1), full = len / size;
    mine += full << 13 | (uint32_t)(full * size != len);
  }
  uint32_t all;
  uint32_t at = scan_exclusive(mine, s, 2, &all);
  int32_t* work = p.staged + 2 + n;
  const uint32_t fulls = all >> 13, partials = all & 0x1fffu;
  auto bin_of = [&](uint32_t rest) { return kBins - 1 - (int)(((uint64_t)(rest - 1) * kBins) / size); };
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)(s_len[b] + 1), full = len / size, rest = len - full * size;
    p.staged[2 + b] = (int32_t)((at >> 13) + (at & 0x1fffu));
    if (rest) atomicAdd(&s_bins[bin_of(rest)], 1u);
    at += full << 13 | (uint32_t)(rest != 0);
    s_end[b] = at >> 13;
  }
  __syncthreads();
  if (wave == 0) {  // the bins' first places: four bins per lane
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = s_bins[4 * lane + k];
      sum += c[k];
    }
    uint32_t first = fulls + wave_scan(sum) - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_bins[4 * lane + k] = first;
      first += c[k];
    }
  }
  if (tid == 64 % threads) s.empty_at = fulls + partials;
  __syncthreads();
  // The order within a bin, and among the rows without context (last: their workgroups write
  // zeros), is the threads': it decides when an item runs, not what it computes.
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)(s_len[b] + 1), full = len / size, rest = len - full * size;
    if (rest || len == 0) {
      const uint32_t i = atomicAdd(rest ? &s_bins[bin_of(rest)] : &s.empty_at, 1u);
      work[2 * i] = b;
      work[2 * i + 1] = (int32_t)full;
    }
  }
  for (uint32_t i = tid; i < fulls; i += threads) {
    const int b = find(s_end, n, i);
    work[2 * i] = b;
    work[2 * i + 1] = (int32_t)(i - (b ? s_end[b - 1] : 0));
  }
  if (tid == 0) {
    p.staged[0] = (int32_t)size;
    p.staged[1] = (int32_t)(fulls + partials + empties);
  }
}

// DECODE: one row per request, and the v2 split after it (one workgroup).
template <bool DECODE>
__global__ __launch_bounds__(1024) void step_tables_kernel(const TablesParams p) {
  extern __shared__ uint32_t smem[];
  __shared__ Scratch s;
  const int n = p.n_requests;
  uint32_t* s_end = smem;                                       // rows of the requests up to and with each
  uint32_t* s_upto = smem + n;                                  // new blocks, the same, if all could be served
  int32_t* s_before = reinterpret_cast<int32_t*>(smem + 2 * n);  // tokens before the step; -1: not served
  int32_t* s_last = reinterpret_cast<int32_t*>(smem + 3 * n);    // the block of the last of them
  int32_t* s_free = reinterpret_cast<int32_t*>(smem + 4 * n);    // DECODE: the first free blocks
  const int tid = threadIdx.x, threads = blockDim.x;
  const int per = (n + threads - 1) / threads;
  const int lo = min(tid * per, n), hi = min(n, lo + per);
  auto rows_of = [&](int b) { return DECODE ? 1 : p.rows[b]; };

  const int taken = min(max(*p.taken, 0), p.n_free);
  const int room = p.n_free - taken;
  if (tid == 0) {
    s.given = s.left_out = s.longest = s.empty_at = 0;
    s.total = 0;
  }
  uint32_t sum = lo;  // rows before this thread's requests
  if constexpr (DECODE) {
    for (int i = tid; i < AYK_TABLES_SIZES + kBins; i += threads) (i < kBins ? s.bins[i] : s.items[i - kBins]) = 0;
    for (int i = tid; i < min(min(n, room), kAhead); i += threads) s_free[i] = p.free_blocks[taken + i];
  } else {
    uint32_t rows = 0;
    for (int b = lo; b < hi; ++b) rows = add_sat(rows, (uint32_t)max(p.rows[b], 0));
    sum = scan_exclusive(rows, s, 0);
  }
  const int64_t limit = (int64_t)p.max_blocks * p.block_size;
  uint32_t need = 0;
  for (int b = lo; b < hi; ++b) {
    const int r = rows_of(b), len = p.lengths[b];
    sum = add_sat(sum, (uint32_t)max(r, 0));
    bool live = r >= 0 && len > 0 && r <= len && len <= limit && sum <= (uint32_t)p.n_rows;
    const int had = live ? blocks_for(p, len - r) : 0;
    const int last = had > 0 ? p.block_table[(int64_t)b * p.table_stride + had - 1] : -1;
    // the padding block where the last token before the step lies: a block it was never given
    if (last == 0) live = false;
    const int want = live ? blocks_for(p, len) - had : 0;
    need = add_sat(need, (uint32_t)want);
    s_end[b] = sum;
    s_upto[b] = (uint32_t)want;  // made a running sum below
    s_before[b] = live ? len - r : -1;
    s_last[b] = last;
  }
  need = scan_exclusive(need, s, 1);
  uint32_t given = 0, left_out = 0, longest = 0, empty = 0;
  unsigned long long total = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t want = s_upto[b];
    need = add_sat(need, want);
    const bool served = s_before[b] >= 0 && (want == 0 || need <= (uint32_t)room);
    if (served && want > 0) given = need;
    if (!served) {
      left_out += p.lengths[b] != 0;
      s_before[b] = -1;
    }
    s_upto[b] = need;
    if constexpr (DECODE) {
      const uint32_t len = (uint32_t)(s_before[b] + 1);
      longest = max(longest, len);
      total += len;
      empty += len == 0;
    }
  }
  if (given) atomicMax(&s.given, given);
  if (left_out) atomicAdd(&s.left_out, left_out);
  if constexpr (DECODE) {
    if (longest) atomicMax(&s.longest, longest);
    if (total) atomicAdd(&s.total, total);
    if (empty) atomicAdd(&s.empty_at, empty);
  }
  __syncthreads();
  given = s.given;

  // the rows
  for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < p.n_rows; i += (int64_t)gridDim.x * threads) {
    const int row = (int)i;
    const int b = DECODE ? row : find(s_end, n, (uint32_t)row);
    int32_t pos = 0;
    int64_t slot = 0;
    if (b < n && s_before[b] >= 0) {
      const int before = s_before[b];
      pos = DECODE ? before : before + row - (int)(b ? s_end[b - 1] : 0u);
      const int at = block_at(p, pos), had = blocks_for(p, before);
      int id;
      if (at < had) {
        id = s_last[b];  // a row's block is new or the one of the last token before the step
      } else {
        const int k = (int)(b ? s_upto[b - 1] : 0u) + at - had;
        id = DECODE && k < kAhead ? s_free[k] : p.free_blocks[taken + k];
      }
      slot = (int64_t)id * p.block_size + (pos - at * p.block_size);
      if (DECODE && at >= had) p.block_table[(int64_t)b * p.table_stride + at] = id;
    }
    if (p.request_of_row) p.request_of_row[row] = b < n ? b : 0;
    p.positions[row] = pos;
    p.slot_mapping[row] = slot;
  }
  if constexpr (DECODE) {
    stage_split(p, s_before, s_end, s);
    // (its barriers are past every read of the lengths and the pool's state)
  } else {
    // the new blocks' entries
    for (uint32_t i = blockIdx.x * threads + tid; i < given; i += gridDim.x * threads) {
      const int b = find(s_upto, n, i);
      const int had = blocks_for(p, s_before[b]);
      p.block_table[(int64_t)b * p.table_stride + had + (i - (b ? s_upto[b - 1] : 0u))] = p.free_blocks[taken + i];
    }
    __syncthreads();
    if (gridDim.x > 1) {  // the last workgroup to get here, when all have read the lengths and the state
      if (tid == 0) {
        const uint32_t before = __hip_atomic_fetch_add(reinterpret_cast<uint32_t*>(p.after + 2), 1u, __ATOMIC_ACQ_REL,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        s.last = before + 1 == gridDim.x;
      }
      __syncthreads();
      if (!s.last) return;
    }
  }
  for (int b = lo; b < hi; ++b) {
    const int rows = DECODE ? 1 : (int)(s_end[b] - (b ? s_end[b - 1] : 0u));
    p.kv_lengths[b] = s_before[b] >= 0 ? s_before[b] + rows : 0;
  }
  if (tid == 0) {
    p.after[0] = taken + (int32_t)given;
    p.after[1] = (int32_t)s.left_out;
    p.after[2] = 0;
  }
}

}  // namespace

hipError_t launch_step_tables(const TablesParams& p, hipStream_t stream) {
  const size_t words = 4 * (size_t)p.n_requests;
  if (p.staged) {  // one workgroup: the split needs every row's length
    const int threads = p.n_requests <= 64 ? 256 : p.n_requests <= 256 ? 512 : 1024;
    const size_t ahead = p.n_requests < kAhead ? (size_t)p.n_requests : (size_t)kAhead;
    hipLaunchKernelGGL(step_tables_kernel<true>, dim3(1), dim3(threads), (words + ahead) * sizeof(int32_t), stream, p);
  } else {  // a row per thread, as far as one round of the GPU goes
    const int64_t groups = ((int64_t)p.n_rows + 255) / 256;
    const unsigned grid = (unsigned)(groups < 1 ? 1 : groups > 256 ? 256 : groups);
    hipLaunchKernelGGL(step_tables_kernel<false>, dim3(grid), dim3(256), words * sizeof(int32_t), stream, p);
  }
  return hipGetLastError();
}

}  // namespace ayk
