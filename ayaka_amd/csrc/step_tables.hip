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
// token lies, a decode bucket's partition sizes, and the free blocks its rows could at most be
// given), the sums are wave scans on DPP in saturating 32-bit integers, and the split's candidate
// sizes are summed at once, 32 sizes by as many slices of the requests as the workgroup has threads
// for. Steps of many rows spread over workgroups of 256 rows; the last of them to finish (by a
// counter) writes the words that the others read, so the pool's state and the lengths may be
// updated in place.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "ayaka_hip_internal.h"
#include "kv_address.h"

namespace ayk {

namespace {

constexpr int kSizes = AYK_TABLES_SIZES;
constexpr int kBins = 256;
// Free blocks a decode bucket fetches ahead (its rows need one each at most).
constexpr int kAhead = 1024;

template <int WAVES>
struct Scratch {
  uint32_t sums[3][WAVES];    // the waves' totals of each scan
  uint32_t found[5][WAVES];   // and of what the requests come to
  uint32_t size[kSizes], magic[kSizes], shift[kSizes], items[kSizes];
  uint32_t bins[kBins];
  uint32_t empty_at, last;
};

// x + y, or UINT32_MAX: the sums only ever meet limits below that.
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// x of the lane the control names, 0 where it names none (or its rows are masked off).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}

// f over the lanes up to and with this one (f(x, 0) = x); lane 63 has the wave's.
template <class F>
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, F f) {
  x = f(x, dpp<0x111>(x));  // row_shr: within 16 lanes
  x = f(x, dpp<0x112>(x));
  x = f(x, dpp<0x114>(x));
  x = f(x, dpp<0x118>(x));
  x = f(x, dpp<0x142, 0xA>(x));  // row_bcast15 into rows 1 and 3
  x = f(x, dpp<0x143, 0xC>(x));  // row_bcast31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) { return x > y ? x : y; }

// Sum of x over the workgroup's threads before this one, and over all of them. One barrier; each of
// a workgroup's scans has a `sums` of its own.
template <int WAVES>
__device__ __forceinline__ uint32_t scan_exclusive(uint32_t x, uint32_t (&sums)[WAVES], uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t upto = wave_scan(x, add_sat);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const uint32_t v = sums[w];
    before = add_sat(before, w < wave ? v : 0u);
    total = add_sat(total, v);
  }
  all = total;
  return add_sat(before, dpp<0x138>(upto));  // wave_shr: the lane before
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

// The v2 split of the rows' lengths into p.staged: s_before[b] + 1 each, below 1 for none; `longest`
// of them, `total` their sum (saturating), `empties` rows without context. s_end is free to use.
template <int THREADS>
__device__ __forceinline__ void stage_split(const TablesParams& p, const int32_t* s_before, uint32_t* s_end,
                                            Scratch<THREADS / 64>& s, int longest, uint32_t total, uint32_t empties) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.n_requests, per = (n + THREADS - 1) / THREADS;
  const int lo = min(tid * per, n), hi = min(n, lo + per);
  {
    // Work items of every size: thread t sums size t % 32 over every (threads / 32)-th request. A
    // request counts 2^18 partitions at most (more than any list holds), so no sum overflows.
    const int c = tid % kSizes;
    const uint32_t magic = s.magic[c];
    const int32_t shift = s.shift[c];
    uint32_t items = 0;
    for (int b = tid / kSizes; b < n; b += THREADS / kSizes) {
      const int before = s_before[b];
      items += before >= 0 ? min(divide((uint32_t)before, magic, shift) + 1, 1u << 18) : 0u;
    }
    atomicAdd(&s.items[c], items);
  }
  __syncthreads();
  // A size's time, in positions: its work spread over the compute units plus 0.3 of its longest
  // item (what the last to finish trails by); a launch of one round takes its longest item. Over
  // 600 drawn batches this picks sizes 2.6% behind the scheduled model's on average. Every wave
  // decides for itself, a size per lane: the least {time's upper bits, size's place}.
  const int slot = lane % kSizes;
  const uint32_t items = s.items[slot];
  uint32_t key = 0xffffffffu;
  {
    const int candidate = (int)s.size[slot];
    const float item = (float)(min(candidate, longest) + p.cost);
    const float groups = (float)p.groups, units = (float)p.compute_units;
    float time = ((float)total + (float)p.cost * (float)items) * groups / units + 0.3f * item;
    if ((float)items * groups <= units) time = item;
    // sizes up to the first that covers the longest row; of those whose lists are so long that
    // start-up costs decide (8 rounds of the GPU), the largest
    const bool offered = slot < p.n_sizes && (slot == 0 || (int)s.size[slot - 1] < longest);
    if ((float)items * groups > 8.f * units) time = 1e30f * (float)(1 + kSizes - slot);
    if (offered && items + empties <= (uint32_t)p.capacity) key = (__float_as_uint(time) & ~31u) | (uint32_t)slot;
  }
  key = ~__builtin_amdgcn_readlane(wave_scan(~key, larger), 63);
  uint32_t size = (uint32_t)max((int)s.size[0], (longest + 63) / 64 * 64);  // no size's list fits: a partition per row
  if (key != 0xffffffffu) size = s.size[key & 31u];
  size = __builtin_amdgcn_readfirstlane(size);

  // Full partitions and partial ones before each row in one sum (13 bits hold every request's
  // partial one, the API holds the list to 2^18 items).
  uint32_t mine = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)max(s_before[b] + 1, 0), full = len / size;
    mine += full << 13 | (uint32_t)(full * size != len);
    s_end[b] = full;
  }
  uint32_t all;
  uint32_t at = scan_exclusive(mine, s.sums[2], all);
  int32_t* work = p.staged + 2 + n;
  const uint32_t fulls = all >> 13, partials = all & 0x1fffu;
  const float per_bin = (float)kBins / (float)(size + 1);
  auto bin_of = [&](uint32_t rest) { return max(kBins - 1 - (int)((float)rest * per_bin), 0); };
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)max(s_before[b] + 1, 0), full = s_end[b], rest = len - full * size;
    p.staged[2 + b] = (int32_t)((at >> 13) + (at & 0x1fffu));
    if (rest) atomicAdd(&s.bins[bin_of(rest)], 1u);
    at += full << 13 | (uint32_t)(rest != 0);
    s_end[b] = at >> 13;
  }
  if (tid == 0) s.empty_at = fulls + partials;
  __syncthreads();
  if (wave == 0) {  // the bins' first places: four bins per lane
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = s.bins[4 * lane + k];
      sum += c[k];
    }
    uint32_t first = fulls + wave_scan(sum, add_sat) - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s.bins[4 * lane + k] = first;
      first += c[k];
    }
  }
  // full partitions by their place in the list, while wave 0 is at the bins
  for (uint32_t i = tid; i < fulls; i += THREADS) {
    const int b = find(s_end, n, i);
    work[2 * i] = b;
    work[2 * i + 1] = (int32_t)(i - (b ? s_end[b - 1] : 0));
  }
  __syncthreads();
  // The order within a bin, and among the rows without context (last: their workgroups write
  // zeros), is the threads': it decides when an item runs, not what it computes.
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)max(s_before[b] + 1, 0);
    const uint32_t full = s_end[b] - (b ? s_end[b - 1] : 0), rest = len - full * size;
    if (rest || len == 0) {
      const uint32_t i = atomicAdd(rest ? &s.bins[bin_of(rest)] : &s.empty_at, 1u);
      work[2 * i] = b;
      work[2 * i + 1] = (int32_t)full;
    }
  }
  if (tid == 0) {
    p.staged[0] = (int32_t)size;
    p.staged[1] = (int32_t)(fulls + partials + empties);
  }
}

// DECODE: one row per request, and the v2 split after it (one workgroup).
template <bool DECODE, int THREADS>
__global__ __launch_bounds__(THREADS) void step_tables_kernel(const TablesParams p) {
  extern __shared__ uint32_t smem[];
  constexpr int WAVES = THREADS / 64;
  __shared__ Scratch<WAVES> s;
  const int n = p.n_requests;
  uint32_t* s_end = smem;                                        // rows of the requests up to and with each
  uint32_t* s_upto = smem + n;                                   // new blocks, the same, if all could be served
  int32_t* s_before = reinterpret_cast<int32_t*>(smem + 2 * n);  // tokens before the step; below 0: not served
  int32_t* s_last = reinterpret_cast<int32_t*>(smem + 3 * n);    // the block of the last of them
  int32_t* s_free = reinterpret_cast<int32_t*>(smem + 4 * n);    // DECODE: the first free blocks
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (n + THREADS - 1) / THREADS;
  const int lo = min(tid * per, n), hi = min(n, lo + per);

  const int taken = min(max(*p.taken, 0), p.n_free);
  const int room = p.n_free - taken;
  const int64_t limit = (int64_t)p.max_blocks * p.block_size;
  uint32_t rows = 0;
  for (int b = lo; b < hi; ++b) {
    const int r = DECODE ? 1 : p.rows[b], len = p.lengths[b];
    // what a request may be by itself; a row count past any length is not
    const bool live = r >= 0 && len > 0 && r <= len && len <= limit;
    const int had = live ? blocks_for(p, len - r) : 0;
    s_last[b] = had > 0 ? p.block_table[(int64_t)b * p.table_stride + had - 1] : -1;
    s_end[b] = (uint32_t)max(r, 0);
    s_before[b] = live ? len - r : len != 0 ? -1 : -2;  // -2: padding
    rows = add_sat(rows, (uint32_t)max(r, 0));
  }
  if constexpr (DECODE) {
    static_assert(THREADS >= kBins, "cleared in one pass");
    if (tid < kBins) s.bins[tid] = 0;
    if (tid < kSizes) {
      s.items[tid] = 0;
      s.size[tid] = (uint32_t)p.sizes[tid];
      s.magic[tid] = p.size_magic[tid];
      s.shift[tid] = (uint32_t)p.size_shift[tid];
    }
    for (int i = tid; i < min(min(n, room), kAhead); i += THREADS) s_free[i] = p.free_blocks[taken + i];
  }
  uint32_t all, sum = lo;  // rows before this thread's requests
  if constexpr (!DECODE) sum = scan_exclusive(rows, s.sums[0], all);
  uint32_t need = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t r = s_end[b];
    const int before = s_before[b];
    sum = add_sat(sum, r);
    // (an entry of 0, the padding block, where the last token before the step lies: a block that the
    // request was never given)
    const bool live = before >= 0 && sum <= (uint32_t)p.n_rows && s_last[b] != 0;
    const int want = live ? blocks_for(p, before + (int)r) - blocks_for(p, before) : 0;
    need = add_sat(need, (uint32_t)want);
    s_end[b] = sum;
    s_upto[b] = (uint32_t)want;  // made a running sum below
    if (before >= 0 && !live) s_before[b] = -1;
  }
  need = scan_exclusive(need, s.sums[1], all);
  uint32_t given = 0, left_out = 0, longest = 0, total = 0, empty = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t want = s_upto[b];
    need = add_sat(need, want);
    int before = s_before[b];
    if (before >= 0 && want > 0) {
      if (need <= (uint32_t)room) given = need;
      else s_before[b] = before = -1;
    }
    left_out += before == -1;
    s_upto[b] = need;
    if constexpr (DECODE) {
      const uint32_t len = (uint32_t)max(before + 1, 0);
      longest = larger(longest, len);
      total = add_sat(total, len);
      empty += len == 0;
    }
  }
  // what the requests come to: over the wave, and (after the barrier) over the workgroup
  given = wave_scan(given, larger);
  left_out = wave_scan(left_out, add_sat);
  if constexpr (DECODE) {
    longest = wave_scan(longest, larger);
    total = wave_scan(total, add_sat);
    empty = wave_scan(empty, add_sat);
  }
  if (lane == 63) {
    s.found[0][wave] = given;
    s.found[1][wave] = left_out;
    s.found[2][wave] = longest;
    s.found[3][wave] = total;
    s.found[4][wave] = empty;
  }
  __syncthreads();
  given = left_out = longest = total = empty = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    given = larger(given, s.found[0][w]);
    left_out += s.found[1][w];
    if constexpr (DECODE) {
      longest = larger(longest, s.found[2][w]);
      total = add_sat(total, s.found[3][w]);
      empty += s.found[4][w];
    }
  }

  // the rows
  for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < p.n_rows; i += (int64_t)p.workgroups * THREADS) {
    const int row = (int)i;
    const int b = DECODE ? row : find(s_end, n, (uint32_t)row);
    int32_t pos = 0;
    int64_t slot = 0;
    if (b < n && s_before[b] >= 0) {
      const int before = s_before[b];
      pos = DECODE ? before : before + row - (int)(b ? s_end[b - 1] : 0u);
      const int at = block_at(p, pos), had = blocks_for(p, before);
      int id = s_last[b];  // a row's block is new or the one of the last token before the step
      if (at >= had) {
        const int k = (int)(b ? s_upto[b - 1] : 0u) + at - had;
        // (nontemporal, or the compiler joins the two into one flat load)
        if (DECODE && k < kAhead) id = s_free[k];
        else id = __builtin_nontemporal_load(p.free_blocks + taken + k);
        if (DECODE) p.block_table[(int64_t)b * p.table_stride + at] = id;
      }
      slot = (int64_t)id * p.block_size + (pos - at * p.block_size);
    }
    if constexpr (!DECODE) p.request_of_row[row] = b < n ? b : 0;
    p.positions[row] = pos;
    p.slot_mapping[row] = slot;
  }
  if constexpr (!DECODE) {
    // the new blocks' entries
    for (uint32_t i = blockIdx.x * THREADS + tid; i < given; i += p.workgroups * THREADS) {
      const int b = find(s_upto, n, i);
      const int had = blocks_for(p, s_before[b]);
      p.block_table[(int64_t)b * p.table_stride + had + (i - (b ? s_upto[b - 1] : 0u))] = p.free_blocks[taken + i];
    }
    __syncthreads();
    if (p.workgroups > 1) {  // the last workgroup to get here, when all have read the lengths and the state
      if (tid == 0) {
        const uint32_t before = __hip_atomic_fetch_add(reinterpret_cast<uint32_t*>(p.after + 2), 1u, __ATOMIC_ACQ_REL,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        s.last = before + 1 == (uint32_t)p.workgroups;
      }
      __syncthreads();
      if (!s.last) return;
    }
  }
  // (a decode bucket's barriers are past every read of the lengths and the pool's state)
  for (int b = lo; b < hi; ++b) {
    const int r = DECODE ? 1 : (int)(s_end[b] - (b ? s_end[b - 1] : 0u));
    p.kv_lengths[b] = s_before[b] >= 0 ? s_before[b] + r : 0;
  }
  if (tid == 0) {
    p.after[0] = taken + (int32_t)given;
    p.after[1] = (int32_t)left_out;
    p.after[2] = 0;
  }
  if constexpr (DECODE) stage_split<THREADS>(p, s_before, s_end, s, (int)longest, total, empty);
}

template <int THREADS>
void launch_decode(const TablesParams& p, hipStream_t stream) {
  const size_t words = 4 * (size_t)p.n_requests + (size_t)(p.n_requests < kAhead ? p.n_requests : kAhead);
  hipLaunchKernelGGL((step_tables_kernel<true, THREADS>), dim3(1), dim3(THREADS), words * sizeof(int32_t), stream, p);
}

}  // namespace

hipError_t launch_step_tables(const TablesParams& params, hipStream_t stream) {
  TablesParams p = params;
  p.workgroups = 1;
  if (p.staged) {  // one workgroup: the split needs every row's length
    if (p.n_requests <= 64) launch_decode<256>(p, stream);
    else if (p.n_requests <= 256) launch_decode<512>(p, stream);
    else launch_decode<1024>(p, stream);
  } else {  // a row per thread, as far as one round of the GPU goes
    const int64_t groups = ((int64_t)p.n_rows + 255) / 256;
    p.workgroups = (int32_t)(groups < 1 ? 1 : groups > 256 ? 256 : groups);
    hipLaunchKernelGGL((step_tables_kernel<false, 256>), dim3(p.workgroups), dim3(256),
                       4 * (size_t)p.n_requests * sizeof(int32_t), stream, p);
  }
  return hipGetLastError();
}

}  // namespace ayk
