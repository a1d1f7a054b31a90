// Step tables built on the GPU (gfx950): blocks for the requests that lack them, every row's
// request, position and slot, and a decode bucket's v2 split (see ayaka_hip_tables.h).
//
// Two sums over the requests say everything: the rows before a request, and the new blocks handed
// out before it. A workgroup makes both in LDS -- a few thousand requests at most, so each makes
// them for itself rather than waiting for another to -- and then every row, and every new block,
// finds its request by bisection and computes its own numbers, independent of all the others. What
// bounds it is latency: a handful of dependent loads, two scans, one bisection. Steps of many rows
// spread over workgroups of kRowsPerGroup rows; the last of them to finish (by a counter) writes
// the words that the others read, so the pool's state and the lengths may be updated in place.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "ayaka_hip_internal.h"
#include "kv_address.h"

namespace ayk {

namespace {

constexpr int kBins = 256;

// The workgroup's waves' shares of a sum: inclusive scans and totals over all its threads.
struct Scratch {
  int64_t wave_sum[16];
  int64_t total;
  int32_t wave_max[16];
  int32_t flag;
};

// Sum of `x` over the threads before this one; `total` over all of them. Ends on a barrier.
__device__ __forceinline__ int64_t scan_exclusive(int64_t x, Scratch& s, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int64_t sum = x;
#pragma unroll
  for (int st = 1; st < 64; st <<= 1) {
    const int64_t other = __shfl_up(sum, st);
    if (lane >= st) sum += other;
  }
  if (lane == 63) s.wave_sum[wave] = sum;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    const int64_t v = s.wave_sum[w];
    before += w < wave ? v : 0;
    all += v;
  }
  __syncthreads();  // the next scan writes wave_sum
  total = all;
  return before + sum - x;
}

__device__ __forceinline__ int32_t reduce_max(int32_t x, Scratch& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int st = 1; st < 64; st <<= 1) x = max(x, __shfl_xor(x, st));
  if (lane == 0) s.wave_max[wave] = x;
  __syncthreads();
  for (int w = 0; w < waves; ++w) x = max(x, s.wave_max[w]);
  __syncthreads();
  return x;
}

__device__ __forceinline__ int32_t clamp32(int64_t x) { return x > INT32_MAX ? INT32_MAX : (int32_t)x; }

// The first request whose running sum passes i, or n.
__device__ __forceinline__ int find(const int32_t* sums, int n, int32_t i) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int block_at(const TablesParams& p, int t) {
  return (int)((__umulhi((uint32_t)t, p.bs_magic) + (uint32_t)t) >> p.bs_shift);
}
__device__ __forceinline__ int blocks_for(const TablesParams& p, int tokens) {
  return tokens > 0 ? block_at(p, tokens - 1) + 1 : 0;
}

// The v2 split of the rows' lengths (s_len) into p.staged. s_end is free to use.
__device__ void stage_split(const TablesParams& p, const int32_t* s_len, int32_t* s_end, Scratch& s) {
  __shared__ float s_time[AYK_TABLES_SIZES];
  __shared__ int32_t s_bins[kBins];
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
  const int n = p.n_requests, per = (n + threads - 1) / threads;
  const int lo = min(tid * per, n), hi = min(n, lo + per);
  int32_t longest = 0;
  for (int b = lo; b < hi; ++b) longest = max(longest, s_len[b]);
  longest = reduce_max(longest, s);

  // A size's time, in positions: its work spread over the compute units plus 0.3 of its longest
  // item (what the last to finish trails by); a launch of one round takes its longest item. Over
  // 600 drawn batches this picks sizes 2.6% behind the scheduled model's on average.
  for (int c = wave; c < p.n_sizes; c += waves) {
    const int size = p.sizes[c];
    int64_t items = 0, list = 0, total = 0;
    for (int b = lane; b < n; b += 64) {
      const int len = s_len[b];
      const int parts = len > 0 ? (int)((uint32_t)(len - 1) / (uint32_t)size) + 1 : 0;
      items += parts;
      list += max(parts, 1);
      total += len;
    }
#pragma unroll
    for (int st = 1; st < 64; st <<= 1) {
      items += __shfl_xor(items, st);
      list += __shfl_xor(list, st);
      total += __shfl_xor(total, st);
    }
    if (lane == 0) {
      const float item = (float)(min(size, longest) + p.cost);
      const float groups = (float)p.groups, units = (float)p.compute_units;
      float time = ((float)total + (float)p.cost * (float)items) * groups / units + 0.3f * item;
      if (items * p.groups <= p.compute_units) time = item;
      const bool offered = c == 0 || p.sizes[c - 1] < longest;
      const bool long_list = items * p.groups > 8 * (int64_t)p.compute_units;  // start-up costs dominate
      s_time[c] = !offered || list > p.capacity ? INFINITY : long_list ? 1e30f * (1.0f + (float)(AYK_TABLES_SIZES - c))
                                                                       : time;
    }
  }
  __syncthreads();
  int size = max(p.sizes[0], (int)(((int64_t)longest + 63) / 64 * 64));  // one partition per row
  float best = INFINITY;
  for (int c = 0; c < p.n_sizes; ++c) {
    if (s_time[c] < best) {
      best = s_time[c];
      size = p.sizes[c];
    }
  }

  // full partitions, partial ones and rows without context before each row, in one sum
  int64_t mine = 0;
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)s_len[b], full = len / (uint32_t)size, rest = len % (uint32_t)size;
    mine += ((int64_t)full << 32) | ((int64_t)(rest != 0) << 16) | (int64_t)(len == 0);
  }
  int64_t all;
  int64_t at = scan_exclusive(mine, s, all);
  for (int i = tid; i < kBins; i += threads) s_bins[i] = 0;
  __syncthreads();
  auto bin_of = [&](uint32_t rest) { return kBins - 1 - (int)(((int64_t)(rest - 1) * kBins) / size); };
  int32_t* work = p.staged + 2 + n;
  const int fulls = (int)(all >> 32), parts = (int)((all >> 16) & 0xffff), empties = (int)(all & 0xffff);
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)s_len[b], full = len / (uint32_t)size, rest = len % (uint32_t)size;
    p.staged[2 + b] = (int)(at >> 32) + (int)((at >> 16) & 0xffff);
    if (rest) atomicAdd(&s_bins[bin_of(rest)], 1);
    if (len == 0) {  // partition 0 writes the row's zeros; last
      const int i = fulls + parts + (int)(at & 0xffff);
      work[2 * i] = b;
      work[2 * i + 1] = 0;
    }
    at += ((int64_t)full << 32) | ((int64_t)(rest != 0) << 16) | (int64_t)(len == 0);
    s_end[b] = (int32_t)(at >> 32);
  }
  __syncthreads();
  if (wave == 0) {  // the bins' first places: four bins per lane
    int32_t c[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = s_bins[4 * lane + k];
      sum += c[k];
    }
    int32_t upto = sum;
#pragma unroll
    for (int st = 1; st < 64; st <<= 1) {
      const int32_t other = __shfl_up(upto, st);
      if (lane >= st) upto += other;
    }
    int32_t first = fulls + upto - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_bins[4 * lane + k] = first;
      first += c[k];
    }
  }
  __syncthreads();
  // the order within a bin is the threads' (it decides when an item runs, not what it computes)
  for (int b = lo; b < hi; ++b) {
    const uint32_t len = (uint32_t)s_len[b], rest = len % (uint32_t)size;
    if (rest == 0) continue;
    const int i = atomicAdd(&s_bins[bin_of(rest)], 1);
    work[2 * i] = b;
    work[2 * i + 1] = (int32_t)(len / (uint32_t)size);
  }
  for (int i = tid; i < fulls; i += threads) {
    const int b = find(s_end, n, i);
    work[2 * i] = b;
    work[2 * i + 1] = i - (b ? s_end[b - 1] : 0);
  }
  if (tid == 0) {
    p.staged[0] = size;
    p.staged[1] = fulls + parts + empties;
  }
}

// DECODE: one row per request, and the v2 split after it (one workgroup).
template <bool DECODE>
__global__ __launch_bounds__(1024) void step_tables_kernel(const TablesParams p) {
  extern __shared__ int32_t smem[];
  __shared__ Scratch s;
  const int n = p.n_requests;
  int32_t* s_end = smem;           // rows of the requests up to and with each
  int32_t* s_upto = smem + n;      // new blocks, the same (as if all could be served)
  int32_t* s_len = smem + 2 * n;   // lengths of the requests served, 0 of the others
  const int tid = threadIdx.x, threads = blockDim.x;
  const int per = (n + threads - 1) / threads;
  const int lo = min(tid * per, n), hi = min(n, lo + per);
  auto rows_of = [&](int b) { return DECODE ? 1 : p.rows[b]; };

  const int taken = min(max(*p.taken, 0), p.n_free);
  const int room = p.n_free - taken;
  int64_t sum = 0, total = 0;
  if constexpr (!DECODE) {
    for (int b = lo; b < hi; ++b) sum += max(p.rows[b], 0);
    sum = scan_exclusive(sum, s, total);
  } else {
    sum = lo;
  }
  const int64_t limit = (int64_t)p.max_blocks * p.block_size;
  int64_t need = 0;
  for (int b = lo; b < hi; ++b) {
    const int r = rows_of(b), len = p.lengths[b];
    sum += max(r, 0);
    bool live = r >= 0 && len > 0 && r <= len && len <= limit && sum <= p.n_rows;
    const int had = live ? blocks_for(p, len - r) : 0;
    // the padding block where the last token before the step lies: a block it was never given
    if (had > 0 && p.block_table[(int64_t)b * p.table_stride + had - 1] == 0) live = false;
    const int want = live ? blocks_for(p, len) - had : 0;
    need += want;
    s_end[b] = clamp32(sum);
    s_upto[b] = want;             // made a running sum below
    s_len[b] = live ? len : 0;
  }
  need = scan_exclusive(need, s, total);
  int32_t given = 0;
  int64_t left_out = 0;
  for (int b = lo; b < hi; ++b) {
    const int want = s_upto[b];
    need += want;
    const bool served = s_len[b] > 0 && (want == 0 || need <= room);
    if (served && want > 0) given = (int32_t)need;
    if (!served) {
      left_out += p.lengths[b] != 0;
      s_len[b] = 0;
    }
    s_upto[b] = clamp32(need);
  }
  given = reduce_max(given, s);
  int64_t short_of = 0;
  scan_exclusive(left_out, s, short_of);  // its barriers also publish the three arrays

  // the rows
  for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < p.n_rows; i += (int64_t)gridDim.x * threads) {
    const int row = (int)i;
    const int b = DECODE ? row : find(s_end, n, row);
    int32_t pos = 0;
    int64_t slot = 0;
    if (b < n && s_len[b] > 0) {
      const int r = rows_of(b), before = s_len[b] - r;
      pos = before + row - (s_end[b] - r);
      const int at = block_at(p, pos), had = blocks_for(p, before);
      const int id = at < had ? p.block_table[(int64_t)b * p.table_stride + at]
                              : p.free_blocks[taken + (b ? s_upto[b - 1] : 0) + at - had];
      slot = (int64_t)id * p.block_size + (pos - at * p.block_size);
    }
    if (p.request_of_row) p.request_of_row[row] = b < n ? b : 0;
    p.positions[row] = pos;
    p.slot_mapping[row] = slot;
  }
  // the new blocks
  for (int i = blockIdx.x * threads + tid; i < given; i += gridDim.x * threads) {
    const int b = find(s_upto, n, i);
    const int had = blocks_for(p, s_len[b] - rows_of(b));
    p.block_table[(int64_t)b * p.table_stride + had + i - (b ? s_upto[b - 1] : 0)] = p.free_blocks[taken + i];
  }
  if constexpr (DECODE) {
    stage_split(p, s_len, s_end, s);
    __syncthreads();  // every thread has read the lengths and the pool's state
  } else {
    __syncthreads();
    if (gridDim.x > 1) {  // the last workgroup to get here, when all have read the lengths and the state
      if (tid == 0) {
        const uint32_t before = __hip_atomic_fetch_add(reinterpret_cast<uint32_t*>(p.after + 2), 1u, __ATOMIC_ACQ_REL,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        s.flag = before + 1 == gridDim.x;
      }
      __syncthreads();
      if (!s.flag) return;
    }
  }
  for (int b = lo; b < hi; ++b) p.kv_lengths[b] = s_len[b];
  if (tid == 0) {
    p.after[0] = taken + given;
    p.after[1] = (int32_t)short_of;
    p.after[2] = 0;
  }
}

}  // namespace

hipError_t launch_step_tables(const TablesParams& p, hipStream_t stream) {
  // A decode bucket is one workgroup (its split needs every row's length); a row per thread up to
  // 1024. Other steps take a row per thread of 256-thread workgroups, as far as one round of the
  // GPU goes.
  const size_t lds = 3 * sizeof(int32_t) * (size_t)p.n_requests;
  if (p.staged) {
    const int threads = p.n_requests <= 256 ? 256 : p.n_requests <= 512 ? 512 : 1024;
    hipLaunchKernelGGL(step_tables_kernel<true>, dim3(1), dim3(threads), lds, stream, p);
  } else {
    const int64_t groups = ((int64_t)p.n_rows + 255) / 256;
    const unsigned grid = (unsigned)(groups < 1 ? 1 : groups > 256 ? 256 : groups);
    hipLaunchKernelGGL(step_tables_kernel<false>, dim3(grid), dim3(256), lds, stream, p);
  }
  return hipGetLastError();
}

}  // namespace ayk
