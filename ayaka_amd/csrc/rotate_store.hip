// Rotary positions and the cache write behind them, in one launch (gfx950).
//
// A pair (x, y) of a head's elements at position t becomes
//   (x cos a - y sin a, y cos a + x sin a) * magnitude,   a = t * frequency(pair),
// computed in fp32 and rounded once to the element type. Pairs are elements i and i + r/2 of the
// first r elements of a head, or 2i and 2i + 1; the elements behind r pass through.
//
// Up to three streams of rows share the launch (queries, keys, values; of a latent cache the queries'
// rotary parts, the key's rotary part and the latent). Each reads rows at strides of its own, so the
// parts of one projection's output need no copies, and writes rows at strides or cache slots. Rows
// whose slot lies in the padding block or outside the pool are not stored.
//
// Angles are kept in turns, and in 64 bits: turns(t, pair) = t * turns_per_position(pair), of which
// only the fraction matters, so a position of 2^24 loses nothing (in fp32 its angle would be off by
// whole radians) and no table of cosines bounds the positions or is read. That costs one 64-bit
// multiply and one polynomial per (row, pair), shared through LDS by all heads of the row.
//
// Bound: bytes, each element is read and written once; a launch of a few rows is the chain position,
// angle, barrier, store. A lane moves two 16-byte vectors where alignment allows (the two halves of
// its pairs), requested before the angles are made. Measured: 188 MB of a prefill step of 32 + 8 + 8 heads
// of 128 in 31 us where they are in the last cache (6.1 TB/s), 43 us (4.4 TB/s) where they are not; 141 MB
// of 128 heads' rotary parts and their latents, a third of each row of the queries read, 37 us (3.8 TB/s);
// one row of each of 256 requests 5 us (48 heads) and 3 us (a latent cache, 16), of 4 requests 3 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ayaka_hip_internal.h"

namespace ayk {
namespace {

constexpr int kThreads = 256;
// (row, pair) cosines and sines of one workgroup
constexpr int kMostAngles = 2048;
static_assert(kMostAngles >= kRotateMostWidth / 2, "one row's pairs");

// n / d for 0 <= n < 2^31 (as block_of in attention_common.h).
__device__ __forceinline__ uint32_t quotient(uint32_t n, Divisor d) {
  return (uint32_t)(((uint64_t)__umulhi(n, d.magic) + n) >> d.shift);
}

// {cos, sin} of `turns` full turns. The remainder of a quarter turn, at most pi/4 either way, goes
// through the series of sine and cosine, cut where the next term is below 2^-25.
__device__ __forceinline__ float2 cos_sin_of_turns(double turns) {
  const double quarters = 4.0 * (turns - __builtin_rint(turns));
  const double k = __builtin_rint(quarters);
  const float r = (float)((quarters - k) * 1.5707963267948966);
  const float s = r * r;
  const float sine = __builtin_fmaf(
      r * s, __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f),
      r);
  const float cosine = __builtin_fmaf(
      s, __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f),
                                          1.f / 24.f),
                        -0.5f),
      1.f);
  const int q = (int)k & 3;
  const float a = (q & 1) ? sine : cosine, b = (q & 1) ? cosine : sine;
  return make_float2(q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b);
}

// Element types: 0 fp16, 1 bf16, 3 fp32 (the C ABI's codes).
template <int TYPE>
struct Element;
template <>
struct Element<0> {
  typedef uint16_t T;
  static __device__ __forceinline__ float wide(T x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ T round(float f) { return __builtin_bit_cast(T, (_Float16)f); }
};
template <>
struct Element<1> {
  typedef uint16_t T;
  static __device__ __forceinline__ float wide(T x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ T round(float f) { return __builtin_bit_cast(T, (__bf16)f); }
};
template <>
struct Element<3> {
  typedef float T;
  static __device__ __forceinline__ float wide(T x) { return x; }
  static __device__ __forceinline__ T round(float f) { return f; }
};

template <int BYTES>
struct Words;
template <>
struct Words<16> { typedef uint32_t T __attribute__((ext_vector_type(4))); };
template <>
struct Words<8> { typedef uint32_t T __attribute__((ext_vector_type(2))); };
template <>
struct Words<4> { typedef uint32_t T; };
template <>
struct Words<2> { typedef uint16_t T; };

// V elements per vector; a task is two vectors of one head: the two halves of V pairs, V pairs side
// by side, or 2V elements that pass through.
template <int TYPE, int V, bool SIDE_BY_SIDE>
__global__ __launch_bounds__(kThreads) void rotate_store_kernel(const RotateParams p) {
  typedef typename Element<TYPE>::T T;
  typedef typename Words<V * sizeof(T)>::T W;
  __shared__ float2 s_turn[kMostAngles];
  const int tid = threadIdx.x;
  const int first = blockIdx.x * p.rows_per_workgroup;
  const int rows = min(p.rows_per_workgroup, p.n_rows - first);
  const uint32_t tasks = (uint32_t)rows * p.tasks_per_row;
  // this workgroup's share of the tasks
  uint32_t task = blockIdx.y * kThreads + tid;
  const uint32_t step = gridDim.y * kThreads;

  struct Task {
    const T* from[2];
    T* to[2];
    int pair;  // of the row's s_turn entries; -1: pass through
    bool stored;
  };
  auto find = [&](uint32_t i) {
    Task t;
    const uint32_t local = quotient(i, p.by_tasks);
    uint32_t rest = i - local * p.tasks_per_row;
    const int64_t row = first + (int)local;
    const int which = (rest >= (uint32_t)p.begin[1]) + (rest >= (uint32_t)p.begin[2]);
    const RotateStream& s = p.stream[which];
    rest -= p.begin[which];
    const uint32_t head = quotient(rest, s.by_tasks);
    const int j = (int)(rest - head * s.tasks_per_head);
    const int turned = s.rotated / (2 * V);  // tasks of a head that rotate
    int lo = j * 2 * V, hi = lo + V;
    t.pair = -1;
    if (j < turned) {
      t.pair = (int)local * p.pairs + j * V;
      if (!SIDE_BY_SIDE) lo = j * V, hi = lo + s.rotated / 2;
    }
    const T* from = static_cast<const T*>(s.from) + row * s.from_row + head * s.from_head;
    int64_t at = row * s.to_row;
    t.stored = true;
    if (s.by_slot) {
      const int64_t slot = p.slots[row];
      t.stored = slot >= p.block_size && slot < p.num_slots;
      const uint32_t kept = t.stored ? (uint32_t)slot : 0u;
      const uint32_t block = quotient(kept, p.by_block);
      at = block * s.to_block + (int64_t)(kept - block * (uint32_t)p.block_size) * s.to_row;
    }
    T* to = static_cast<T*>(s.to) + at + head * s.to_head;
    t.from[0] = from + lo;
    t.from[1] = from + hi;
    t.to[0] = to + lo;
    t.to[1] = to + hi;
    return t;
  };
  auto finish = [&](const Task& t, W a, W b) {
    T x[2 * V];
    __builtin_memcpy(x, &a, sizeof(W));
    __builtin_memcpy(x + V, &b, sizeof(W));
    if (t.pair >= 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = SIDE_BY_SIDE ? 2 * e : e, j = SIDE_BY_SIDE ? 2 * e + 1 : e + V;
        const float2 turn = s_turn[t.pair + e];
        const float u = Element<TYPE>::wide(x[i]), v = Element<TYPE>::wide(x[j]);
        x[i] = Element<TYPE>::round(__builtin_fmaf(u, turn.x, -(v * turn.y)));
        x[j] = Element<TYPE>::round(__builtin_fmaf(v, turn.x, u * turn.y));
      }
      __builtin_memcpy(&a, x, sizeof(W));
      __builtin_memcpy(&b, x + V, sizeof(W));
    }
    if (t.stored) {
      *reinterpret_cast<W*>(t.to[0]) = a;
      *reinterpret_cast<W*>(t.to[1]) = b;
    }
  };

  // the first task's elements travel while the angles are made
  Task t;
  W a{}, b{};
  const bool some = task < tasks;
  if (some) {
    t = find(task);
    a = *reinterpret_cast<const W*>(t.from[0]);
    b = *reinterpret_cast<const W*>(t.from[1]);
  }
  for (int i = tid; i < rows * p.pairs; i += kThreads) {
    const int local = i / p.pairs;
    float2 turn = cos_sin_of_turns((double)p.positions[first + local] * p.turns[i - local * p.pairs]);
    turn.x *= p.magnitude;
    turn.y *= p.magnitude;
    s_turn[i] = turn;
  }
  __syncthreads();
  if (some) finish(t, a, b);
  for (task += step; task < tasks; task += step) {
    t = find(task);
    a = *reinterpret_cast<const W*>(t.from[0]);
    b = *reinterpret_cast<const W*>(t.from[1]);
    finish(t, a, b);
  }
}

template <int TYPE, int V>
hipError_t launch_vector(const RotateParams& p, dim3 grid, bool side_by_side, hipStream_t stream) {
  if (side_by_side)
    hipLaunchKernelGGL((rotate_store_kernel<TYPE, V, true>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((rotate_store_kernel<TYPE, V, false>), grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

// Elements per vector that every address, stride and half of the streams is a multiple of.
static int vector_elements(const RotateParams& p, int size, bool side_by_side) {
  uint64_t in_elements = 0, addresses = 0;
  for (const RotateStream& s : p.stream) {
    if (s.heads == 0) continue;
    in_elements |= (uint64_t)(s.from_row | s.to_row | s.to_block);
    if (s.heads > 1) in_elements |= (uint64_t)(s.from_head | s.to_head);
    in_elements |= (uint64_t)(s.rotated / 2) | (uint64_t)((s.width - s.rotated) / 2);
    addresses |= reinterpret_cast<uintptr_t>(s.from) | reinterpret_cast<uintptr_t>(s.to);
  }
  int v = 16 / size;
  while (v > 1 && (in_elements % v != 0 || addresses % (uint64_t)(v * size) != 0)) v /= 2;
  return v;
}

hipError_t launch_rotate_store(RotateParams p, int type, bool side_by_side, int compute_units, hipStream_t stream) {
  if (p.n_rows == 0) return hipSuccess;
  const int v = vector_elements(p, type == 3 ? 4 : 2, side_by_side);
  int32_t tasks = 0;
  for (int i = 0; i < 3; ++i) {
    RotateStream& s = p.stream[i];
    p.begin[i] = tasks;
    s.tasks_per_head = s.width / (2 * v);
    s.by_tasks = divisor_of(std::max(1, s.tasks_per_head));
    tasks += s.heads * s.tasks_per_head;
  }
  p.tasks_per_row = tasks;
  if (tasks == 0) return hipSuccess;
  p.by_tasks = divisor_of(tasks);
  // Rows per workgroup and workgroups per row: rows share a workgroup (up to 2 tasks a lane; with 4 the prefill step above took 44 us, with 2 43) once
  // there are two workgroups for every compute unit, and a row of many heads is dealt to several
  // while there are fewer.
  const int wanted = 2 * compute_units;
  int rows = std::min({std::max(1, p.n_rows / wanted), std::max(1, 2 * kThreads / tasks), kMostAngles / std::max(1, p.pairs)});
  rows = std::max(1, rows);
  const int groups = (p.n_rows + rows - 1) / rows;
  const int split = std::max(1, std::min((rows * tasks + kThreads - 1) / kThreads, wanted / groups));
  p.rows_per_workgroup = rows;
  const dim3 grid((unsigned)groups, (unsigned)split);
#define AYK_ROTATE(TYPE, V) return launch_vector<TYPE, V>(p, grid, side_by_side, stream)
  if (type == 3) {
    if (v == 4) AYK_ROTATE(3, 4);
    if (v == 2) AYK_ROTATE(3, 2);
    AYK_ROTATE(3, 1);
  }
  if (type == 1) {
    if (v == 8) AYK_ROTATE(1, 8);
    if (v == 4) AYK_ROTATE(1, 4);
    if (v == 2) AYK_ROTATE(1, 2);
    AYK_ROTATE(1, 1);
  }
  if (v == 8) AYK_ROTATE(0, 8);
  if (v == 4) AYK_ROTATE(0, 4);
  if (v == 2) AYK_ROTATE(0, 2);
  AYK_ROTATE(0, 1);
#undef AYK_ROTATE
}

}  // namespace ayk
