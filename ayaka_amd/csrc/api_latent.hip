// The C ABI of include/ayaka_hip_latent.h: argument checks, geometry, and the launches.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "api_common.h"
#include "ayaka_hip_internal.h"
#include "ayaka_hip_latent.h"

namespace {

using ayk_api::compute_units;
using ayk_api::fail;
using ayk_api::launched;
using ayk_api::misaligned;
using ayk_api::ok;

constexpr float kLog2e = 1.4426950408889634f;

// What both rotating writes ask of the rotation, the pool and the element type.
int check_rotation(const char* op, int32_t n_rows, int32_t heads, int32_t width, int32_t pairs, const void* positions,
                   const void* turns, float magnitude, int32_t dtype) {
  if (n_rows < 0) return fail(AYK_ERR_ARGUMENT, "%s: n_rows is negative (%d)", op, n_rows);
  if (dtype != AYK_DTYPE_FP16 && dtype != AYK_DTYPE_BF16 && dtype != AYK_DTYPE_FP32)
    return fail(AYK_ERR_UNSUPPORTED, "%s: dtype %d is not fp16 (0), bf16 (1) or fp32 (3)", op, dtype);
  if (heads < 0) return fail(AYK_ERR_ARGUMENT, "%s: num_heads is negative (%d)", op, heads);
  if (width < 2 || width > ayk::kRotateMostWidth || width % 2 != 0)
    return fail(AYK_ERR_UNSUPPORTED, "%s: a width of %d is not even and in [2, %d]", op, width, ayk::kRotateMostWidth);
  if (pairs < 0 || 2 * pairs > width)
    return fail(AYK_ERR_ARGUMENT, "%s: %d pairs do not fit a width of %d", op, pairs, width);
  if (!std::isfinite(magnitude)) return fail(AYK_ERR_ARGUMENT, "%s: magnitude must be finite", op);
  if (n_rows > 0 && pairs > 0 && (!positions || !turns || misaligned(8, {turns})))
    return fail(AYK_ERR_ARGUMENT, "%s: positions or turns is null, or turns not 8-byte aligned", op);
  return AYK_OK;
}

int check_pool(const char* op, int32_t num_blocks, int32_t block_size) {
  if (block_size < 1 || block_size > 65536)
    return fail(AYK_ERR_UNSUPPORTED, "%s: block_size %d is not in [1, 65536]", op, block_size);
  if (num_blocks <= 0) return fail(AYK_ERR_ARGUMENT, "%s: num_blocks %d", op, num_blocks);
  if ((int64_t)num_blocks * block_size > INT32_MAX)
    return fail(AYK_ERR_UNSUPPORTED, "%s: %d blocks of %d positions exceed 2^31 slots", op, num_blocks, block_size);
  return AYK_OK;
}

// Elements beside each other start where their type may.
bool aligned_rows(int32_t dtype, std::initializer_list<const void*> addresses) {
  return !misaligned(dtype == AYK_DTYPE_FP32 ? 4 : 2, addresses);
}

ayk::RotateStream stream_of(const void* from, int64_t from_row, int64_t from_head, void* to, int64_t to_row,
                            int64_t to_head, int32_t heads, int32_t width, int32_t rotated) {
  ayk::RotateStream s{};
  s.from = from;
  s.to = to;
  s.from_row = from_row;
  s.from_head = from_head;
  s.to_row = to_row;
  s.to_head = to_head;
  s.heads = heads;
  s.width = width;
  s.rotated = rotated;
  return s;
}

// One launch takes up to 2^31 tasks of at least two elements.
int launch_rotation(const char* op, ayk::RotateParams& p, int32_t dtype, int32_t interleaved, void* stream) {
  int64_t elements = 0;
  for (const ayk::RotateStream& s : p.stream) elements += (int64_t)s.heads * s.width;
  if (elements / 2 * 8 > INT32_MAX)
    return fail(AYK_ERR_UNSUPPORTED, "%s: %lld elements of a row exceed one launch", op, (long long)elements);
  return launched(ayk::launch_rotate_store(p, dtype, interleaved != 0, compute_units(), static_cast<hipStream_t>(stream)),
                  op);
}

}  // namespace

extern "C" {

int ayk_rotate_and_cache(const void* q, int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row,
                         int64_t q_out_head, const void* k, int64_t k_row, int64_t k_head, void* k_out,
                         int64_t k_out_row, int64_t k_out_head, const void* v, int64_t v_row, int64_t v_head,
                         void* k_cache, void* v_cache, const int32_t* positions, const int64_t* slot_mapping,
                         const double* turns, int32_t pairs, int32_t interleaved, float magnitude, int32_t n_rows,
                         int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                         int32_t block_size, int32_t layout, int32_t dtype, void* stream) {
  const char* op = "ayk_rotate_and_cache";
  int rc = check_rotation(op, n_rows, num_heads, head_dim, pairs, positions, turns, magnitude, dtype);
  if (rc != AYK_OK) return rc;
  if (num_kv_heads < 0) return fail(AYK_ERR_ARGUMENT, "%s: num_kv_heads is negative (%d)", op, num_kv_heads);
  const bool store = k_cache != nullptr;
  if (store != (v_cache != nullptr))
    return fail(AYK_ERR_ARGUMENT, "%s: k_cache and v_cache are given together or not at all", op);
  if (store) {
    if ((rc = check_pool(op, num_blocks, block_size)) != AYK_OK) return rc;
    if (layout != AYK_LAYOUT_NHD && layout != AYK_LAYOUT_HND)
      return fail(AYK_ERR_UNSUPPORTED, "%s: layout %d is not NHD (0) or HND (1)", op, layout);
  }
  if (n_rows == 0) return ok();
  if ((num_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || (store ? !v || !slot_mapping : !k_out))))
    return fail(AYK_ERR_ARGUMENT, "%s: a required pointer is null", op);
  if (!aligned_rows(dtype, {q, q_out, k, k_out, v, k_cache, v_cache}))
    return fail(AYK_ERR_ARGUMENT, "%s: an address is not a multiple of the element's size", op);
  ayk::RotateParams p{};
  p.positions = positions;
  p.slots = slot_mapping;
  p.turns = turns;
  p.magnitude = magnitude;
  p.pairs = pairs;
  p.n_rows = n_rows;
  p.block_size = store ? block_size : 1;
  p.num_slots = store ? num_blocks * block_size : 0;
  p.by_block = ayk::divisor_of(p.block_size);
  p.stream[0] = stream_of(q, q_row, q_head, q_out, q_out_row, q_out_head, num_heads, head_dim, 2 * pairs);
  if (store) {
    const bool hnd = layout == AYK_LAYOUT_HND;
    const int64_t token = hnd ? head_dim : (int64_t)num_kv_heads * head_dim;
    const int64_t head = hnd ? (int64_t)block_size * head_dim : head_dim;
    p.stream[1] = stream_of(k, k_row, k_head, k_cache, token, head, num_kv_heads, head_dim, 2 * pairs);
    p.stream[2] = stream_of(v, v_row, v_head, v_cache, token, head, num_kv_heads, head_dim, 0);
    for (int i = 1; i < 3; ++i) {
      p.stream[i].to_block = (int64_t)block_size * num_kv_heads * head_dim;
      p.stream[i].by_slot = 1;
    }
  } else {
    p.stream[1] = stream_of(k, k_row, k_head, k_out, k_out_row, k_out_head, num_kv_heads, head_dim, 2 * pairs);
  }
  return launch_rotation(op, p, dtype, interleaved, stream);
}

int ayk_store_latent(const void* latent, int64_t latent_row, const void* k_rope, int64_t k_row, const void* q,
                     int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row, int64_t q_out_head, void* cache,
                     const int32_t* positions, const int64_t* slot_mapping, const double* turns, int32_t pairs,
                     int32_t interleaved, float magnitude, int32_t n_rows, int32_t num_heads, int32_t latent_dim,
                     int32_t rope_dim, int32_t num_blocks, int32_t block_size, int32_t dtype, void* stream) {
  const char* op = "ayk_store_latent";
  int rc = check_rotation(op, n_rows, num_heads, rope_dim, pairs, positions, turns, magnitude, dtype);
  if (rc != AYK_OK) return rc;
  if (latent_dim < 2 || latent_dim > 65536 || latent_dim % 2 != 0)
    return fail(AYK_ERR_UNSUPPORTED, "%s: latent_dim %d is not even and in [2, 65536]", op, latent_dim);
  if (pairs != 0 && 2 * pairs != rope_dim)
    return fail(AYK_ERR_ARGUMENT, "%s: %d pairs are neither 0 nor half of rope_dim %d", op, pairs, rope_dim);
  if (pairs == 0 && num_heads != 0)
    return fail(AYK_ERR_ARGUMENT, "%s: %d heads of queries and nothing to rotate them by", op, num_heads);
  if ((rc = check_pool(op, num_blocks, block_size)) != AYK_OK) return rc;
  if (n_rows == 0) return ok();
  if (!latent || !k_rope || !cache || !slot_mapping || (num_heads > 0 && (!q || !q_out)))
    return fail(AYK_ERR_ARGUMENT, "%s: a required pointer is null", op);
  if (!aligned_rows(dtype, {latent, k_rope, q, q_out, cache}))
    return fail(AYK_ERR_ARGUMENT, "%s: an address is not a multiple of the element's size", op);
  ayk::RotateParams p{};
  p.positions = positions;
  p.slots = slot_mapping;
  p.turns = turns;
  p.magnitude = magnitude;
  p.pairs = pairs;
  p.n_rows = n_rows;
  p.block_size = block_size;
  p.num_slots = num_blocks * block_size;
  p.by_block = ayk::divisor_of(block_size);
  const int64_t width = latent_dim + rope_dim;
  uint8_t* tail = static_cast<uint8_t*>(cache) + (int64_t)latent_dim * (dtype == AYK_DTYPE_FP32 ? 4 : 2);
  p.stream[0] = stream_of(q, q_row, q_head, q_out, q_out_row, q_out_head, num_heads, rope_dim, rope_dim);
  p.stream[1] = stream_of(k_rope, k_row, 0, tail, width, 0, 1, rope_dim, 2 * pairs);
  p.stream[2] = stream_of(latent, latent_row, 0, cache, width, 0, 1, latent_dim, 0);
  for (int i = 1; i < 3; ++i) {
    p.stream[i].to_block = block_size * width;
    p.stream[i].by_slot = 1;
  }
  return launch_rotation(op, p, dtype, interleaved, stream);
}

size_t ayk_latent_attention_workspace_bytes(int32_t n_rows, int32_t n_requests, int32_t num_heads, int32_t latent_dim) {
  if (n_rows < 1 || n_requests < 1 || num_heads < 1 || (latent_dim != 256 && latent_dim != 512)) return 0;
  const int units = compute_units();
  return ayk::latent_workspace_bytes(latent_dim, ayk::latent_tile_pairs(n_rows, n_requests, num_heads, units), units);
}

int ayk_latent_attention(void* out, const void* q, const void* cache, const int32_t* block_table, int64_t table_stride,
                         const int32_t* kv_lengths, const int32_t* rows, int32_t n_requests, int32_t n_rows,
                         int32_t num_heads, int32_t latent_dim, int32_t rope_dim, int32_t num_blocks,
                         int32_t block_size, int32_t max_blocks, int32_t dtype, float scale, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const int pairs = n_rows < 1 || n_requests < 1 || num_heads < 1
                        ? 16 : ayk::latent_tile_pairs(n_rows, n_requests, num_heads, compute_units());
  return ayk_latent_attention_tiles(out, q, cache, block_table, table_stride, kv_lengths, rows, n_requests, n_rows, num_heads,
                                    latent_dim, rope_dim, num_blocks, block_size, max_blocks, dtype, scale, pairs, workspace,
                                    workspace_bytes, stream);
}

int32_t ayk_latent_tile_pairs(const int32_t* rows, const int32_t* kv_lengths, int32_t n_requests, int32_t num_heads) {
  if (!rows || !kv_lengths || n_requests < 1 || num_heads < 1) return 16;
  return ayk::latent_tile_pairs(rows, kv_lengths, n_requests, num_heads, compute_units());
}

size_t ayk_latent_tiles_workspace_bytes(int32_t latent_dim, int32_t tile_pairs) {
  if ((latent_dim != 256 && latent_dim != 512) || (tile_pairs != 16 && tile_pairs != 32 && tile_pairs != 64)) return 0;
  return ayk::latent_workspace_bytes(latent_dim, tile_pairs, compute_units());
}

int ayk_latent_attention_tiles(void* out, const void* q, const void* cache, const int32_t* block_table,
                               int64_t table_stride, const int32_t* kv_lengths, const int32_t* rows,
                               int32_t n_requests, int32_t n_rows, int32_t num_heads, int32_t latent_dim,
                               int32_t rope_dim, int32_t num_blocks, int32_t block_size, int32_t max_blocks,
                               int32_t dtype, float scale, int32_t tile_pairs, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const char* op = "ayk_latent_attention";
  if (tile_pairs != 16 && tile_pairs != 32 && tile_pairs != 64)
    return fail(AYK_ERR_ARGUMENT, "%s: tile_pairs %d is not 16, 32 or 64", op, tile_pairs);
  if (n_rows < 0 || n_requests < 0)
    return fail(AYK_ERR_ARGUMENT, "%s: n_rows %d, n_requests %d", op, n_rows, n_requests);
  if (latent_dim != 256 && latent_dim != 512)
    return fail(AYK_ERR_UNSUPPORTED, "%s: latent_dim %d is not 256 or 512", op, latent_dim);
  if (rope_dim != 64) return fail(AYK_ERR_UNSUPPORTED, "%s: rope_dim %d is not 64", op, rope_dim);
  if (dtype != AYK_DTYPE_FP16 && dtype != AYK_DTYPE_BF16)
    return fail(AYK_ERR_UNSUPPORTED, "%s: dtype %d is not fp16 (0) or bf16 (1)", op, dtype);
  if (num_heads < 1) return fail(AYK_ERR_ARGUMENT, "%s: num_heads %d", op, num_heads);
  const int rc = check_pool(op, num_blocks, block_size);
  if (rc != AYK_OK) return rc;
  if (max_blocks < 0 || max_blocks >= (1 << 24) || table_stride < max_blocks)
    return fail(AYK_ERR_ARGUMENT, "%s: max_blocks %d (below 2^24), table_stride %lld", op, max_blocks,
                (long long)table_stride);
  if (n_rows == 0 || n_requests == 0) return ok();
  if (!out || !q || !cache || !block_table || !kv_lengths || !rows)
    return fail(AYK_ERR_ARGUMENT, "%s: a required pointer is null", op);
  if (misaligned(16, {out, q, cache, workspace}))
    return fail(AYK_ERR_ARGUMENT, "%s: out, q, cache and workspace must be 16-byte aligned", op);
  const size_t need = ayk_latent_tiles_workspace_bytes(latent_dim, tile_pairs);
  if (!workspace || workspace_bytes < need)
    return fail(AYK_ERR_WORKSPACE, "%s: the workspace holds %zu bytes, %zu are needed", op, workspace_bytes, need);
  // the kernel counts (row, head) pairs and the units of all tiles in 31 bits
  const int pairs = tile_pairs;
  const int64_t positions = (int64_t)max_blocks * block_size;
  const int64_t tiles = (int64_t)n_rows * num_heads / pairs + n_requests;
  if ((int64_t)n_rows * num_heads > INT32_MAX || positions > INT32_MAX - 64 ||
      tiles * ayk::latent_tile_units(pairs, positions) > INT32_MAX)
    return fail(AYK_ERR_UNSUPPORTED, "%s: %d rows of %d heads over tables of %lld positions exceed one launch", op, n_rows,
                num_heads, (long long)positions);
  ayk::LatentParams p{};
  p.out = out;
  p.q = static_cast<const uint16_t*>(q);
  p.cache = static_cast<const uint16_t*>(cache);
  p.block_table = block_table;
  p.kv_lengths = kv_lengths;
  p.rows = rows;
  p.table_stride = table_stride;
  p.n_requests = n_requests;
  p.n_rows = n_rows;
  p.heads = num_heads;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.by_block = ayk::divisor_of(block_size);
  p.max_len = (int32_t)positions;
  p.scale_log2 = scale * kLog2e;
  const int units = compute_units();
  p.places = static_cast<int32_t*>(workspace);
  p.part_ml = reinterpret_cast<float*>(p.places + 8 * units);
  p.part_o = p.part_ml + 4 * (int64_t)units * pairs;
  return launched(ayk::launch_latent_attention(p, latent_dim, dtype == AYK_DTYPE_BF16, pairs, units,
                                               static_cast<hipStream_t>(stream)),
                  op);
}

size_t ayk_latent_chunks_workspace_bytes(int64_t ws_rows, int32_t heads_at_once) {
  if (ws_rows < 0 || ws_rows % ayk::kLatentChunkTokens != 0 || ws_rows > INT32_MAX || heads_at_once < 1) return 0;
  // rotary parts, then keys, values and exponents of each head
  return (size_t)ws_rows * 128 + (size_t)heads_at_once * ((size_t)ws_rows * 512 + (size_t)ws_rows / ayk::kLatentChunkTokens * 8);
}

int ayk_latent_chunks(void* out, const void* q, const void* cache, const void* keys, const void* values,
                      const int32_t* block_table, int64_t table_stride, const int32_t* token_tiles,
                      int32_t n_token_tiles, const int32_t* row_tiles, int32_t n_row_tiles, int64_t ws_rows,
                      int32_t heads_at_once, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                      int32_t num_blocks, int32_t block_size, int32_t dtype, float scale, void* workspace,
                      size_t workspace_bytes, void* stream) {
  return ayk_latent_chunks_split(out, q, cache, keys, values, block_table, table_stride, token_tiles, n_token_tiles, row_tiles,
                                 n_row_tiles, ws_rows, heads_at_once, num_heads, latent_dim, rope_dim, num_blocks,
                                 block_size, dtype, scale, 1, workspace, workspace_bytes, stream);
}

size_t ayk_latent_chunks_parts_bytes(int32_t n_row_tiles, int32_t heads_at_once, int32_t splits) {
  if (n_row_tiles < 1 || heads_at_once < 1 || splits < 2 || splits > 64) return 0;
  return (size_t)n_row_tiles * heads_at_once * splits * ayk::kLatentChunkRows * (128 + 2) * 4;
}

int ayk_latent_chunks_split(void* out, const void* q, const void* cache, const void* keys, const void* values,
                            const int32_t* block_table, int64_t table_stride, const int32_t* token_tiles,
                            int32_t n_token_tiles, const int32_t* row_tiles, int32_t n_row_tiles, int64_t ws_rows,
                            int32_t heads_at_once, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                            int32_t num_blocks, int32_t block_size, int32_t dtype, float scale, int32_t splits,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "ayk_latent_chunks";
  if (splits < 1 || splits > 64) return fail(AYK_ERR_ARGUMENT, "%s: splits %d is not in [1, 64]", op, splits);
  if (latent_dim != 256 && latent_dim != 512)
    return fail(AYK_ERR_UNSUPPORTED, "%s: latent_dim %d is not 256 or 512", op, latent_dim);
  if (rope_dim != 64) return fail(AYK_ERR_UNSUPPORTED, "%s: rope_dim %d is not 64", op, rope_dim);
  if (dtype != AYK_DTYPE_FP16 && dtype != AYK_DTYPE_BF16)
    return fail(AYK_ERR_UNSUPPORTED, "%s: dtype %d is not fp16 (0) or bf16 (1)", op, dtype);
  if (num_heads < 1 || heads_at_once < 1)
    return fail(AYK_ERR_ARGUMENT, "%s: num_heads %d, heads_at_once %d", op, num_heads, heads_at_once);
  const int rc = check_pool(op, num_blocks, block_size);
  if (rc != AYK_OK) return rc;
  if (n_token_tiles < 0 || n_row_tiles < 0 || ws_rows < 0 || ws_rows % ayk::kLatentChunkTokens != 0 || ws_rows > INT32_MAX)
    return fail(AYK_ERR_ARGUMENT, "%s: %d token tiles, %d row tiles, ws_rows %lld (a multiple of 128)", op, n_token_tiles,
                n_row_tiles, (long long)ws_rows);
  if (n_row_tiles == 0) return ok();
  if (!out || !q || !cache || !keys || !values || !block_table || !row_tiles || (n_token_tiles > 0 && !token_tiles))
    return fail(AYK_ERR_ARGUMENT, "%s: a required pointer is null", op);
  if (misaligned(16, {out, q, cache, keys, values, workspace}))
    return fail(AYK_ERR_ARGUMENT, "%s: out, q, cache, keys, values and workspace must be 16-byte aligned", op);
  if (heads_at_once > num_heads) heads_at_once = num_heads;
  size_t expanded = ayk_latent_chunks_workspace_bytes(ws_rows, heads_at_once);
  if (splits > 1) expanded = (expanded + 15) & ~(size_t)15;  // (where the parts follow)
  const size_t need = expanded + ayk_latent_chunks_parts_bytes(n_row_tiles, heads_at_once, splits);
  if (need > workspace_bytes || (need > 0 && !workspace))
    return fail(AYK_ERR_WORKSPACE, "%s: the workspace holds %zu bytes, %zu are needed", op, workspace_bytes, need);
  const int64_t cut_tiles = (int64_t)n_row_tiles * splits;
  if ((n_token_tiles > cut_tiles ? n_token_tiles : cut_tiles) * heads_at_once > INT32_MAX)
    return fail(AYK_ERR_UNSUPPORTED, "%s: %d and %d tiles of %d heads exceed one launch", op, n_token_tiles, n_row_tiles,
                heads_at_once);
  ayk::LatentChunkParams p{};
  p.out = out;
  p.q = static_cast<const uint16_t*>(q);
  p.cache = static_cast<const uint16_t*>(cache);
  p.keys = static_cast<const uint16_t*>(keys);
  p.values = static_cast<const uint16_t*>(values);
  p.block_table = block_table;
  p.token_tiles = token_tiles;
  p.row_tiles = row_tiles;
  p.table_stride = table_stride;
  p.ws_rows = ws_rows;
  p.n_token_tiles = n_token_tiles;
  p.n_row_tiles = n_row_tiles;
  p.heads = num_heads;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.by_block = ayk::divisor_of(block_size);
  p.scale_log2 = scale * kLog2e;
  p.group_heads = heads_at_once;
  p.splits = splits;
  p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + expanded);
  p.part_ml = p.part_o + cut_tiles * heads_at_once * ayk::kLatentChunkRows * 128;
  p.ws_rope = static_cast<uint16_t*>(workspace);
  p.ws_keys = p.ws_rope + ws_rows * 64;
  p.ws_values = p.ws_keys + heads_at_once * ws_rows * 128;
  p.ws_exponents = reinterpret_cast<int32_t*>(p.ws_values + heads_at_once * ws_rows * 128);
  return launched(ayk::launch_latent_chunks(p, latent_dim, dtype == AYK_DTYPE_BF16, static_cast<hipStream_t>(stream)), op);
}

}  // extern "C"
