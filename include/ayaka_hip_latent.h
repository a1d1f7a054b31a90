/*
 * ayaka_hip_latent.h -- C ABI of rotary positions joined to the cache write, and of caches of latent
 * vectors with the attention that reads them.
 *
 * Conventions and error codes are those of ayaka_hip.h: device pointers unless said otherwise, nothing
 * allocated or synchronised, work queued on `stream`. Element types are AYK_DTYPE_*; strides are in
 * elements, and an element of a head is next to the one before it.
 *
 * A latent cache is one contiguous tensor [num_blocks, block_size, latent_dim + rope_dim]: each slot
 * holds a token's latent vector and behind it the token's rotated key part, shared by all heads. Slots,
 * blocks and tables are those of ayaka_hip.h (block 0 is the padding block).
 *
 * Rotation. Pair i of a row at position t turns by t * turns[i] full turns (turns: float64, on the
 * device, one per pair; a frequency in radians per position over 2 pi): (x, y) becomes
 * (x cos - y sin, y cos + x sin) * magnitude, computed in fp32 with the angle reduced in 64 bits, and
 * rounded once. Of the first r = 2 * pairs elements of a head pair i is (i, i + r / 2), or (2i, 2i + 1)
 * where `interleaved` is not 0; elements behind them are copied.
 */
#ifndef AYAKA_HIP_LATENT_H
#define AYAKA_HIP_LATENT_H

#include "ayaka_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rotate a step's queries and keys and write keys and values into a cache.
 *   q [n_rows, num_heads, head_dim] at strides (q_row, q_head) -> q_out at (q_out_row, q_out_head); q_out
 *     may be q at the same strides, and overlaps nothing else. num_heads 0: no queries.
 *   k, v [n_rows, num_kv_heads, head_dim] at strides (k_row, k_head), (v_row, v_head).
 * With caches (k_cache and v_cache of `layout`, as ayk_reshape_and_cache) row i of the rotated keys and of
 * the values goes to slot slot_mapping[i]; rows whose slot is in the padding block or outside the pool
 * are not stored. Without (k_cache NULL): the rotated keys go to k_out at strides (k_out_row, k_out_head)
 * (k_out may be k, as q_out), values, slots, layout and block sizes are not looked at.
 * dtype: fp16, bf16 or fp32, of everything. 2 * pairs <= head_dim, head_dim even and at most 1024.
 * num_blocks * block_size < 2^31.
 */
int ayk_rotate_and_cache(const void* q, int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row,
                         int64_t q_out_head, const void* k, int64_t k_row, int64_t k_head, void* k_out,
                         int64_t k_out_row, int64_t k_out_head, const void* v, int64_t v_row, int64_t v_head,
                         void* k_cache, void* v_cache, const int32_t* positions, const int64_t* slot_mapping,
                         const double* turns, int32_t pairs, int32_t interleaved, float magnitude, int32_t n_rows,
                         int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                         int32_t block_size, int32_t layout, int32_t dtype, void* stream);

/*
 * Write a step's latents and rotated key parts into a latent cache, and rotate the queries' rotary parts.
 *   latent [n_rows, latent_dim] at stride latent_row; k_rope [n_rows, rope_dim] at stride k_row
 *   q [n_rows, num_heads, rope_dim] at (q_row, q_head) -> q_out at (q_out_row, q_out_head), which may be q at
 *     the same strides. num_heads 0: no queries.
 * pairs is rope_dim / 2, or 0: nothing is rotated (positions and turns are not looked at, num_heads must be
 * 0). Rows whose slot is in the padding block or outside the pool are not stored. dtype: fp16, bf16 or
 * fp32. latent_dim and rope_dim even, rope_dim at most 1024; num_blocks * block_size < 2^31.
 */
int ayk_store_latent(const void* latent, int64_t latent_row, const void* k_rope, int64_t k_row, const void* q,
                     int64_t q_row, int64_t q_head, void* q_out, int64_t q_out_row, int64_t q_out_head, void* cache,
                     const int32_t* positions, const int64_t* slot_mapping, const double* turns, int32_t pairs,
                     int32_t interleaved, float magnitude, int32_t n_rows, int32_t num_heads, int32_t latent_dim,
                     int32_t rope_dim, int32_t num_blocks, int32_t block_size, int32_t dtype, void* stream);

/*
 * Attention over a latent cache on its rows as they are (absorbed form):
 *   score(row, head, t) = scale * q[row, head] . cache_row(t)
 *   out[row, head]      = sum over t of softmax(score)(t) * latent(t)
 * q [n_rows, num_heads, latent_dim + 64], out [n_rows, num_heads, latent_dim], contiguous and 16-byte
 * aligned, as the cache; dtype fp16 (weights in fp16: within 2^-11 of themselves or 2^-32 of a row's largest) or bf16
 * (16 bits of a weight or more); latent_dim 256 or 512, rope_dim 64. The step has n_requests
 * requests of rows[b] rows each, in order (n_rows in all), which are the last of kv_lengths[b] tokens; a
 * row attends to the positions up to its own; requests of length 0 give zeros. rows, kv_lengths and the
 * table are read on the device only: the call can be captured and replayed with others. Rows past the sum
 * of rows[] are not written. out overlaps no input.
 * workspace: ayk_latent_attention_workspace_bytes, 16-byte aligned, the call's own while it runs.
 */
size_t ayk_latent_attention_workspace_bytes(int32_t n_rows, int32_t n_requests, int32_t num_heads, int32_t latent_dim);
int ayk_latent_attention(void* out, const void* q, const void* cache, const int32_t* block_table, int64_t table_stride,
                         const int32_t* kv_lengths, const int32_t* rows, int32_t n_requests, int32_t n_rows,
                         int32_t num_heads, int32_t latent_dim, int32_t rope_dim, int32_t num_blocks,
                         int32_t block_size, int32_t max_blocks, int32_t dtype, float scale, void* workspace,
                         size_t workspace_bytes, void* stream);

/*
 * The same with tiles of tile_pairs (row, head) pairs, 16, 32 or 64, which read a context together.
 * ayk_latent_attention takes what is best for contexts of 2048 positions; where a caller knows a step's lengths,
 * ayk_latent_tile_pairs says what is best for them (rows and kv_lengths in host memory).
 */
int32_t ayk_latent_tile_pairs(const int32_t* rows, const int32_t* kv_lengths, int32_t n_requests, int32_t num_heads);
size_t ayk_latent_tiles_workspace_bytes(int32_t latent_dim, int32_t tile_pairs);
int ayk_latent_attention_tiles(void* out, const void* q, const void* cache, const int32_t* block_table,
                               int64_t table_stride, const int32_t* kv_lengths, const int32_t* rows,
                               int32_t n_requests, int32_t n_rows, int32_t num_heads, int32_t latent_dim,
                               int32_t rope_dim, int32_t num_blocks, int32_t block_size, int32_t max_blocks,
                               int32_t dtype, float scale, int32_t tile_pairs, void* workspace,
                               size_t workspace_bytes, void* stream);

/*
 * The same cache with keys and values expanded from the latents, for chunks of many rows:
 *   key(h, t) = [keys[h] . latent(t) | rotary part(t)],  value(h, t) = values[h] . latent(t)
 *   out[row, h] = sum over t of softmax(scale * q[row, h] . key(h, .))(t) * value(h, t)
 * q [n_rows, num_heads, 128 + 64], out [n_rows, num_heads, 128], keys and values [num_heads, 128,
 * latent_dim], contiguous and 16-byte aligned, as the cache; dtype fp16 or bf16; latent_dim 256 or 512.
 * Expanded keys and values are fp16 under a power of two for every 128 tokens, head and kind (within 2^-11
 * of themselves down to 2^-27 of the largest there, then within 2^-38 of it). Weights are fp16 too, within 2^-11 of
 * themselves or, values' powers of two included, 2^-32 of a row's largest.
 * The step comes as two device lists of int32 quadruples, made on the host:
 *   token_tiles (request, first position, the request's length, workspace row): every 128 positions of each
 *     request with rows, its workspace rows following each other and starting at a multiple of 128;
 *   row_tiles (first row, rows, workspace row of the request's position 0, position of the first row): up to
 *     128 consecutive rows of a request, whose positions follow each other; rows without a context have the
 *     position -rows (and get zeros). Rows in no tile are not written.
 * ws_rows: workspace rows, a multiple of 128. heads_at_once heads are expanded, then attended to, at a time.
 * workspace: ayk_latent_chunks_workspace_bytes(ws_rows, heads_at_once), 16-byte aligned.
 */
size_t ayk_latent_chunks_workspace_bytes(int64_t ws_rows, int32_t heads_at_once);
int ayk_latent_chunks(void* out, const void* q, const void* cache, const void* keys, const void* values,
                      const int32_t* block_table, int64_t table_stride, const int32_t* token_tiles,
                      int32_t n_token_tiles, const int32_t* row_tiles, int32_t n_row_tiles, int64_t ws_rows,
                      int32_t heads_at_once, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                      int32_t num_blocks, int32_t block_size, int32_t dtype, float scale, void* workspace,
                      size_t workspace_bytes, void* stream);

/*
 * The same with the context of each row tile cut into `splits` parts, 1 to 64, for steps whose row tiles and
 * heads are fewer than the compute units. workspace: ayk_latent_chunks_workspace_bytes rounded up to 16, and
 * ayk_latent_chunks_parts_bytes more.
 */
size_t ayk_latent_chunks_parts_bytes(int32_t n_row_tiles, int32_t heads_at_once, int32_t splits);
int ayk_latent_chunks_split(void* out, const void* q, const void* cache, const void* keys, const void* values,
                            const int32_t* block_table, int64_t table_stride, const int32_t* token_tiles,
                            int32_t n_token_tiles, const int32_t* row_tiles, int32_t n_row_tiles, int64_t ws_rows,
                            int32_t heads_at_once, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                            int32_t num_blocks, int32_t block_size, int32_t dtype, float scale, int32_t splits,
                            void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AYAKA_HIP_LATENT_H */
