/*
 * ayaka_hip_block_scaled.h -- C ABI of the block-scaled 8-bit KV cache (codec "fp8_e4m3_block").
 *
 * Conventions, error codes, layouts and enums are those of ayaka_hip.h: plain C functions over
 * device pointers that allocate, free and synchronise nothing and return AYK_OK or an AYK_ERR_*
 * code with a message in ayk_last_error().
 *
 * The cache holds OCP fp8 e4m3 codes, 1 byte per element, in either layout, and beside them
 * `scales`, float32 [num_blocks, num_kv_heads, 2], contiguous, 8-byte aligned: a key scale and a
 * value scale for every block and key/value head. An element is worth code * scale. A scale is a
 * power of two 2^e, -40 <= e <= 80, or 0 for a block of nothing but zeros; a fresh cache's scales
 * are zeros. Both the write and attention read a scale that is not one of these as the nearest below
 * it: 2^-40 or 2^80 beyond the range, and 0 for anything not above 0. A block's value scale of 0 says
 * that its codes are zeros: attention takes whatever they are as at most 448 * 2^-40. Head widths are 64, 128 and 256; caches are written from and read by fp16 and bf16
 * models. Rows (k, v, q, out) are 16-byte aligned, caches 8-byte. The reference defines the codec
 * field and only the "raw" codec (python/ayaka/ops/kvcache.py:35-36, :54-55).
 */
#ifndef AYAKA_HIP_BLOCK_SCALED_H
#define AYAKA_HIP_BLOCK_SCALED_H

#include "ayaka_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * KV write: row i of k and v (fp16 or bf16 per src_dtype, [n_rows, num_kv_heads, head_dim],
 * contiguous) is encoded into slot slot_mapping[i]. KVCacheOps.store
 * (python/ayaka/ops/backends/torch/kvcache.py:65-80) for this codec.
 *
 * The rows that land in one block must be adjacent rows of the call, each slot at most once (as a
 * planned step's are: a request's rows are consecutive and no two requests write one block). With
 * o the first offset of a block that the call writes, the offsets below o hold the block's earlier
 * tokens and everything behind the call's rows is dead. Per block, head and tensor:
 *   need = the least 2^e (-40 <= e <= 80) with every finite |x| of the call's rows <= 448 * 2^e,
 *          0 if they are all zero
 *   new scale = need if o is 0, else the larger of need and the block's scale
 *   earlier tokens, where the scale grew: code -> e4m3(code * old / new)
 *   new tokens: e4m3(x / new), rounded to nearest even; magnitudes above 448 (possible only at
 *          e = 80) become 448, infinities and NaN the NaN code
 * Rows whose slot lies in block 0 (padding) or outside the pool are dropped: block 0 and its
 * scales are left as they are.
 */
int ayk_store_block_scaled(const void* k, const void* v, void* k_cache, void* v_cache, float* scales,
                           const int64_t* slot_mapping, int64_t n_rows, int32_t num_kv_heads, int32_t head_dim,
                           int32_t num_blocks, int32_t block_size, int32_t layout, int32_t src_dtype, void* stream);

/*
 * Attention over a block-scaled cache: the entry points of ayaka_hip.h with the cache's scales in
 * the place of kv_dtype, k_scale and v_scale, and otherwise their arguments, semantics, work lists,
 * workspaces and flags (AYK_FLAG_QK_DPP is refused, as over every fp8 cache; dtype is fp16 or bf16):
 *   ayk_paged_attention_v1_block_scaled       ayk_paged_attention_v1
 *   ayk_paged_attention_v2_block_scaled       ayk_paged_attention_v2
 *   ayk_paged_prefill_block_scaled            ayk_paged_prefill
 *   ayk_paged_attention_windows_block_scaled  ayk_paged_attention_windows
 * Position t of a request counts with the scales of its block: its score is
 * scale * key scale * q.code and its value code * value scale. Weights times their value scales are
 * rounded to 16 bits in units of the largest: half a step, 2^-11, down to 2^-14 of it and an absolute
 * 2^-25 of it below, so what blocks far quieter than the loudest add to an element is resolved to
 * that. A NaN code at a position a row does
 * not attend to does not reach the row; one at a position it attends to makes the elements it
 * belongs to NaN (a value's) or the row's head (a key's).
 */
int ayk_paged_attention_v1_block_scaled(void* out, const void* q, const void* k_cache, const void* v_cache,
                                        const float* scales, const int32_t* block_table, int64_t table_stride,
                                        const int32_t* kv_lengths, const int32_t* request_of_row,
                                        const int32_t* positions, int32_t n_rows, int32_t num_heads,
                                        int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks, int32_t block_size,
                                        int32_t max_blocks, int32_t layout, int32_t dtype, float scale, int32_t flags,
                                        void* stream);
int ayk_paged_attention_v2_block_scaled(void* out, const void* q, const void* k_cache, const void* v_cache,
                                        const float* scales, const int32_t* block_table, int64_t table_stride,
                                        const int32_t* kv_lengths, const int32_t* request_of_row,
                                        const int32_t* positions, int32_t n_rows, int32_t num_heads,
                                        int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks, int32_t block_size,
                                        int32_t max_blocks, int32_t layout, int32_t dtype, float scale,
                                        int32_t partition_size, int32_t max_partitions, const int32_t* work_items,
                                        int32_t n_work_items, const int32_t* staged, void* workspace,
                                        size_t workspace_bytes, uint32_t* arrivals, int32_t flags, void* stream);
int ayk_paged_prefill_block_scaled(void* out, const void* q, const void* k_cache, const void* v_cache,
                                   const float* scales, const int32_t* block_table, int64_t table_stride,
                                   const int32_t* kv_lengths, const int32_t* request_of_row, const int32_t* positions,
                                   const int32_t* tiles, int32_t n_tiles, int32_t tile_pairs, int32_t n_rows,
                                   int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                                   int32_t block_size, int32_t max_blocks, int32_t layout, int32_t dtype, float scale,
                                   int32_t partition_size, void* workspace, size_t workspace_bytes, void* stream);
int ayk_paged_attention_windows_block_scaled(void* out, const void* q, const void* k_cache, const void* v_cache,
                                             const float* scales, const int32_t* block_table, int64_t table_stride,
                                             const int32_t* kv_lengths, const int32_t* request_of_row,
                                             const int32_t* positions, const int32_t* tiles, int32_t n_tiles,
                                             int32_t n_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                             int32_t num_blocks, int32_t block_size, int32_t max_blocks, int32_t layout,
                                             int32_t dtype, float scale, int32_t partition_size, void* workspace,
                                             size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AYAKA_HIP_BLOCK_SCALED_H */
