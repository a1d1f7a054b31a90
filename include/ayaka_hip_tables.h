/*
 * ayaka_hip_tables.h -- C ABI of the step tables built on the GPU: the blocks a step's requests
 * lack, and every row's position and slot, from the requests' lengths in device memory.
 *
 * Conventions and error codes are those of ayaka_hip.h. All pointers are device pointers unless
 * said otherwise; nothing is read on the host, so the calls can be captured into a graph and need
 * no lengths there. A decode bucket is then ready for attention (ayk_paged_attention_v2 reads the
 * staged split); a step of any rows is ready for the KV write, while its attention still takes a
 * tile or work list made from lengths the host knows. The rules are those the reference applies on the
 * host: positions and slots as python/ayaka/ops/backends/torch/attention.py:64-164, a decode
 * bucket's as :308-374 (SLOT = table[position / block_size] * block_size + position % block_size).
 */
#ifndef AYAKA_HIP_TABLES_H
#define AYAKA_HIP_TABLES_H

#include "ayaka_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most requests of one step. */
#define AYK_TABLES_MAX_REQUESTS 4096
/* Most work items of one step. */
#define AYK_TABLES_MAX_ITEMS (1 << 18)
/* Most partition sizes ayk_advance_decode_tables chooses from. */
#define AYK_TABLES_MAX_SIZES 32

/*
 * Request b brings rows[b] rows, the last of the lengths[b] tokens it has after the step. It holds
 * the first ceil((lengths[b] - rows[b]) / block_size) entries of its row of block_table and needs
 * ceil(lengths[b] / block_size); the entries it lacks are filled with free_blocks[taken[0] ...],
 * handed out in request order. Rows are numbered through the requests in order, and of each the
 * call writes request_of_row, positions (lengths[b] - rows[b] + j) and slot_mapping.
 *
 * A request is not served if it asks for what cannot be: negative rows, more rows than tokens, more
 * blocks than max_blocks, a row past n_rows; if the last entry it should hold is the padding block 0
 * (a step before this one did not serve it, and its length was raised all the same); or if the free
 * blocks run out at it (from there on, in request order, only requests that need no block are
 * served). Nothing of its table row is written,
 * its rows get position 0 and slot 0 (which the KV write drops or keeps to the padding block), and
 * it counts into after[1] unless its length is 0 (padding: not an error). Rows behind the last
 * request's get request 0, position 0, slot 0. A negative rows[b] numbers no rows.
 *   kv_lengths[b] = lengths[b] if served, else 0 (the attention calls then treat it as padding)
 *   after[0] = taken[0] + the blocks handed out, after[1] = the requests not served
 * after holds 4 words, zeros before the first call that uses it; after[2] is the calls' own and is
 * left at zero. after[0] may be taken[0] itself (the pool advances in place) and kv_lengths may be
 * lengths; the other outputs overlap nothing. Calls that overlap in time need separate `after`s. A
 * taken[0] outside [0, n_free] counts as the nearer end. Table entries a request holds are used as
 * they are: the KV write drops slots outside its pool, the attention calls read block 0 for them.
 * Results do not depend on scheduling.
 */
int ayk_build_tables(const int32_t* rows, const int32_t* lengths, int32_t n_requests, int32_t* block_table,
                     int64_t table_stride, int32_t max_blocks, const int32_t* free_blocks, int32_t n_free,
                     const int32_t* taken, int32_t* after, int32_t block_size, int32_t* request_of_row,
                     int32_t* positions, int64_t* slot_mapping, int32_t n_rows, int32_t* kv_lengths, void* stream);

/*
 * The same for a decode bucket: one row per request, row b request b's (request_of_row is not
 * written), and with it the step's v2 split staged for ayk_paged_attention_v2: `staged` receives
 * {partition size, item count, each row's first partial slot, (row, partition) pairs}, as that
 * call's `staged` and `work_items` (staged + 2 + n_requests) read them, of at most `capacity`
 * items. The size is the one of sizes[0 .. n_sizes) (HOST memory; rising multiples of 64 up to 2^30) whose
 * work, dealt to compute_units workgroups of one item and head group (`groups` per item) each
 * costing its positions plus `cost`, is modelled to end first, or one partition per row where no
 * size's items fit; partitions are listed full ones first, then falling by 1/256 of the size.
 */
int ayk_advance_decode_tables(const int32_t* lengths, int32_t n_requests, int32_t* block_table, int64_t table_stride,
                              int32_t max_blocks, const int32_t* free_blocks, int32_t n_free, const int32_t* taken,
                              int32_t* after, int32_t block_size, int32_t* positions, int64_t* slot_mapping,
                              int32_t* kv_lengths, int32_t* staged, int32_t capacity, const int32_t* sizes,
                              int32_t n_sizes, int32_t groups, int32_t cost, int32_t compute_units, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AYAKA_HIP_TABLES_H */
