/*
 * libdadgpt_attn.so — KV caches in pages on the MI355X (gfx950): append (with rotary positions) and
 * attention of each sequence's new tokens, one or thousands, over its pages. No reference
 * counterpart: the reference's KVCache (src/model.hpp:140-152) is one stretch for one sequence.
 *
 * Conventions, status codes and dadgpt_last_error() as <dadgpt/gpu_attention.h>: device pointers,
 * 16-byte aligned unless an entry says otherwise; every argument checked on the host before any
 * HIP call; work on `stream` (NULL: the null stream) of the current device; nothing allocated.
 *
 * The cache. k_pages and v_pages [n_pages, n_kv_heads, page, d_head]: `page` (16, 32, 64 or 128) tokens
 * of every KV head to a page; d_head 32 or 64. Token j of sequence s lies in slot j % page of page
 * block_table[s][j / page]; block_table is DEVICE int32 [n_seq, max_pages], 4-byte aligned, and
 * max_pages * page is at most DADGPT_PAGED_MAX_LEN. Query head h reads KV head h / (n_heads / n_kv_heads).
 *
 * A step. `rows` rows hold the new tokens of all sequences one after the other: sequence s owns
 * rows row_start[s] .. row_start[s + 1] - 1 (DEVICE int32 [n_seq + 1], not decreasing, within [0, rows];
 * a count of 0 is allowed), at most max_rows of them (what it has beyond them is left out). lens
 * (DEVICE int32 [n_seq], clamped to [0, max_pages * page]) counts the tokens of each sequence WITH its
 * new rows, so row t of a sequence's `count` is token lens[s] - count + t. Rows behind the last
 * sequence's, and rows left out, are not read, and their outputs are left as they were.
 *
 * An entry of the block table outside [0, n_pages) names no page: rows are not written there, and its
 * tokens are not seen. Entries past the sequence's length are not looked at.
 */
#ifndef DADGPT_PAGED_CACHE_H
#define DADGPT_PAGED_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "gpu_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DADGPT_PAGED_MAX_LEN (65535 * 256)

/* Writes the new rows into the pages, rotating q and k on the way as dadgpt_rope_* (<dadgpt/rope.h>)
 * with each row's token number as its position; freqs NULL: no rotation (rot_dim 0 then).
 * Row r of q holds n_heads * d_head elements from r * ld_q on, those of k and v n_kv_heads * d_head
 * from r * ld_kv on: slices of a fused projection's rows, or tensors of their own. q_out's rows are
 * ld_out apart; q_out may be q (ld_out = ld_q). q and q_out may both be NULL: k and v alone (ld_q and
 * ld_out are not looked at). Pitches are multiples of 8 elements, at most 2^24. Rows before token 0 (a count above the length) are not
 * written. Two sequences must not append into one page. Outputs overlap nothing else. */
int dadgpt_paged_append_bf16(uint16_t* k_pages, uint16_t* v_pages, uint16_t* q_out, int64_t ld_out,
                             const uint16_t* q, int64_t ld_q, const uint16_t* k,
                             const uint16_t* v, int64_t ld_kv, const int32_t* block_table, const int32_t* row_start,
                             const int32_t* lens, int n_seq, int n_heads, int n_kv_heads, int rows,
                             int max_rows, int n_pages, int page, int max_pages, int d_head,
                             const double* freqs, int rot_dim, int interleaved, float magnitude,
                             void* stream);
int dadgpt_paged_append_f32(float* k_pages, float* v_pages, float* q_out, int64_t ld_out,
                            const float* q, int64_t ld_q, const float* k, const float* v,
                            int64_t ld_kv, const int32_t* block_table, const int32_t* row_start,
                            const int32_t* lens, int n_seq, int n_heads, int n_kv_heads, int rows,
                            int max_rows, int n_pages, int page, int max_pages, int d_head,
                            const double* freqs, int rot_dim, int interleaved, float magnitude,
                            void* stream);

/* out = softmax(scale q k^T) v for every new row, over its sequence's tokens up to and with its own.
 * Equal steps give equal bits. The order of the sums, and for bf16 whether the weights are rounded to it for
 * the product with v (above 32 rows of max_rows * n_heads / n_kv_heads, as dadgpt_flash_attention_* does),
 * depend on the step's shape and all its lengths, so a sequence in a step with others may differ from
 * the same sequence alone by those roundings.
 * Row r of q (out) holds n_heads * d_head elements from r * ld_q (ld_out) on; out may be q (ld_out =
 * ld_q). A row none of whose keys weighs anything (it lies before token 0, all its pages are missing,
 * all its scores are -inf) gets zeros. A NaN key or value makes the rows that see it NaN, an infinite value
 * its column infinite; values that a row does not see, but that another row of the step sees, may reach it as
 * 0 * v: a NaN or infinity there can make it NaN too. (fp32 elements above 3.39e38 may count as infinite.)
 * The workspace is as the decode calls': dadgpt_paged_workspace_bytes (0: NULL allowed) of this shape, or
 * of one with larger n_seq, rows, max_rows or max_pages, ZERO-FILLED once, 16-byte aligned, and passed
 * whole; every call leaves its counters at zero. Calls that share one must not overlap in time. */
size_t dadgpt_paged_workspace_bytes(int n_seq, int n_heads, int n_kv_heads, int rows, int max_rows,
                                    int page, int max_pages, int d_head);
int dadgpt_paged_attention_bf16(uint16_t* out, int64_t ld_out, const uint16_t* q, int64_t ld_q,
                                const uint16_t* k_pages, const uint16_t* v_pages,
                                const int32_t* block_table, const int32_t* row_start,
                                const int32_t* lens, int n_seq, int n_heads, int n_kv_heads,
                                int rows, int max_rows, int n_pages, int page, int max_pages,
                                int d_head, float scale, void* workspace, size_t workspace_bytes,
                                void* stream);
int dadgpt_paged_attention_f32(float* out, int64_t ld_out, const float* q, int64_t ld_q,
                               const float* k_pages, const float* v_pages,
                               const int32_t* block_table, const int32_t* row_start,
                               const int32_t* lens, int n_seq, int n_heads, int n_kv_heads,
                               int rows, int max_rows, int n_pages, int page, int max_pages,
                               int d_head, float scale, void* workspace, size_t workspace_bytes,
                               void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DADGPT_PAGED_CACHE_H */
