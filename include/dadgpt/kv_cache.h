/*
 * libdadgpt_attn.so — bounded KV caches on the MI355X (gfx950): caches held in 8 bits, and eviction
 * by accumulated attention weight. No reference counterpart: the reference's KVCache
 * (src/model.hpp:140-152) keeps every token in fp32.
 *
 * Conventions, status codes and dadgpt_last_error() as <dadgpt/gpu_attention.h>: device pointers,
 * 16-byte aligned unless an entry says otherwise; every argument checked on the host before any
 * HIP call; work on `stream` (NULL: the null stream) of the current device; nothing allocated.
 * Outputs and workspaces that overlap each other or an input are refused, except as an entry says.
 * Cache layout [n_seq, n_heads, max_len, d_head] as the decode calls', d_head 32 or 64; lens are
 * DEVICE int32 [n_seq], clamped to [0, max_len].
 */
#ifndef DADGPT_KV_CACHE_H
#define DADGPT_KV_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "gpu_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 8-bit cache. Codes are OCP e4m3 (uint8_t [n_seq, n_heads, max_len, d_head], 16-byte
 * aligned) with a float scale for each block of `block` tokens (16, 32, 64 or 128) of a
 * (sequence, head): scales [n_seq, n_heads, ceil(max_len / block)], 4-byte aligned. A value is
 * code * scale. The append chooses the least power of two, at least 2^-100, for which the block's
 * largest finite magnitude is at most 448 scale, so every implementation of the definition gets
 * the same codes: round-to-nearest-even of x / scale; infinities and NaN are held as NaN and do
 * not count towards the scale. */

/* Blocks of a cache of max_len rows (the scales' last dimension); 0 for a block size other than
 * those above. */
int dadgpt_kv8_blocks(int max_len, int block);

/* Appends rows t < counts[s] of k and v at cache rows lens[s] + t (lens is not changed; the caller
 * advances it). counts: DEVICE int32 [n_seq], clamped to [0, rows], or NULL for `rows` each. Rows
 * that would lie at or past max_len are dropped. Row t of head h of sequence s of k starts at
 * element s*k_strides->batch + h*k_strides->head + t*k_strides->row (likewise v), so the rows may
 * be read out of a projection's token-major output; strides are non-negative multiples of 8
 * elements. A block that already holds rows below lens[s] keeps its scale unless the new rows need
 * a larger one; then those rows are re-rounded to the new scale (exact but for codes that fall
 * below e4m3's normal range). What a block holds from lens[s] on does not count and is left as it
 * was where no row is appended. */
int dadgpt_kv8_append_bf16(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale,
                           const uint16_t* k, const uint16_t* v,
                           const dadgpt_head_strides* k_strides,
                           const dadgpt_head_strides* v_strides, const int32_t* lens,
                           const int32_t* counts, int n_seq, int n_heads, int rows, int max_len,
                           int d_head, int block, void* stream);
int dadgpt_kv8_append_f32(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale,
                          const float* k, const float* v, const dadgpt_head_strides* k_strides,
                          const dadgpt_head_strides* v_strides, const int32_t* lens,
                          const int32_t* counts, int n_seq, int n_heads, int rows, int max_len,
                          int d_head, int block, void* stream);

/* Decode attention over an 8-bit cache (q and out bf16 or fp32 [n_seq, n_heads, d_head], out may be
 * q; any float scales). window = 0 sees every row below lens[s] (sinks must be 0 then); window >= 1 has the mask
 * of dadgpt_decode_attention_window_*. A length of 0 gives a zero output row. The workspace is as
 * the decode calls': dadgpt_decode_kv8_workspace_bytes (0: NULL allowed), sized for the largest
 * shape it serves, ZERO-FILLED once, and passed whole; every call leaves its counters at zero.
 * Calls that share one must not overlap in time. With a window, what min(max_len, window + sinks)
 * rows need is enough. */
size_t dadgpt_decode_kv8_workspace_bytes(int n_seq, int n_heads, int max_len, int d_head);
int dadgpt_decode_attention_kv8_bf16(uint16_t* out, const uint16_t* q, const uint8_t* k_cache,
                                     const uint8_t* v_cache, const float* k_scale,
                                     const float* v_scale, const int32_t* lens, int n_seq,
                                     int n_heads, int max_len, int d_head, int block, float scale,
                                     int window, int sinks, void* workspace,
                                     size_t workspace_bytes, void* stream);
int dadgpt_decode_attention_kv8_f32(float* out, const float* q, const uint8_t* k_cache,
                                    const uint8_t* v_cache, const float* k_scale,
                                    const float* v_scale, const int32_t* lens, int n_seq,
                                    int n_heads, int max_len, int d_head, int block, float scale,
                                    int window, int sinks, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* ---- Eviction by accumulated attention weight, over bf16 and fp32 caches. */

/* The decode of dadgpt_decode_attention_{bf16,f32}, which also accumulates every key's attention
 * probability: weights_out[s][h][j] = weights[s][h][j] + p_j for j < lens[s], and weights[s][h][j]
 * from there on. The caller sets a row's weight (to 0) when it appends the row. out may be q. weights
 * and weights_out are fp32 [n_seq, n_heads, max_len], 4-byte aligned, and may be one buffer; otherwise
 * they must not overlap. The workspace (dadgpt_decode_weights_workspace_bytes, 0: NULL allowed)
 * needs no initial contents and holds nothing between calls; calls that overlap in time need one
 * each. */
size_t dadgpt_decode_weights_workspace_bytes(int n_seq, int n_heads, int max_len, int d_head);
int dadgpt_decode_attention_weights_bf16(uint16_t* out, float* weights_out, const uint16_t* q,
                                         const uint16_t* k_cache, const uint16_t* v_cache,
                                         const float* weights, const int32_t* lens, int n_seq,
                                         int n_heads, int max_len, int d_head, float scale,
                                         void* workspace, size_t workspace_bytes, void* stream);
int dadgpt_decode_attention_weights_f32(float* out, float* weights_out, const float* q,
                                        const float* k_cache, const float* v_cache,
                                        const float* weights, const int32_t* lens, int n_seq,
                                        int n_heads, int max_len, int d_head, float scale,
                                        void* workspace, size_t workspace_bytes, void* stream);

/* Cuts every (sequence, head) back to `budget` rows. One with lens[s] <= budget keeps all its rows;
 * a longer one keeps its first `sinks`, its last `recent`, and of the rows between those with the
 * largest weights, budget rows in all (sinks + recent <= budget); equal weights go to the lowest
 * row, -0 equals 0, NaN is below everything. The kept rows keep their order: row r of the output
 * cache is row kept[s][h][r] of the input, r < lens_out[s] = min(lens[s], budget).
 *   k_out, v_out  [n_seq, n_heads, max_out, d_head], max_out >= min(budget, max_len); rows from
 *                 lens_out on are left as they were
 *   weights_out   [n_seq, n_heads, max_out] fp32, 4-byte aligned; from lens_out on left as they
 *                 were: a row that is appended there later needs its weight set (to 0)
 *   kept          int32 [n_seq, n_heads, budget], 4-byte aligned; -1 from lens_out on
 *   lens_out      int32 [n_seq], 4-byte aligned; may be lens
 * In place: k_out = k and v_out = v together, with max_out = max_len; weights_out may be weights
 * (max_out = max_len). No other overlap is accepted. */
int dadgpt_kv_evict_bf16(uint16_t* k_out, uint16_t* v_out, float* weights_out, int32_t* kept,
                         int32_t* lens_out, const uint16_t* k, const uint16_t* v,
                         const float* weights, const int32_t* lens, int n_seq, int n_heads,
                         int max_len, int max_out, int d_head, int budget, int sinks, int recent,
                         void* stream);
int dadgpt_kv_evict_f32(float* k_out, float* v_out, float* weights_out, int32_t* kept,
                        int32_t* lens_out, const float* k, const float* v, const float* weights,
                        const int32_t* lens, int n_seq, int n_heads, int max_len, int max_out,
                        int d_head, int budget, int sinks, int recent, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DADGPT_KV_CACHE_H */
