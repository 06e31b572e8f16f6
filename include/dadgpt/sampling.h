/*
 * libdadgpt_attn.so — picking tokens from logits on the MI355X (gfx950) by given random numbers, for
 * a batch of rows, every row with its own settings. The reference picks on the host, one row at a time
 * (sample_token, src/generate.cpp:16-92).
 *
 * Conventions, status codes and dadgpt_last_error() as <dadgpt/gpu_attention.h>: device pointers;
 * every argument checked on the host before any HIP call; work on `stream` (NULL: the null stream)
 * of the current device; nothing allocated.
 */
#ifndef DADGPT_SAMPLING_H
#define DADGPT_SAMPLING_H

#include <stddef.h>
#include <stdint.h>

#include "gpu_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DADGPT_SAMPLE_MAX_VOCAB (1 << 19)

/* tokens[r] for every row r of logits (vocab elements from r * ld on, at least 4-byte aligned rows of
 * fp32, 2-byte of bf16), and probs[r] (may be NULL) the probability that it was drawn with:
 *   1. w_i = exp((logit_i - largest logit) / temperature). A temperature that is not above 0 takes the
 *      first largest logit, with probability 1, and looks at nothing else.
 *   2. In descending order of the logits (ties: lowest index first) only a head of the list stays:
 *      the first top_k (0 or less: all), of these the fewest whose weights sum to at least top_p of
 *      theirs (1 or more, NaN: all; at least one), and of these the ones with w_i >= min_p (NaN: all;
 *      at least the first).
 *   3. The token is the first i, in the order of the vocabulary, at which the sum of the weights that
 *      stayed, up to and with i, exceeds uniforms[r] times the whole sum; uniforms are in [0, 1), what
 *      is outside (NaN) counts as the nearest end (0).
 * Logits of NaN and -inf are never picked; where there are +inf logits, they alone are, with equal
 * weights. A row that has nothing else gets token -1 and probability 0. Weights are computed in
 * double and summed as multiples of 2^-44, in integers: the result does not depend on the order, and a
 * token of less than 2^-45 of the largest weight is not drawn, by a uniform number of 0 either.
 * temperature, top_p, min_p (float) and top_k (int32) are DEVICE arrays [rows], 4-byte aligned, each
 * may be NULL: 1, all, 0, all. Outputs overlap nothing else. */
int dadgpt_sample_bf16(int32_t* tokens, float* probs, const uint16_t* logits, int64_t ld, int rows,
                       int vocab, const float* uniforms, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p, void* stream);
int dadgpt_sample_f32(int32_t* tokens, float* probs, const float* logits, int64_t ld, int rows,
                      int vocab, const float* uniforms, const float* temperature,
                      const int32_t* top_k, const float* top_p, const float* min_p, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DADGPT_SAMPLING_H */
