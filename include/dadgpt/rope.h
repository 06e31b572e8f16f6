/*
 * libdadgpt_attn.so — rotary positions on the MI355X (gfx950), forward and backward. No reference
 * counterpart: the reference's positions are learned embeddings (src/model.cpp:17-56).
 *
 * Conventions, status codes and dadgpt_last_error() as <dadgpt/gpu_attention.h>: device pointers,
 * 16-byte aligned unless an entry says otherwise; every argument checked on the host before any
 * HIP call; work on `stream` (NULL: the null stream) of the current device; nothing allocated.
 */
#ifndef DADGPT_ROPE_H
#define DADGPT_ROPE_H

#include <stddef.h>
#include <stdint.h>

#include "gpu_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* How frequencies are scaled for contexts `factor` times as long as the `original_len` tokens that a
 * model was trained on; f_i = base^(-2i / rot_dim) is pair i's unscaled frequency. */
enum {
  DADGPT_ROPE_UNSCALED = 0,
  DADGPT_ROPE_LINEAR = 1, /* f_i / factor: positions are squeezed into the trained range */
  DADGPT_ROPE_BASE = 2,   /* f_i of base * factor^(rot_dim / (rot_dim - 2)): the slowest pair turns
                             1 / factor as fast, the fastest as before; rot_dim >= 4 */
  DADGPT_ROPE_PARTS = 3   /* by the turns t_i = original_len f_i / 2 pi of a pair over the trained
                             context: as it was from `fast` turns on, f_i / factor up to `slow`, and
                             between them f_i (g + (1 - g) / factor), g = (t_i - slow) / (fast - slow) */
};

/* The frequencies (radians a position) of the rot_dim / 2 pairs into HOST memory, in double. rot_dim is
 * even and positive, base and factor are positive and finite; PARTS wants original_len >= 1 and
 * slow < fast, the others ignore the three. */
int dadgpt_rope_frequencies(double* freqs, int rot_dim, double base, int scaling, double factor,
                            int original_len, double slow, double fast);

/* Rotates the first rot_dim elements of every head of q [B, H, S, d_head] and k [B, Hkv, S, d_head]
 * into q_out and k_out; the others are copied. Pair i of a head is its elements (i, i + rot_dim / 2), or
 * (2i, 2i + 1) with `interleaved`, and becomes
 *     magnitude * (x cos a - y sin a, x sin a + y cos a),   a = position * freqs[i].
 * Element d of row s of head h of batch b lies at b*batch + h*head + s*row + d of its tensor;
 * strides: HOST array of those of q, k, q_out and k_out, non-negative multiples of 8 elements. Heads
 * of a fused projection's rows, contiguous [B*H, S, d_head] and anything between will do.
 *   freqs      DEVICE double [rot_dim / 2], 8-byte aligned
 *   positions  DEVICE int32 [B, S], 4-byte aligned, any values; NULL: row s is at position s
 * rot_dim is a multiple of 8 of at most d_head (32 or 64). k and k_out may be NULL (Hkv 0): q alone.
 * Angles are reduced in double, so that far positions keep fp32 accuracy; results are computed in
 * fp32, two products and a sum, and bf16's rounded once. In place: q_out = q (k_out = k) with the same strides. No other overlap of an output with
 * another tensor is accepted, but tensors of the same strides may lie in each other's gaps. */
int dadgpt_rope_bf16(uint16_t* q_out, uint16_t* k_out, const uint16_t* q, const uint16_t* k,
                     const dadgpt_head_strides* strides, int B, int H, int Hkv, int S, int d_head,
                     const double* freqs, int rot_dim, int interleaved, float magnitude,
                     const int32_t* positions, void* stream);
int dadgpt_rope_f32(float* q_out, float* k_out, const float* q, const float* k,
                    const dadgpt_head_strides* strides, int B, int H, int Hkv, int S, int d_head,
                    const double* freqs, int rot_dim, int interleaved, float magnitude,
                    const int32_t* positions, void* stream);

/* Its gradient: dq and dk (overwritten) of dq_out and dk_out, with the forward's other arguments.
 * The rotation is linear, so it is the rotation by the negative angles; strides are those of dq_out,
 * dk_out, dq and dk, and in place is dq = dq_out (dk = dk_out). */
int dadgpt_rope_backward_bf16(uint16_t* dq, uint16_t* dk, const uint16_t* dq_out,
                              const uint16_t* dk_out, const dadgpt_head_strides* strides, int B,
                              int H, int Hkv, int S, int d_head, const double* freqs, int rot_dim,
                              int interleaved, float magnitude, const int32_t* positions,
                              void* stream);
int dadgpt_rope_backward_f32(float* dq, float* dk, const float* dq_out, const float* dk_out,
                             const dadgpt_head_strides* strides, int B, int H, int Hkv, int S,
                             int d_head, const double* freqs, int rot_dim, int interleaved,
                             float magnitude, const int32_t* positions, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DADGPT_ROPE_H */
