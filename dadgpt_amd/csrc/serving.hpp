// Host-side launch interface of the rotary positions, the paged caches and the sampling (rope.hip,
// paged.hip, paged_attn.hip, sampling.hip), behind capi_serving.cpp, which checks every argument.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"

namespace dadgpt {

struct Strides64 {
  long long batch, head, row;
};

// Rotary positions of q [B, H, S, D] and k [B, Hkv, S, D] (Hkv may be 0). Strides in the order
// q, k, q_out, k_out; `magnitude` multiplies the rotated elements, `inverse` turns them back.
struct Rope {
  const double* freqs;
  int rot_dim;
  bool interleaved, inverse;
  float magnitude;
};
struct RopeShape {
  int B, H, Hkv, S, D;
  Strides64 t[4];
};
hipError_t launch_rope_bf16(bf16* q_out, bf16* k_out, const bf16* q, const bf16* k,
                            const RopeShape& shape, const Rope& rope, const int* positions,
                            hipStream_t stream);
hipError_t launch_rope_f32(float* q_out, float* k_out, const float* q, const float* k,
                           const RopeShape& shape, const Rope& rope, const int* positions,
                           hipStream_t stream);

// A step over a paged cache (include/dadgpt/paged_cache.h).
struct PagedStep {
  const int *table, *row_start, *lens;
  int n_seq, H, Hkv, rows, max_rows, n_pages, page, max_pages, D;
};
// q_out and q may be null (k and v alone).
hipError_t launch_paged_append_bf16(bf16* k_pages, bf16* v_pages, bf16* q_out, long long ld_out,
                                    const bf16* q, long long ld_q, const bf16* k, const bf16* v,
                                    long long ld_kv, const PagedStep& step, const Rope& rope, hipStream_t stream);
hipError_t launch_paged_append_f32(float* k_pages, float* v_pages, float* q_out, long long ld_out,
                                   const float* q, long long ld_q, const float* k, const float* v,
                                   long long ld_kv, const PagedStep& step, const Rope& rope, hipStream_t stream);

// Whether the step's grid is within the launch limits.
bool paged_fits(const PagedStep& step, int elem_bytes);
// Bytes that this step's launch uses, and those that serve it and every step with no larger n_seq, rows,
// max_rows and max_pages.
size_t paged_workspace_needed(const PagedStep& step, int elem_bytes);
size_t paged_workspace_bytes(const PagedStep& step);
hipError_t launch_paged_attention_bf16(bf16* out, long long ld_out, const bf16* q, long long ld_q,
                                       const bf16* k_pages, const bf16* v_pages,
                                       const PagedStep& step, float scale, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream);
hipError_t launch_paged_attention_f32(float* out, long long ld_out, const float* q, long long ld_q,
                                      const float* k_pages, const float* v_pages,
                                      const PagedStep& step, float scale, void* workspace,
                                      size_t workspace_bytes, hipStream_t stream);

// Sampling (include/dadgpt/sampling.h); the arrays of settings may be null.
struct SampleSettings {
  const float *uniforms, *temperature, *top_p, *min_p;
  const int* top_k;
};
hipError_t launch_sample_bf16(int* tokens, float* probs, const bf16* logits, long long ld, int rows,
                              int vocab, const SampleSettings& settings, hipStream_t stream);
hipError_t launch_sample_f32(int* tokens, float* probs, const float* logits, long long ld, int rows,
                             int vocab, const SampleSettings& settings, hipStream_t stream);

}  // namespace dadgpt
