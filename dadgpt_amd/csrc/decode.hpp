// What the decode kernels share (one query token per sequence and head against a ragged cache):
// the elements' arithmetic, streaming and coherent accesses, the keys a window leaves, and the
// merge of a cache's waves and chunks.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

#if defined(__gfx942__) || defined(__gfx950__) || !defined(__HIP_DEVICE_COMPILE__)
#define DADGPT_DECODE_SC1_COHERENT 1
#else
#define DADGPT_DECODE_SC1_COHERENT 0
#endif

namespace dadgpt {
namespace {

template <typename T>
struct Elem;
template <>
struct Elem<bf16> {
  static constexpr int kPer16B = 8;
  static __device__ __forceinline__ void unpack(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16_lo(w[i]);
      f[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  // q . k over the 8 bf16 pairs of two 16-byte words: four v_dot2_f32_bf16 on the packed
  // operands (bf16 products are exact in fp32), with no unpacking of either side.
  static __device__ __forceinline__ float dot(const u32x4& q, const u32x4& k) {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t qi = q[i], ki = k[i];
      acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, qi),
                                            __builtin_bit_cast(bf16x2, ki), acc, false);
    }
    return acc;
  }
  static __device__ __forceinline__ bf16 from(float x) { return static_cast<bf16>(x); }
};
template <>
struct Elem<float> {
  static constexpr int kPer16B = 4;
  static __device__ __forceinline__ void unpack(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ float dot(const u32x4& q, const u32x4& k) {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = fmaf(__uint_as_float(q[i]), __uint_as_float(k[i]), acc);
    return acc;
  }
  static __device__ __forceinline__ float from(float x) { return x; }
};

__device__ __forceinline__ int clamp_len(int L, int max_len) {
  return L < 0 ? 0 : (L > max_len ? max_len : L);
}

// Cache rows are read once: non-temporal loads.
__device__ __forceinline__ u32x4 ld_stream(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// Agent-scope relaxed accesses: each is coherent across the XCDs by itself.
__device__ __forceinline__ void st_agent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float ld_agent(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Workspace of a split decode: one uint32 arrival counter per (sequence, head) from the start
// (the region rounded up to 256 bytes), and the fp32 partials [n_seq*H][n_chunk][D+2] packed
// against the END of the caller's buffer. A buffer sized for the largest shape it serves thus
// never has a later call's partials over any counter of a call of another shape, and the
// counters, rearmed by every call, stay zero between calls.
size_t counter_bytes(int n_seq, int H) {
  return (sizeof(unsigned) * (size_t)n_seq * H + 255) & ~(size_t)255;
}
size_t partial_bytes(int n_seq, int H, int n_chunk, int D) {
  return sizeof(float) * (size_t)n_seq * H * n_chunk * (D + 2);
}


// The keys that the last row of a cache of `len` rows sees, counted without the gap between the
// sinks and the window: key i lies in row row(i).
template <bool WIN>
struct VisibleKeys {
  int count, sinks, gap;
  __device__ __forceinline__ VisibleKeys(int len, const WindowArg<WIN>& w)
      : count(len), sinks(0), gap(0) {
    if constexpr (WIN) {
      sinks = w.sinks;
      gap = max(len - w.window, sinks) - sinks;  // rows sinks .. sinks + gap - 1 are not seen
      count = len - gap;
    }
  }
  __device__ __forceinline__ int row(int i) const { return WIN && i >= sinks ? i + gap : i; }
};
template <int D, int WAVES>
struct MergeLds {
  float o[WAVES][D];
  float m[WAVES], l[WAVES];
  int last;
};

// Merges the workgroup's waves (running maximum mx in log2 units, sum lsum, unnormalised o of
// EPL columns from `col`, given by the lanes with `holds`) and writes the cache's output row, or,
// where the cache has nch > 1 chunks, publishes the chunk's partial; the last chunk to arrive
// merges all of them. An empty cache (nch 0) gives zeros; NAN_ZERO also where the sum of an unsplit
// cache is NaN (the plain decode's behaviour; the others pass NaN on).
template <bool NAN_ZERO, typename T, int D, int WAVES, int EPL>
__device__ __forceinline__ void merge_chunks(MergeLds<D, WAVES>& sm, T* out, const float (&o)[EPL],
                                             float mx, float lsum, int wave, int lane, bool holds,
                                             int col, int chunk, int nch, float* part,
                                             unsigned* counter) {
  const int tid = threadIdx.x;
  if (holds) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) sm.o[wave][col + e] = o[e];
  }
  if (lane == 0) {
    sm.m[wave] = mx;
    sm.l[wave] = lsum;
  }
  __syncthreads();

  // merge the waves (threads 0..D-1 own one output column each)
  float wm = neg_inf(), wl = 0.f, wo = 0.f;
  if (tid < D) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) wm = fmaxf(wm, sm.m[w]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = sm.m[w] == neg_inf() ? 0.f : fast_exp2(sm.m[w] - wm);
      wl += sm.l[w] * f;
      wo += sm.o[w][tid] * f;
    }
  }
  if (nch <= 1) {  // the whole cache is this chunk
    if (tid < D) out[tid] = Elem<T>::from((NAN_ZERO ? wl > 0.f : nch == 1) ? wo / wl : 0.f);
    return;
  }

  // Split cache: publish this chunk's partial; the last chunk to arrive merges all of them.
  if (tid < D) {
    float* my = part + chunk * (D + 2);
    st_agent(my + 2 + tid, wo);
    if (tid == 0) {
      st_agent(my, wm);
      st_agent(my + 1, wl);
    }
  }
#if DADGPT_DECODE_SC1_COHERENT
  // This thread's stores are complete at the device coherence point (the asm is also a
  // compiler barrier for them); the barrier then covers the whole workgroup's.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
    sm.last = before == (unsigned)(nch - 1);
  }
#else
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_ACQ_REL,
                                                   __HIP_MEMORY_SCOPE_AGENT);
    sm.last = before == (unsigned)(nch - 1);
  }
#endif
  __syncthreads();
  if (!sm.last) return;

  if (tid < D) {
    // The partials of kMergeBatch chunks are all loaded before any is used (one memory round
    // trip per batch: this merge ends the kernel for the caches that finish last), and the
    // batches merge online. For nch <= kMergeBatch this is sum_c l_c 2^(m_c - max) in chunk
    // order, as a two-pass merge. A chunk whose scores are all -inf has that as its maximum and
    // weighs nothing; while there is no other, 0 stands in for the running maximum.
    constexpr int kMergeBatch = 4;
    float gm = neg_inf(), gl = 0.f, go = 0.f;
    for (int c0 = 0; c0 < nch; c0 += kMergeBatch) {
      float mv[kMergeBatch], lv[kMergeBatch], ov[kMergeBatch];
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j) {
        const float* pc = part + min(c0 + j, nch - 1) * (D + 2);  // past nch: unused
        mv[j] = ld_agent(pc);
        lv[j] = ld_agent(pc + 1);
        ov[j] = ld_agent(pc + 2 + tid);
      }
      float bm = gm;
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j)
        if (c0 + j < nch) bm = fmaxf(bm, mv[j]);
      const float base = bm == neg_inf() ? 0.f : bm;
      const float fo = fast_exp2(gm - base);  // 0 before the first batch (gl = go = 0 then)
      gl *= fo;
      go *= fo;
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j)
        if (c0 + j < nch) {
          const float f = fast_exp2(mv[j] - base);
          gl += lv[j] * f;
          go += ov[j] * f;
        }
      gm = bm;
    }
    out[tid] = Elem<T>::from(go / gl);
  }
  // All nch arrivals of this call are in: rearm the counter for the next call.
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace
}  // namespace dadgpt
