// Rotary positions, for the kernels that move heads from one place to another (rope.hip, paged.hip):
// a thread owns 2 VEC elements of a head of a token, VEC pairs or, past rot_dim, elements that are only
// copied.
#pragma once

#include "common.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace rotary {

// cos and sin of VEC pairs' angles, times the magnitude.
template <int VEC>
struct Turn {
  float c[VEC], s[VEC];
};

// The angle pos * f in turns, reduced in double (its error is pos * f * 2^-52 and below 2^-24 of what
// is left), then the library's sin(pi x) and cos(pi x), which need no reduction of their own; for bf16
// (FAST) the instructions for sin and cos of a number of turns, off by at most 2^-22.9, and 2^-20 of a small
// sine (measured over [-1/2, 1/2]), far below half a step of the result, 2^-9.
template <int VEC, bool FAST>
__device__ __forceinline__ Turn<VEC> turn_of(const double* __restrict__ freqs, int pos,
                                             float magnitude, bool inverse) {
  constexpr double kTurns = 0.15915494309189533577;  // 1 / 2 pi
  Turn<VEC> t;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const double a = (double)pos * (freqs[e] * kTurns);
    const float x = (float)(a - __builtin_rint(a));
    float s, c;
    if constexpr (FAST)
      s = __builtin_amdgcn_sinf(x), c = __builtin_amdgcn_cosf(x);
    else
      sincospif(2.0f * x, &s, &c);
    t.c[e] = c * magnitude;
    t.s[e] = (inverse ? -s : s) * magnitude;
  }
  return t;
}

template <int WORDS>
struct Words;
template <>
struct Words<2> {
  typedef u32x2 type;
};
template <>
struct Words<4> {
  typedef u32x4 type;
};

// VEC consecutive elements as they lie in memory: 8 or 16 bytes.
template <typename T, int VEC>
struct Piece {
  typedef typename Words<VEC * (int)sizeof(T) / 4>::type type;
  type w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const type*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<type*>(p) = w; }
  __device__ __forceinline__ void floats(float* x) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = __uint_as_float(w[i]);
    }
  }
  __device__ __forceinline__ void from(const float* x) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(x[i]);
    }
  }
};

// What a thread's chunk c (of d_head / (2 VEC)) of a head is: where its two pieces start, and whether
// they are rotated.
struct Chunk {
  int at[2];
  bool rotated;
};
template <int VEC, bool INTER>
__device__ __forceinline__ Chunk chunk_of(int c, int rot_dim) {
  const bool rotated = 2 * c * VEC < rot_dim;
  if (!INTER && rotated) return Chunk{{c * VEC, c * VEC + rot_dim / 2}, true};
  return Chunk{{2 * c * VEC, 2 * c * VEC + VEC}, rotated};
}

// Turns the pairs of two pieces in fp32, each result rounded once to T.
template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void turn_pieces(Piece<T, VEC>& a, Piece<T, VEC>& b,
                                            const Turn<VEC>& t) {
  float x[2 * VEC], y[2 * VEC];
  a.floats(x);
  b.floats(x + VEC);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : VEC + e;
    y[i] = fmaf(x[i], t.c[e], -(x[j] * t.s[e]));
    y[j] = fmaf(x[i], t.s[e], x[j] * t.c[e]);
  }
  a.from(y);
  b.from(y + VEC);
}

// Elements of a piece: 8 where the pairs come in whole eights (bf16), otherwise 4.
template <typename T>
inline bool wide(int rot_dim, int D) {
  return sizeof(T) == 2 && rot_dim % 16 == 0 && D % 16 == 0;
}

}  // namespace rotary
}  // namespace dadgpt
