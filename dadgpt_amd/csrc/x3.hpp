// fp32 products at fp32 accuracy on the bf16 matrix cores, and what the fp32 attention kernels
// (attn_f32.hip, paged_attn.hip) build of them: tiles split as they are staged, scores, weights times
// values, and the exponential.
#pragma once

#include "common.hpp"
#include "tiles.hpp"

namespace dadgpt {
namespace {

// Row (within a 32-row chunk) that score register u of lane half h stands for, when the A
// operand rows were read through sigma32: 16 * (u / 8) + 8 * h + u % 8.
__device__ __forceinline__ constexpr int reg_row(int u, int h) {
  return 16 * (u >> 3) + 8 * h + (u & 7);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// e^x to ~1.3 ulp (measured over [-87, 44] against double exp: 1.24 ulp, the library expf
// 0.85) in six VALU operations instead of the library's thirteen: x log2(e) as a rounded
// product e plus its exact remainder r (an FMA, with log2(e) split into two floats), then
// 2^e on the hardware exp2 and the first-order correction 2^(e+r) = 2^e (1 + r ln 2). Results
// below 2^-126 flush to zero and above 2^128 are +inf (no range reduction): the softmax
// weights these kernels exponentiate are either negligible there or take the rescaling path.
// An infinite x gives NaN (its remainder is inf - inf): callers keep -inf out.
__device__ __forceinline__ float exp_acc(float x) {
  constexpr float kL1 = 1.44269502162933349609375f;  // log2(e) rounded to float
  constexpr float kL2 = 1.925963033500011079e-08f;   // log2(e) - kL1
  const float e = x * kL1;
  const float r = fmaf(x, kL2, fmaf(x, kL1, -e));
  const float p = __builtin_amdgcn_exp2f(e);
  return fmaf(p, r * kLn2, p);
}

// A chunk whose weights reach this in some row moves that row's running maximum: with
// weights below 2^64, the running sums stay far inside fp32 range over any sequence length.
constexpr float kMaxW = 0x1p64f;

// fp32 products on the bf16 matrix cores. A float x is split into three bf16 values
// x = x1 + x2 + x3 (each the round-to-nearest of what the previous ones leave, so the three
// carry 24 significant bits and the rest is below 2^-27 |x|); a product x y is then the six
// cross terms whose weight is at least 2^-18 (x1y1, x1y2, x2y1, x1y3, x3y1, x2y2), each exact
// in fp32 and summed by the MFMA in fp32. Six v_mfma_f32_32x32x16_bf16 (32 cycles each) do
// the work of eight v_mfma_f32_32x32x2_f32 (64 cycles each), and, unlike the fp32 MFMA, they
// run beside the VALU. Measured over random 32x32x64 products: largest error 2.5e-7 of
// sum |x_k y_k|, against 3.5e-7 for the fp32 MFMA.
struct X3 {
  bf16x8 v[3];
};

// pack_bf16x2 for a word whose halves are taken apart again: opaque, because the compiler would
// otherwise convert the low half a second time instead of shifting it out of the word (48 of
// dK/dV's 576 VALU instructions per chunk). ONCE = false leaves the compiler the second
// conversion, which does not wait for the first: shorter for a wave that has its SIMD to itself.
template <bool ONCE = true>
__device__ __forceinline__ uint32_t pack_once(float lo, float hi) {
  uint32_t w = pack_bf16x2(lo, hi);
  if constexpr (ONCE) asm("" : "+v"(w));
  return w;
}

template <bool ONCE = true>
__device__ __forceinline__ X3 split3(const float (&x)[8]) {
  u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a0 = x[2 * i], a1 = x[2 * i + 1];
    const uint32_t p = pack_once<ONCE>(a0, a1);
    const float b0 = a0 - bf16_lo(p), b1 = a1 - bf16_hi(p);  // exact
    const uint32_t q = pack_once<ONCE>(b0, b1);
    const float c0 = b0 - bf16_lo(q), c1 = b1 - bf16_hi(q);  // exact
    w[0][i] = p;
    w[1][i] = q;
    w[2][i] = pack_bf16x2(c0, c1);
  }
  return X3{{as_bf16x8(w[0]), as_bf16x8(w[1]), as_bf16x8(w[2])}};
}

// acc += A B over a 16-deep slice, A and B as X3 (smallest terms first).
__device__ __forceinline__ f32x16 mfma_x6(const X3& a, const X3& b, f32x16 acc) {
  acc = mfma32(a.v[1], b.v[1], acc);
  acc = mfma32(a.v[2], b.v[0], acc);
  acc = mfma32(a.v[0], b.v[2], acc);
  acc = mfma32(a.v[1], b.v[0], acc);
  acc = mfma32(a.v[0], b.v[1], acc);
  return mfma32(a.v[0], b.v[0], acc);
}

// A 64-row tile split into three bf16 planes in LDS, each in the row-major swizzled layout of
// the bf16 kernels (tiles.hpp), so the score operands are ds_read_b128 and the transposed
// ones ds_read_b64_tr_b16 reads. Each float is split once per workgroup, when the tile is
// staged, instead of once per wave that reads it.
template <int D, int TR, typename T>
__device__ __forceinline__ void store_x3(const T& t, bf16* planes) {
#pragma unroll
  for (int i = 0; i < T::kPieces; ++i) {
    const int u = threadIdx.x + T::kThreads * i, row = u / (D / 4), c = u % (D / 4);
    const int off = rm_off<D>(row, c >> 1) + 4 * (c & 1);  // 4 floats: half a 16-byte chunk
    const f32x4 x = t.piece(i);
    uint32_t w[3][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float a0 = x[2 * k], a1 = x[2 * k + 1];
      const uint32_t p = pack_once(a0, a1);
      const float b0 = a0 - bf16_lo(p), b1 = a1 - bf16_hi(p);
      const uint32_t q = pack_once(b0, b1);
      w[0][k] = p;
      w[1][k] = q;
      w[2][k] = pack_bf16x2(b0 - bf16_lo(q), b1 - bf16_hi(q));
    }
#pragma unroll
    for (int pl = 0; pl < 3; ++pl)
      *reinterpret_cast<u32x2*>(planes + pl * TR * D + off) = u32x2{w[pl][0], w[pl][1]};
  }
}

// The B operand of a score product from a global row: lane half h supplies columns
// 16 ds + 8 h + 0..7 of `row`, split into three bf16 planes.
template <int D, bool ONCE = true>
__device__ __forceinline__ void load_split_row(X3 (&x)[D / 16], const float* row, int h) {
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    float a[8];
    const f32x4 v0 = *reinterpret_cast<const f32x4*>(row + 16 * ds + 8 * h);
    const f32x4 v1 = *reinterpret_cast<const f32x4*>(row + 16 * ds + 8 * h + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = v0[e], a[4 + e] = v1[e];
    x[ds] = split3<ONCE>(a);
  }
}

template <int D, int TR>
__device__ __forceinline__ f32x16 score_tile_p(const bf16* planes, int chunk_row0,
                                               const X3 (&qb)[D / 16], int lane) {
  const int krow = chunk_row0 + sigma32(lane & 31), hi = lane >> 5;
  f32x16 acc = zero16();
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    X3 a;
#pragma unroll
    for (int pl = 0; pl < 3; ++pl)
      a.v[pl] = lds_op(planes + pl * TR * D, rm_off<D>(krow, 2 * ds + hi));
    acc = mfma_x6(a, qb[ds], acc);
  }
  return acc;
}

template <int D, int TR, bool ONCE = true>
__device__ __forceinline__ void accumulate_t_p(f32x16 (&acc)[D / 32], const bf16* planes,
                                               int chunk_row0, const f32x16& p, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[8 * j + e];
    const X3 pb = split3<ONCE>(x);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      X3 a;
#pragma unroll
      for (int pl = 0; pl < 3; ++pl)
        a.v[pl] = lds_tr_op<D>(planes + pl * TR * D, chunk_row0 + 16 * j, 32 * db, lane);
      acc[db] = mfma_x6(a, pb, acc[db]);
    }
  }
}

}  // namespace
}  // namespace dadgpt
