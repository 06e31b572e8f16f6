// Bounded KV caches for gfx950: caches held in 8 bits (append and decode), decode that accumulates
// each key's attention weight, and eviction by that weight. All of it is bound by HBM (one query
// token per sequence and head, as in decode.hip, or a copy), so none of it uses MFMA.
//
// 8-bit cache: codes [n_seq, H, max_len, D] in OCP e4m3, and a float scale for each block of
// `block` tokens of a (sequence, head): the value is code * scale. The scale is the least power of
// two with max|x| <= 448 scale over the block's finite values, so quantising multiplies by an
// exact reciprocal and rounds once (to nearest even), and a block whose scale has to grow re-rounds
// what it holds by an exact shift (only codes that fall into e4m3's subnormals lose a bit).
#include "common.hpp"
#include "decode.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace dadgpt {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The wave's loads are in. A workgroup barrier alone does not wait for loads in flight, which a
// store by another wave after it must not overtake.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ------------------------------------------------------------------------ 8-bit append

constexpr int kAppendWaves = 4;
constexpr uint32_t kInfBits = 0x7f800000u;

// Eight consecutive source elements, as they lie in memory until they are looked at.
template <typename T>
struct Eight;
template <>
struct Eight<bf16> {
  u32x4 w = {0u, 0u, 0u, 0u};
  __device__ __forceinline__ void load(const bf16* p) { w = ld_g128u(p); }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
  }
  // not to be kept as floats from one look to the next
  __device__ __forceinline__ void keep() { asm("" : "+v"(w)); }
};
template <>
struct Eight<float> {
  float f[8] = {};
  __device__ __forceinline__ void load(const float* p) {
    const u32x4 a = ld_g128u(p), b = ld_g128u(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(a[i]), f[4 + i] = __uint_as_float(b[i]);
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f[i];
  }
  __device__ __forceinline__ void keep() {}
};

// Eight e4m3 codes of x * mul (rounded to nearest even; |x * mul| <= 448, or NaN).
__device__ __forceinline__ u32x2 to_e4m3(const float (&x)[8], float mul) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * mul, x[4 * i + 1] * mul, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * mul, x[4 * i + 3] * mul, c, true);
    w[i] = (uint32_t)c;
  }
  return w;
}
__device__ __forceinline__ void from_e4m3(float (&x)[4], uint32_t w) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
}

// The least power of two s with a <= 448 s (448 = 1.75 * 2^8), at least 2^-100, for the bits of a
// finite a >= 0.
__device__ __forceinline__ float e4m3_scale(uint32_t a) {
  const int e = (int)(a >> 23) - 127 - 8 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// WPB waves for each touched block of a (sequence, head) and tensor: D/8 lanes a row, NI rows a lane,
// all of them loaded before the block's maximum is taken and still in registers when it is known.
// Grid (heads, K and V: 4 waves a workgroup; touched blocks; sequences), heads fastest, so that
// neighbours read one stretch of the projection's token-major rows. Bound by that chain (lengths, rows,
// maximum, codes, once a workgroup) more than by HBM: 16 x 12 prompts of 1 to 1024 tokens in blocks of
// 32, 38 MB, 11.5 us in bf16, 63 MB, 14.6 in fp32; one token for each of 32 x 12 caches 3.4.
template <typename T, int D, int NI, int WPB>
__global__ __launch_bounds__(64 * kAppendWaves) void kv8_append_kernel(
    uint8_t* __restrict__ k8, uint8_t* __restrict__ v8, float* __restrict__ k_scale,
    float* __restrict__ v_scale, const T* __restrict__ k, const T* __restrict__ v,
    const HeadStrides64 ks, const HeadStrides64 vs, const int* __restrict__ lens,
    const int* __restrict__ counts, int H, int rows, int max_len) {
  constexpr int LPR = D / 8, RPI = 64 / LPR, BLOCK = NI * RPI * WPB;
  const int lane = threadIdx.x & 63, sub = lane % LPR, grp = lane / LPR;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % WPB;
  const int unit = (blockIdx.x * kAppendWaves + wave) / WPB;
  const bool is_v = unit & 1;
  const int head = unit >> 1, seq = blockIdx.z, at = blockIdx.y;
  if (head >= H) return;  // (with more than one wave a block, whole workgroups)
  const int begin = clamp_len(lens[seq], max_len);
  const int count = counts == nullptr ? rows : clamp_len(counts[seq], rows);
  const int end = begin + min(count, max_len - begin);
  const int blk = begin / BLOCK + at, lo = blk * BLOCK;
  if (lo >= end || begin >= end) return;
  const int first = lo + part * NI * RPI + grp;  // the lane's rows: every RPI-th

  const HeadStrides64& st = is_v ? vs : ks;
  const T* src = (is_v ? v : k) + seq * st.batch + head * st.head + sub * 8;
  const long long hrow = (long long)seq * H + head;
  uint8_t* dst = (is_v ? v8 : k8) + (hrow * max_len + first) * D + sub * 8;
  float* scale = (is_v ? v_scale : k_scale) + hrow * ((max_len + BLOCK - 1) / BLOCK) + blk;

  Eight<T> x[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = first + i * RPI;
    if (r >= begin && r < end) x[i].load(src + (long long)(r - begin) * st.row);
  }
  const bool has_old = lo < begin;
  const float s_old = has_old ? *scale : 0.f;
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float f[8];
    x[i].floats(f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
      amax = max(amax, a >= kInfBits ? 0u : a);
    }
    x[i].keep();
  }
  // (bits of non-negative floats order as the floats do)
  float most = lanes::group_max<64>(__uint_as_float(amax));
  if constexpr (WPB > 1) {
    __shared__ float sm[kAppendWaves];
    if (lane == 0) sm[wave] = most;
    wait_loads();  // (s_old: another wave stores the new scale)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPB; ++i) most = fmaxf(most, sm[wave - part + i]);
  }
  const uint32_t am = __float_as_uint(most);
  const float s_new = fmaxf(s_old, e4m3_scale(am));
  const float inv = 1.0f / s_new;  // exact
  const bool regrow = has_old && s_new > s_old;  // wave-uniform
  const float ratio = s_old * inv;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = first + i * RPI;
    uint8_t* p = dst + i * RPI * D;
    if (r >= begin && r < end) {
      float f[8];
      x[i].floats(f);
#pragma unroll
      for (int e = 0; e < 8; ++e)  // an infinity is held as e4m3's NaN, as NaN is
        if ((__float_as_uint(f[e]) & 0x7fffffffu) >= kInfBits) f[e] = __uint_as_float(0x7fc00000u);
      *reinterpret_cast<u32x2*>(p) = to_e4m3(f, inv);
    } else if (regrow && r < begin) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      float old[8];
      from_e4m3(reinterpret_cast<float(&)[4]>(old[0]), w[0]);
      from_e4m3(reinterpret_cast<float(&)[4]>(old[4]), w[1]);
      *reinterpret_cast<u32x2*>(p) = to_e4m3(old, ratio);
    }
  }
  if (lane == 0 && part == 0) *scale = s_new;
}

template <typename T, int D>
hipError_t launch_kv8_append_d(uint8_t* k8, uint8_t* v8, float* k_scale, float* v_scale,
                               const T* k, const T* v, const HeadStrides64& ks,
                               const HeadStrides64& vs, const int* lens, const int* counts,
                               int n_seq, int H, int rows, int max_len, int block,
                               hipStream_t stream) {
  auto launch = [&](auto ni, auto wpb) {
    const dim3 grid((2 * H * wpb() + kAppendWaves - 1) / kAppendWaves,
                    kv8_touched_blocks(rows, block), n_seq);
    kv8_append_kernel<T, D, ni(), wpb()><<<grid, 64 * kAppendWaves, 0, stream>>>(
        k8, v8, k_scale, v_scale, k, v, ks, vs, lens, counts, H, rows, max_len);
    return hipGetLastError();
  };
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 4> four;
  switch (block * D / 512) {
    case 1:  // 16 tokens of 32 columns
      if constexpr (D == 32) return launch(one, one);
      break;
    case 2: return launch(two, one);
    case 4: return launch(four, one);
    case 8: return launch(four, two);
    case 16:  // 128 tokens of 64 columns
      if constexpr (D == 64) return launch(four, four);
      break;
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t launch_kv8_append_t(uint8_t* k8, uint8_t* v8, float* k_scale, float* v_scale,
                               const T* k, const T* v, const HeadStrides64& ks,
                               const HeadStrides64& vs, const int* lens, const int* counts,
                               int n_seq, int H, int rows, int max_len, int D, int block,
                               hipStream_t stream) {
  if (D == 64)
    return launch_kv8_append_d<T, 64>(k8, v8, k_scale, v_scale, k, v, ks, vs, lens, counts, n_seq,
                                      H, rows, max_len, block, stream);
  if (D == 32)
    return launch_kv8_append_d<T, 32>(k8, v8, k_scale, v_scale, k, v, ks, vs, lens, counts, n_seq,
                                      H, rows, max_len, block, stream);
  return hipErrorInvalidValue;
}

// ------------------------------------------------------------------------ 8-bit decode

// softmax(scale q . k) v with k = s_k code, v = s_v code: a key's scale multiplies its score, a
// value's its probability, so the codes themselves go into the products. Work split as decode.hip's:
// a chunk of keys per 8-wave workgroup, 16-byte loads that cover whole key rows (16 codes a lane: 4
// lanes a row at D = 64), all of a wave's loads issued before any arithmetic, chunks of one cache
// merged by the last to arrive. 8 x 12 caches of 1 to 32768 rows, 200 MB, 35 us, 5.7 TB/s; 32 x 12
// of 1 to 1024, 25 MB, 8.1 us, of which a launch with next to nothing to read is 4. Windowed: 32 x 12
// of 1 to 1024 under 256 5.6, 8 x 12 of 1 to 32768 under 4096, 47 MB, 11.0.
constexpr int kKv8Waves = 8;
constexpr int kKv8Loads = 8;  // 16-byte loads per lane and tensor
template <int D>
__host__ __device__ constexpr int kv8_chunk_keys() {
  return kKv8Waves * kKv8Loads * 64 / (D / 16);
}

// q . code over a lane's 16 columns: bf16 queries on packed pairs (every e4m3 code is a bf16
// value, products of two bf16 are exact in fp32), fp32 ones in fp32.
template <typename T>
struct Query16;
template <>
struct Query16<bf16> {
  u32x4 w[2];
  __device__ __forceinline__ void load(const bf16* p) {
    w[0] = ld_g128u(p);
    w[1] = ld_g128u(p + 8);
  }
  __device__ __forceinline__ float dot(const u32x4& k) const {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[i], 1.0f, false);
      const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[i], 1.0f, true);
      const uint32_t q0 = w[i / 2][2 * (i % 2)], q1 = w[i / 2][2 * (i % 2) + 1];
      acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, q0), lo, acc, false);
      acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, q1), hi, acc, false);
    }
    return acc;
  }
};
template <>
struct Query16<float> {
  float x[16];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 w = ld_g128u(p + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = __uint_as_float(w[e]);
    }
  }
  __device__ __forceinline__ float dot(const u32x4& k) const {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float c[4];
      from_e4m3(c, k[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = fmaf(x[4 * i + e], c[e], acc);
    }
    return acc;
  }
};

// Sum over the lanes of a wave that agree modulo N (2 or 4).
template <int N>
__device__ __forceinline__ float sum_modulo(float x) {
  if constexpr (N <= 2) x += lanes::dpp<lanes::kRor2>(x);
  x += lanes::dpp<lanes::kRor4>(x);
  x += lanes::dpp<lanes::kRor8>(x);
  return lanes::sum_xor32(lanes::sum_xor16(x));
}

template <typename T, int D, bool WIN>
__global__ __launch_bounds__(64 * kKv8Waves) void kv8_decode_kernel(
    T* __restrict__ out, const T* __restrict__ q, const uint8_t* __restrict__ k8,
    const uint8_t* __restrict__ v8, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, const int* __restrict__ lens, int H, int max_len,
    int block_log2, int blocks, float scale_log2, float* __restrict__ part,
    unsigned* __restrict__ counter, int n_chunk, const WindowArg<WIN> win) {
  constexpr int LPR = D / 16;                 // lanes per key row
  constexpr int KPL = 64 / LPR;               // key rows per wave-wide load
  constexpr int NLD = kKv8Loads, KW = NLD * KPL, C = kv8_chunk_keys<D>();
  __shared__ MergeLds<D, kKv8Waves> sm;

  const int seq = blockIdx.x / H, head = blockIdx.x % H, chunk = blockIdx.y;
  const VisibleKeys<WIN> keys(clamp_len(lens[seq], max_len), win);
  const int L = keys.count;
  const int nch = (L + C - 1) / C;
  // Chunks past the length do nothing; chunk 0 of an empty cache still writes the zero output.
  if (chunk >= (nch > 1 ? nch : 1)) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform: scalar
  const int sub = lane % LPR, grp = lane / LPR;
  const size_t hrow = (size_t)seq * H + head;
  const uint8_t* kh = k8 + hrow * max_len * D + sub * 16;
  const uint8_t* vh = v8 + hrow * max_len * D + sub * 16;
  const float* ksh = k_scale + hrow * blocks;
  const float* vsh = v_scale + hrow * blocks;
  const int key0 = chunk * C + wave * KW;

  float mx = neg_inf(), lsum = 0.f;
  float o[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.f;

  if (key0 < L) {  // wave-uniform: waves past the length skip their loads
    Query16<T> qv;
    qv.load(q + hrow * D + sub * 16);
    // Keys past the length load key L-1 instead (valid, since key0 < L) and are masked out below.
    // Without a window the KPL = 16 rows of a load at D = 64 lie in one block: scalar scales.
    constexpr bool kUniform = !WIN && KPL == 16;
    u32x4 kr[NLD], vr[NLD];
    float ks[NLD], vs[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int row = keys.row(min(key0 + i * KPL + grp, L - 1));
      kr[i] = ld_stream(kh + (size_t)row * D);
      ks[i] = ksh[(kUniform ? min(key0 + i * KPL, L - 1) : row) >> block_log2];
    }
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int row = keys.row(min(key0 + i * KPL + grp, L - 1));
      vr[i] = ld_stream(vh + (size_t)row * D);
      vs[i] = vsh[(kUniform ? min(key0 + i * KPL, L - 1) : row) >> block_log2];
    }
    // Keep the scheduler from sinking loads towards their uses: all of them stay in flight.
    __builtin_amdgcn_sched_barrier(0);

    float s[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float acc = lanes::group_sum<LPR>(qv.dot(kr[i]));
      s[i] = key0 + i * KPL + grp < L ? acc * (ks[i] * scale_log2) : neg_inf();
      mx = fmaxf(mx, s[i]);
    }
    mx = lanes::group_max<64>(mx);
    // where every score is -inf (past fp32's range), 0 stands in for the maximum
    const float base = mx == neg_inf() ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float p = fast_exp2(s[i] - base);  // exactly 0 for masked keys
      lsum += p;
      const float pv = p * vs[i];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float c[4];
        from_e4m3(c, vr[i][w]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * w + e] = fmaf(pv, c[e], o[4 * w + e]);
      }
    }
    lsum = sum_modulo<LPR>(lsum);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = sum_modulo<LPR>(o[e]);
  }
  merge_chunks<false, T, D, kKv8Waves>(sm, out + hrow * D, o, mx, lsum, wave, lane, grp == 0,
                                       sub * 16, chunk, nch, part + hrow * n_chunk * (D + 2),
                                       counter + hrow);
}

template <typename T, int D>
hipError_t launch_kv8_decode_d(T* out, const T* q, const uint8_t* k8, const uint8_t* v8,
                               const float* k_scale, const float* v_scale, const int* lens,
                               int n_seq, int H, int max_len, int block, float scale,
                               const Window* window, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
  const int most = window ? visible_keys(max_len, *window) : max_len;
  if (window != nullptr && most == max_len) window = nullptr;  // every key is seen
  const int nc = (most + kv8_chunk_keys<D>() - 1) / kv8_chunk_keys<D>();
  float* part = nullptr;
  unsigned* counter = nullptr;
  if (nc > 1) {
    const size_t at = (workspace_bytes - partial_bytes(n_seq, H, nc, D)) & ~(size_t)15;
    counter = static_cast<unsigned*>(workspace);
    part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
  }
  const dim3 grid(n_seq * H, nc);
  const int shift = __builtin_ctz((unsigned)block), blocks = (max_len + block - 1) / block;
  if (window != nullptr)
    kv8_decode_kernel<T, D, true><<<grid, 64 * kKv8Waves, 0, stream>>>(
        out, q, k8, v8, k_scale, v_scale, lens, H, max_len, shift, blocks, scale * kLog2e, part,
        counter, nc, {*window});
  else
    kv8_decode_kernel<T, D, false><<<grid, 64 * kKv8Waves, 0, stream>>>(
        out, q, k8, v8, k_scale, v_scale, lens, H, max_len, shift, blocks, scale * kLog2e, part,
        counter, nc, {});
  return hipGetLastError();
}

// ------------------------------------------------------------------------ decode with weights

// decode_kernel's split, with each key's score kept: the probability needs the cache's final
// maximum and sum. A cache of one chunk has them in the workgroup; longer ones leave scores and
// partials in the workspace for weights_kernel.
// ONE: a workgroup runs through its cache's chunks, two at most, and needs neither. 16 x 12 caches
// of 1 to 8192 rows of 64 bf16, 206 MB, 35 us and 5.4 for weights_kernel; 32 x 12 of 1 to 1024, 52 MB,
// 13 us. In place as into another buffer.
constexpr int kWWaves = 8, kWLoads = 8, kWChunks = 2;
template <typename T, int D>
__host__ __device__ constexpr int weights_chunk_keys() {
  return kWWaves * kWLoads * 64 / (D / Elem<T>::kPer16B);
}

template <typename T, int D, bool ONE>
__global__ __launch_bounds__(64 * kWWaves) void weights_decode_kernel(
    T* __restrict__ out, float* wout, const T* __restrict__ q, const T* __restrict__ kc,
    const T* __restrict__ vc, const float* win, const int* __restrict__ lens, int H, int max_len,
    float scale_log2, float* __restrict__ part, float* __restrict__ scores, int n_chunk) {
  constexpr int EPL = Elem<T>::kPer16B, LPR = D / EPL, KPL = 64 / LPR, NLD = kWLoads;
  constexpr int WAVES = kWWaves, NT = 64 * WAVES;
  constexpr int KW = NLD * KPL, C = weights_chunk_keys<T, D>();
  __shared__ float sm_o[WAVES][D];
  __shared__ float sm_m[WAVES], sm_l[WAVES];
  __shared__ float sm_s[C * (ONE ? kWChunks : 1)];

  const int seq = blockIdx.x / H, head = blockIdx.x % H, chunk = blockIdx.y;
  const int L = clamp_len(lens[seq], max_len);
  const int nch = (L + C - 1) / C;
  if (!ONE && chunk >= (nch > 1 ? nch : 1)) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane % LPR, grp = lane / LPR;
  const size_t hrow = (size_t)seq * H + head;
  const T* kh = kc + hrow * max_len * D + sub * EPL;
  const T* vh = vc + hrow * max_len * D + sub * EPL;

  float mx = neg_inf(), lsum = 0.f;
  float o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = 0.f;
  const u32x4 qw = ld_g128u(q + hrow * D + sub * EPL);
  const int local = wave * KW;
  for (int at = 0; chunk * C + at + local < L; at += C) {  // once, unless ONE
    const int key0 = chunk * C + at + local;
    u32x4 kr[NLD], vr[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i)
      kr[i] = ld_stream(kh + (size_t)min(key0 + i * KPL + grp, L - 1) * D);
#pragma unroll
    for (int i = 0; i < NLD; ++i)
      vr[i] = ld_stream(vh + (size_t)min(key0 + i * KPL + grp, L - 1) * D);
    __builtin_amdgcn_sched_barrier(0);
    const float before = mx;
    float s[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float acc = lanes::group_sum<LPR>(Elem<T>::dot(qw, kr[i]));
      s[i] = key0 + i * KPL + grp < L ? acc * scale_log2 : neg_inf();
      mx = fmaxf(mx, s[i]);
      if (sub == 0) sm_s[at + local + i * KPL + grp] = s[i];
    }
    mx = lanes::wave_max_of_groups<LPR>(mx);
    // where every score so far is -inf, 0 stands in for the maximum: those keys' terms are 0
    const float base = mx == neg_inf() ? 0.f : mx;
    if (ONE && at > 0) {
      const float f = fast_exp2(before - base);
      lsum *= f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] *= f;
    }
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float p = fast_exp2(s[i] - base);  // exactly 0 for masked rows
      lsum += p;
      float vf[EPL];
      Elem<T>::unpack(vr[i], vf);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(p, vf[e], o[e]);
    }
    if constexpr (!ONE) break;
  }
  if constexpr (LPR < 8) {
    lsum += __shfl_xor(lsum, LPR, 64);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] += __shfl_xor(o[e], LPR, 64);
  }
  constexpr int K0 = LPR < 8 ? 8 : LPR;
  lsum = lanes::sum_across<K0>(lsum);
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = lanes::sum_across<K0>(o[e]);
  if (grp == 0) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) sm_o[wave][sub * EPL + e] = o[e];
  }
  if (lane == 0) {
    sm_m[wave] = mx;
    sm_l[wave] = lsum;
  }
  __syncthreads();
  float wm = neg_inf(), wl = 0.f, wo = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) wm = fmaxf(wm, sm_m[w]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float f = sm_m[w] == neg_inf() ? 0.f : fast_exp2(sm_m[w] - wm);
    wl += sm_l[w] * f;
    if (tid < D) wo += sm_o[w][tid] * f;
  }
  if constexpr (ONE) {
    if (tid < D) out[hrow * D + tid] = Elem<T>::from(L > 0 ? wo / wl : 0.f);
    const float inv = 1.0f / wl;
    for (int key = tid; key < max_len; key += NT) {
      const float w = win[hrow * max_len + key];
      wout[hrow * max_len + key] = key < L ? w + fast_exp2(sm_s[key] - wm) * inv : w;
    }
    return;
  }
  float* my = part + (hrow * n_chunk + chunk) * (D + 2);
  if (tid < D) {
    my[2 + tid] = wo;
    if (tid == 0) {
      my[0] = wm;
      my[1] = wl;
    }
  }
  for (int i = tid; i < C && chunk * C + i < L; i += NT)
    scores[hrow * max_len + chunk * C + i] = sm_s[i];
}

// The caches of more than one chunk: output rows from the partials (chunk 0's workgroup), and every
// key's weight.
constexpr int kWeightsThreads = 256, kWeightsPer = 8;
template <typename T, int D>
__global__ __launch_bounds__(kWeightsThreads) void weights_kernel(
    T* __restrict__ out, float* wout, const float* win, const int* __restrict__ lens, int H,
    int max_len, const float* __restrict__ part, const float* __restrict__ scores, int n_chunk) {
  constexpr int C = weights_chunk_keys<T, D>(), N = kWeightsPer;
  const int seq = blockIdx.x / H, head = blockIdx.x % H, tid = threadIdx.x;
  const size_t hrow = (size_t)seq * H + head;
  const int L = clamp_len(lens[seq], max_len), nch = max(1, (L + C - 1) / C);
  const int key0 = blockIdx.y * (kWeightsThreads * N) + tid;
  float w[N], s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int key = key0 + i * kWeightsThreads;
    w[i] = key < max_len ? win[hrow * max_len + key] : 0.f;
    s[i] = key < L ? scores[hrow * max_len + key] : 0.f;
  }
  const float* ph = part + hrow * n_chunk * (D + 2);
  float gm = neg_inf(), gl = 0.f;
  for (int c = tid & 63; c < nch; c += 64) gm = fmaxf(gm, ph[c * (D + 2)]);
  gm = lanes::group_max<64>(gm);
  for (int c = tid & 63; c < nch; c += 64)
    gl += ph[c * (D + 2) + 1] * (L > 0 ? fast_exp2(ph[c * (D + 2)] - gm) : 0.f);
  gl = lanes::group_sum<64>(gl);
  const float inv = 1.0f / gl;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int key = key0 + i * kWeightsThreads;
    if (key < max_len)
      wout[hrow * max_len + key] = key < L ? w[i] + fast_exp2(s[i] - gm) * inv : w[i];
  }
  if (blockIdx.y == 0 && tid < D) {
    float go = 0.f;
    for (int c = 0; c < nch && L > 0; ++c)
      go += ph[c * (D + 2) + 2 + tid] * fast_exp2(ph[c * (D + 2)] - gm);
    out[hrow * D + tid] = Elem<T>::from(L > 0 ? go * inv : 0.f);
  }
}

template <typename T, int D>
hipError_t launch_weights_decode_d(T* out, float* wout, const T* q, const T* kc, const T* vc,
                                   const float* win, const int* lens, int n_seq, int H,
                                   int max_len, float scale, void* workspace,
                                   hipStream_t stream) {
  constexpr int C = weights_chunk_keys<T, D>();
  // Two chunks by one workgroup of 8 waves, of which a CU holds two: 16 x 12 caches of 2048 rows of
  // 64 bf16 take 14.4 us over four chunks (15.4 split) where 8 x 12 take 12.6 (11.5 split), and 64
  // of 4096 take 91 (84.5 split): past two chunks the split wins or is even. One workgroup of 16
  // waves for two chunks fits a CU once: 32 x 12 caches of 1024 rows took 15.4 us for 13.9.
  if (max_len <= kWChunks * C) {
    weights_decode_kernel<T, D, true><<<dim3(n_seq * H), 64 * kWWaves, 0, stream>>>(
        out, wout, q, kc, vc, win, lens, H, max_len, scale * kLog2e, nullptr, nullptr, 1);
    return hipGetLastError();
  }
  const int nc = (max_len + C - 1) / C;
  float* part = static_cast<float*>(workspace);
  float* scores = part + (size_t)n_seq * H * nc * (D + 2);
  weights_decode_kernel<T, D, false><<<dim3(n_seq * H, nc), 64 * kWWaves, 0, stream>>>(
      out, wout, q, kc, vc, win, lens, H, max_len, scale * kLog2e, part, scores, nc);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  constexpr int per = kWeightsThreads * kWeightsPer;
  weights_kernel<T, D><<<dim3(n_seq * H, (max_len + per - 1) / per), kWeightsThreads, 0, stream>>>(
      out, wout, win, lens, H, max_len, part, scores, nc);
  return hipGetLastError();
}

// ------------------------------------------------------------------------ eviction

constexpr int kSelHeld = 8;  // keys a thread holds; longer rows are read again for each pass
constexpr int kSelRanked = 512;  // candidates ranked against each other
// Radix passes from the top: 11, 11 and 10 bits.
constexpr int kSelBins = 2048;

// Floats as unsigned words in their order: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > kInfBits) return 0;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive prefix sum over the wave's lanes: DPP shifts within rows of 16, then the last lane of a
// row broadcast to the next one (rows 1 and 3), and of the first half to the second.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

struct SelectLds {
  int hist[kSelBins];
  uint32_t cand_key[kSelRanked];  // a bin's keys, and their rows
  int cand_row[kSelRanked];
  int wave_sum[16];
  int n_cand, digit, left, in_bin;  // the pass's digit, the rank left below it, its bin's size
  uint32_t edge_key;
  int edge_row;
};

// One workgroup per (sequence, head): which rows stay. The first `sinks` and the last `recent` do,
// and of the others (first .. last - 1) the `most` of largest weight, of equal ones the lowest rows.
// That is: the rows before an edge in the order (weight down, row up), and the edge, the row of
// rank `most`, is found by a radix search from the top bits: as soon as its bin holds no more than
// kSelRanked rows (mostly after one pass), these are ranked against each other; if the bits run out
// first, the edge is among rows of one weight, and its row is found by counting them in order.
// Then the indices that stay, in order, and their weights. A chain of about ten steps between
// barriers, for 32 x 12 caches of up to 2048 rows (us from the start, mean): weights in 0.7, counted
// 2.4, digit 2.8, candidates 3.3, edge 4.1, places and stores 5.7. HELD: a thread holds its keys (row
// e * NT + t); else each pass reads the row again (from the caches).
template <int NT, bool HELD>
__global__ __launch_bounds__(NT) void evict_select_kernel(
    int* __restrict__ kept, float* wout, const float* weights, const int* __restrict__ lens, int H,
    int max_len, int max_out, int budget, int sinks, int recent) {
  constexpr int NW = NT / 64;
  static_assert(NW <= 16 && kSelBins % NT == 0);
  __shared__ SelectLds sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seq = blockIdx.x / H;
  const long long hrow = blockIdx.x;
  const int L = clamp_len(lens[seq], max_len);
  const float* w = weights + hrow * max_len;
  int* kp = kept + hrow * budget;
  float* wo = wout + hrow * max_out;
  const int keep = min(L, budget);
  for (int i = keep + tid; i < budget; i += NT) kp[i] = -1;

  const int first = min(sinks, L), last = max(first, L - recent);
  float held[HELD ? kSelHeld : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e) {
      const int i = e * NT + tid;
      held[e] = i < L ? w[i] : 0.f;
    }
  }
  // f(row, weight) for the thread's rows
  auto rows = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int e = 0; e < kSelHeld; ++e) {
        const int i = e * NT + tid;
        if (i < L) f(i, held[e]);
      }
    } else {
      for (int i0 = tid; i0 < L; i0 += kSelHeld * NT) {
        float x[kSelHeld];  // in flight together
#pragma unroll
        for (int e = 0; e < kSelHeld; ++e) x[e] = w[min(i0 + e * NT, L - 1)];
#pragma unroll
        for (int e = 0; e < kSelHeld; ++e) {
          const int i = i0 + e * NT;
          if (i < L) f(i, x[e]);
        }
      }
    }
  };

  // put(place, row, weight) for the rows that pick(row, weight) takes, in order: their places are
  // counted in slabs of kSelHeld rows a thread. Within a slab every wave's loads are in before the
  // first put, and a place is no later than its row, so put may write over the rows (in place).
  auto in_order = [&](auto pick, auto put) {
    int seen = 0;
    for (int b0 = 0; b0 < L; b0 += kSelHeld * NT) {
      float x[kSelHeld];
#pragma unroll
      for (int e = 0; e < kSelHeld; ++e)
        x[e] = HELD ? held[HELD ? e : 0] : w[min(b0 + e * NT + tid, L - 1)];
      unsigned long long m[kSelHeld];
      __syncthreads();  // (hist holds the waves' counts now)
#pragma unroll
      for (int e = 0; e < kSelHeld; ++e) {
        const int i = b0 + e * NT + tid;
        m[e] = __ballot(i < L && pick(i, x[e]));
        if (lane == 0) sm.hist[e * NW + wave] = __popcll(m[e]);
      }
      wait_loads();
      __syncthreads();
      constexpr int PER = kSelHeld * NW / 64;  // of the slabs' waves' counts, a lane
      static_assert(PER == 1 || PER == 2);
      const int n0 = sm.hist[PER * lane], n = PER == 2 ? n0 + sm.hist[PER * lane + 1] : n0;
      const int before = seen + wave_scan(n) - n;
#pragma unroll
      for (int e = 0; e < kSelHeld; ++e) {
        const int c = e * NW + wave;
        int at = __shfl(before, c / PER, 64) + __popcll(m[e] & ((1ull << lane) - 1));
        if (PER == 2 && (wave & 1)) at += __shfl(n0, c / PER, 64);
        if ((m[e] >> lane) & 1) put(at, b0 + e * NT + tid, x[e]);
      }
      if constexpr (HELD) break;  // (one slab)
      seen = __shfl(before + n, 63, 64);
    }
  };

  uint32_t edge_key = 0;
  int edge_row = -1;  // (no row is at the edge or past it)
  if (L > budget) {
    int rank = budget - first - (L - last);  // >= 0, and less than last - first
    uint32_t prefix = 0;
    int shift = 32;
    while (true) {
      const int bits = shift == 10 ? 10 : 11;
      shift -= bits;
      for (int i = tid; i < kSelBins; i += NT) sm.hist[i] = 0;
      if (tid == 0) sm.n_cand = 0;
      __syncthreads();
      rows([&](int i, float x) {
        const uint32_t k = order_key(x);
        if (i >= first && i < last && (shift + bits == 32 || (k >> (shift + bits)) == prefix))
          atomicAdd(&sm.hist[(k >> shift) & ((1u << bits) - 1)], 1);
      });
      __syncthreads();
      // the digit whose rows, counted from the largest down, hold the row of that rank: BINS bins
      // a thread, the highest first
      constexpr int BINS = kSelBins / NT;
      int c[BINS], sum = 0;
#pragma unroll
      for (int e = 0; e < BINS; ++e) sum += c[e] = sm.hist[kSelBins - 1 - (BINS * tid + e)];
      const int inc = wave_scan(sum);
      if (lane == 63) sm.wave_sum[wave] = inc;
      __syncthreads();
      int above = inc - sum;
#pragma unroll
      for (int v = 0; v < NW; ++v) above += v < wave ? sm.wave_sum[v] : 0;
#pragma unroll
      for (int e = 0; e < BINS; ++e) {
        if (above <= rank && rank < above + c[e]) {  // one thread, one bin
          sm.digit = kSelBins - 1 - (BINS * tid + e);
          sm.left = rank - above;
          sm.in_bin = c[e];
        }
        above += c[e];
      }
      __syncthreads();
      prefix = prefix << bits | (uint32_t)sm.digit;
      rank = sm.left;
      const int in_bin = sm.in_bin;
      if (in_bin <= kSelRanked) {
        rows([&](int i, float x) {
          const uint32_t k = order_key(x);
          if (i >= first && i < last && (k >> shift) == prefix) {
            const int at = atomicAdd(&sm.n_cand, 1);
            sm.cand_key[at] = k;
            sm.cand_row[at] = i;
          }
        });
        __syncthreads();
        // a wave takes every NW-th candidate, and its lanes compare the candidate with the others, in
        // registers, 64 at a time (a lane a candidate, walking the others in LDS, took 7k cycles for
        // 30 of them: 18.5 us for the 32 x 12 rows of 2048 that take 9 us now)
        uint32_t kj[kSelRanked / 64];
        int rj[kSelRanked / 64];
#pragma unroll
        for (int b = 0; b < kSelRanked / 64; ++b) {
          kj[b] = 0u, rj[b] = max_len;
          if (64 * b >= in_bin) break;
          const int j = 64 * b + lane;
          if (j < in_bin) kj[b] = sm.cand_key[j], rj[b] = sm.cand_row[j];
        }
        constexpr int N = 4;  // candidates whose LDS reads are in flight together
        for (int i = wave; i < in_bin; i += N * NW) {
          uint32_t k[N];
          int row[N], before[N] = {};
#pragma unroll
          for (int u = 0; u < N; ++u) {
            const int at = min(i + u * NW, in_bin - 1);
            k[u] = sm.cand_key[at];
            row[u] = sm.cand_row[at];
          }
#pragma unroll
          for (int b = 0; b < kSelRanked / 64; ++b) {
            if (64 * b >= in_bin) break;
#pragma unroll
            for (int u = 0; u < N; ++u)
              before[u] += __popcll(__ballot(kj[b] > k[u] || (kj[b] == k[u] && rj[b] < row[u])));
          }
#pragma unroll
          for (int u = 0; u < N; ++u)
            if (before[u] == rank && i + u * NW < in_bin && lane == 0) {
              sm.edge_key = k[u];
              sm.edge_row = row[u];
            }
        }
        __syncthreads();
        edge_key = sm.edge_key;
        edge_row = sm.edge_row;
        break;
      }
      if (shift == 0) {  // more than kSelRanked rows of one weight: the one of that rank, in order
        edge_key = prefix;
        in_order([&](int i, float x) { return i >= first && i < last && order_key(x) == prefix; },
                 [&](int at, int i, float) {
                   if (at == rank) sm.edge_row = i;
                 });
        __syncthreads();
        edge_row = sm.edge_row;
        break;
      }
    }
  }
  auto stays = [&](int i, float x) {
    if (L <= budget || i < first || i >= last) return true;
    const uint32_t k = order_key(x);
    return k > edge_key || (k == edge_key && i < edge_row);
  };
  in_order(stays, [&](int at, int i, float x) {
    if (at < keep) {  // (never past it: `keep` rows stay)
      kp[at] = i;
      wo[at] = x;
    }
  });
}

// The rows that stay, into another cache, by `kept`, 16 bytes a lane, in a grid over rows: a copy (32 x
// 12 caches, 512 of up to 2048 rows of 128 bytes, K and V, 91 MB, 17.3 us, 5.3 TB/s).
constexpr int kMoveThreads = 256, kMovePer = 4;
__global__ __launch_bounds__(kMoveThreads) void evict_gather_kernel(
    char* __restrict__ k_out, char* __restrict__ v_out, int* lens_out, const char* __restrict__ k,
    const char* __restrict__ v, const int* lens, const int* __restrict__ kept, int H, int max_len,
    int max_out, int budget, int row_log2) {
  const long long hrow = blockIdx.x;
  const char* src = (blockIdx.z ? v : k) + ((hrow * max_len) << row_log2);
  char* dst = (blockIdx.z ? v_out : k_out) + ((hrow * max_out) << row_log2);
  const int lanes_log2 = row_log2 - 4, lane = threadIdx.x & ((1 << lanes_log2) - 1);
  const int per = kMoveThreads >> lanes_log2;  // rows a pass
  const int r0 = blockIdx.y * per * kMovePer + (threadIdx.x >> lanes_log2);
  u32x4 x[kMovePer];
  int from[kMovePer];
#pragma unroll
  for (int i = 0; i < kMovePer; ++i) {
    const int r = r0 + i * per;
    from[i] = r < budget ? kept[hrow * budget + r] : -1;
  }
#pragma unroll
  for (int i = 0; i < kMovePer; ++i)
    if (from[i] >= 0) x[i] = ld_stream(src + ((long long)from[i] << row_log2) + 16 * lane);
#pragma unroll
  for (int i = 0; i < kMovePer; ++i)
    if (from[i] >= 0)
      *reinterpret_cast<u32x4*>(dst + ((long long)(r0 + i * per) << row_log2) + 16 * lane) = x[i];
  // (this kernel reads lens nowhere else: lens_out may be lens)
  if (threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && hrow % H == 0)
    lens_out[hrow / H] = min(clamp_len(lens[hrow / H], max_len), budget);
}

// The same within a cache: one workgroup per (sequence, head) and tensor, in passes of kInPlaceRows
// rows. A row moves down or stays (kept[r] >= r), so a pass writes only rows that earlier passes
// or itself have read. Rows that stay where they are are read too and not written: the 32 x 12 caches
// above take 15.4 us, and 8.5 where every cache is within its budget.
constexpr int kInPlaceThreads = 1024, kInPlacePer = 4;
__global__ __launch_bounds__(kInPlaceThreads) void evict_in_place_kernel(
    char* k, char* v, int* lens_out, const int* lens, const int* __restrict__ kept, int H,
    int max_len, int budget, int row_log2) {
  const long long hrow = blockIdx.x;
  if (threadIdx.x == 0 && blockIdx.z == 0 && hrow % H == 0)
    lens_out[hrow / H] = min(clamp_len(lens[hrow / H], max_len), budget);
  char* rows = (blockIdx.z ? v : k) + ((hrow * max_len) << row_log2);
  const int lanes_log2 = row_log2 - 4, lane = threadIdx.x & ((1 << lanes_log2) - 1);
  const int per = kInPlaceThreads >> lanes_log2, mine = threadIdx.x >> lanes_log2;
  for (int r0 = 0; r0 < budget; r0 += per * kInPlacePer) {
    u32x4 x[kInPlacePer];
    int from[kInPlacePer];
#pragma unroll
    for (int i = 0; i < kInPlacePer; ++i) {
      const int r = r0 + i * per + mine;
      from[i] = r < budget ? kept[hrow * budget + r] : -1;
    }
#pragma unroll
    for (int i = 0; i < kInPlacePer; ++i)
      if (from[i] >= 0)
        x[i] = *reinterpret_cast<const u32x4*>(rows + ((long long)from[i] << row_log2) + 16 * lane);
    wait_loads();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kInPlacePer; ++i) {
      const int r = r0 + i * per + mine;
      if (from[i] >= 0 && from[i] != r)
        *reinterpret_cast<u32x4*>(rows + ((long long)r << row_log2) + 16 * lane) = x[i];
    }
  }
}

}  // namespace

hipError_t launch_kv8_append_bf16(uint8_t* k8, uint8_t* v8, float* k_scale, float* v_scale,
                                  const bf16* k, const bf16* v, const HeadStrides64& ks,
                                  const HeadStrides64& vs, const int* lens, const int* counts,
                                  int n_seq, int H, int rows, int max_len, int D, int block,
                                  hipStream_t stream) {
  return launch_kv8_append_t<bf16>(k8, v8, k_scale, v_scale, k, v, ks, vs, lens, counts, n_seq, H,
                                   rows, max_len, D, block, stream);
}
hipError_t launch_kv8_append_f32(uint8_t* k8, uint8_t* v8, float* k_scale, float* v_scale,
                                 const float* k, const float* v, const HeadStrides64& ks,
                                 const HeadStrides64& vs, const int* lens, const int* counts,
                                 int n_seq, int H, int rows, int max_len, int D, int block,
                                 hipStream_t stream) {
  return launch_kv8_append_t<float>(k8, v8, k_scale, v_scale, k, v, ks, vs, lens, counts, n_seq, H,
                                    rows, max_len, D, block, stream);
}

size_t kv8_decode_workspace_bytes(int n_seq, int H, int max_len, int D) {
  const int c = D == 64 ? kv8_chunk_keys<64>() : kv8_chunk_keys<32>();
  const int nc = (max_len + c - 1) / c;
  return nc == 1 ? 0 : counter_bytes(n_seq, H) + partial_bytes(n_seq, H, nc, D);
}
template <typename T>
static hipError_t launch_kv8_decode_t(T* out, const T* q, const uint8_t* k8, const uint8_t* v8,
                               const float* k_scale, const float* v_scale, const int* lens,
                               int n_seq, int H, int max_len, int D, int block, float scale,
                               const Window* window, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
  if (D == 64)
    return launch_kv8_decode_d<T, 64>(out, q, k8, v8, k_scale, v_scale, lens, n_seq, H, max_len,
                                      block, scale, window, workspace, workspace_bytes, stream);
  if (D == 32)
    return launch_kv8_decode_d<T, 32>(out, q, k8, v8, k_scale, v_scale, lens, n_seq, H, max_len,
                                      block, scale, window, workspace, workspace_bytes, stream);
  return hipErrorInvalidValue;
}
hipError_t launch_kv8_decode_bf16(bf16* out, const bf16* q, const uint8_t* k8, const uint8_t* v8,
                                  const float* k_scale, const float* v_scale, const int* lens,
                                  int n_seq, int H, int max_len, int D, int block, float scale,
                                  const Window* window, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  return launch_kv8_decode_t<bf16>(out, q, k8, v8, k_scale, v_scale, lens, n_seq, H, max_len, D,
                                   block, scale, window, workspace, workspace_bytes, stream);
}
hipError_t launch_kv8_decode_f32(float* out, const float* q, const uint8_t* k8, const uint8_t* v8,
                                 const float* k_scale, const float* v_scale, const int* lens,
                                 int n_seq, int H, int max_len, int D, int block, float scale,
                                 const Window* window, void* workspace, size_t workspace_bytes,
                                 hipStream_t stream) {
  return launch_kv8_decode_t<float>(out, q, k8, v8, k_scale, v_scale, lens, n_seq, H, max_len, D,
                                    block, scale, window, workspace, workspace_bytes, stream);
}

size_t weights_decode_workspace_bytes(int n_seq, int H, int max_len, int D) {
  // fp32 chunks are the shorter ones: their count serves both element types
  const int c = D == 64 ? weights_chunk_keys<float, 64>() : weights_chunk_keys<float, 32>();
  const int nc = (max_len + c - 1) / c;
  return nc <= 2 ? 0 : sizeof(float) * (size_t)n_seq * H * ((size_t)nc * (D + 2) + max_len);
}
template <typename T>
static hipError_t launch_weights_decode_t(T* out, float* wout, const T* q, const T* kc, const T* vc,
                                   const float* win, const int* lens, int n_seq, int H,
                                   int max_len, int D, float scale, void* workspace,
                                   hipStream_t stream) {
  if (D == 64)
    return launch_weights_decode_d<T, 64>(out, wout, q, kc, vc, win, lens, n_seq, H, max_len,
                                          scale, workspace, stream);
  if (D == 32)
    return launch_weights_decode_d<T, 32>(out, wout, q, kc, vc, win, lens, n_seq, H, max_len,
                                          scale, workspace, stream);
  return hipErrorInvalidValue;
}
hipError_t launch_weights_decode_bf16(bf16* out, float* wout, const bf16* q, const bf16* kc,
                                      const bf16* vc, const float* win, const int* lens, int n_seq,
                                      int H, int max_len, int D, float scale, void* workspace,
                                      hipStream_t stream) {
  return launch_weights_decode_t<bf16>(out, wout, q, kc, vc, win, lens, n_seq, H, max_len, D,
                                       scale, workspace, stream);
}
hipError_t launch_weights_decode_f32(float* out, float* wout, const float* q, const float* kc,
                                     const float* vc, const float* win, const int* lens, int n_seq,
                                     int H, int max_len, int D, float scale, void* workspace,
                                     hipStream_t stream) {
  return launch_weights_decode_t<float>(out, wout, q, kc, vc, win, lens, n_seq, H, max_len, D,
                                        scale, workspace, stream);
}

hipError_t launch_kv_evict(void* k_out, void* v_out, float* wout, int* kept, int* lens_out,
                           const void* k, const void* v, const float* weights, const int* lens,
                           int n_seq, int H, int max_len, int max_out, int row_bytes, int budget,
                           int sinks, int recent, hipStream_t stream) {
  const unsigned rows = (unsigned)(n_seq * H);
  const int row_log2 = __builtin_ctz((unsigned)row_bytes);
  auto select = [&](auto threads, auto held) {
    evict_select_kernel<threads(), held()><<<rows, threads(), 0, stream>>>(
        kept, wout, weights, lens, H, max_len, max_out, budget, sinks, recent);
  };
  // 16 waves for long caches, up to 8192 rows in registers, while every workgroup has a CU to itself (8
  // -> 16: 8 x 12 caches of 4096 rows 21.0 -> 20.4 us, 2 x 3 of 8192 25.4 -> 20.6, 1 x 12 of 32768 46.1
  // -> 35.0; but 32 x 12 of 4096 39.7 -> 45.3, 64 x 12 of 8192 82.1 -> 94.3).
  constexpr std::integral_constant<int, 512> half;
  constexpr std::integral_constant<int, 1024> full;
  auto select_by = [&](auto threads) {
    if (max_len <= kSelHeld * threads())
      select(threads, std::true_type{});
    else
      select(threads, std::false_type{});
  };
  if (max_len > 2048 && rows <= (unsigned)device_cus())
    select_by(full);
  else
    select_by(half);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (k_out == k) {
    evict_in_place_kernel<<<dim3(rows, 1, 2), kInPlaceThreads, 0, stream>>>(
        static_cast<char*>(k_out), static_cast<char*>(v_out), lens_out, lens, kept, H, max_len,
        budget, row_log2);
  } else {
    const int per = (kMoveThreads * 16 / row_bytes) * kMovePer;
    const int most = budget < max_len ? budget : max_len;
    evict_gather_kernel<<<dim3(rows, (most + per - 1) / per, 2), kMoveThreads, 0, stream>>>(
        static_cast<char*>(k_out), static_cast<char*>(v_out), lens_out,
        static_cast<const char*>(k), static_cast<const char*>(v), lens, kept, H, max_len, max_out,
        budget, row_log2);
  }
  return hipGetLastError();
}

}  // namespace dadgpt
