// Picking tokens by given random numbers for gfx950: temperature, top-k, top-p, min-p and the draw, one
// workgroup a row and one launch, with no sort.
//
// The filters all keep a head of the row's descending order, so what stays is known by a cut: the
// smallest logit that stays, and how many of its ties do. Selecting it: a histogram over 1024 buckets
// of equal width below the maximum, of counts (top-k) or of weights (top-p); the bucket in which the
// running sum crosses the target; and the crossing among the few elements of that bucket by comparing
// each with each. The draw needs sums in the vocabulary's order: one for each wave's piece of a row, then
// the piece in which the target lies.
//
// A pick must not depend on the order in which weights are added: they are computed in double (relative
// error below 1e-14) and held as multiples of 2^-44 of the largest one, in 64-bit integers, whose sums
// are exact in any order, histogram atomics among them. What that rounds off, 2^-45 a weight at
// random, moves a border by about 1e-11 of the sum for 50257 of them.
//
// Bound by one CU's work on a row: four or five passes over it (200 KB of fp32 for 50257 logits, from L2
// after the first), and the exponentials in double (about 16 operations each), which are computed for
// what is still kept only.
#include "common.hpp"
#include "lanes.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kPiece = 4 * kThreads;        // elements that the workgroup takes at a time, 4 a lane
constexpr int kMostPieces = (1 << 19) / kPiece + 1;
constexpr int kBuckets = kThreads;          // of a histogram: one for each thread to scan
constexpr int kList = kThreads;                 // elements of a bucket that are compared each with each
constexpr int kOne = 44;                    // weights are multiples of 2^-44
constexpr float kFaintest = 31.0f;          // e^-31 < 2^-44.7: weighs nothing

typedef unsigned long long u64;

// Keys order as the logits do; 0 is what is never picked: NaN, -inf, past the row's end.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > neg_inf())) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as +0
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kInfKey = 0xff800000u;  // +inf's

// e^z for z <= 0, to 1e-14: 2^n times the series of e^r, |r| <= ln 2 / 2, to its 11th power.
__device__ __forceinline__ double exp_series(double z, int* exponent) {
  constexpr double kLog2e64 = 1.4426950408889634074, kLn2_64 = 0.69314718055994530942;
  const double t = fmax(z * kLog2e64, -100.0), n = __builtin_rint(t);
  const double r = (t - n) * kLn2_64;
  double p = 1.0 / 39916800;
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  *exponent = (int)n;
  return fma(p, r, 1.0);
}
__device__ __forceinline__ double two_to(int n) {
  return __longlong_as_double((long long)(n + 1023) << 52);
}

template <typename X>
__device__ __forceinline__ X wave_scan(X x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const X y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

struct Shared {
  u64 weight[kBuckets];
  uint32_t count[kBuckets];
  uint32_t list[kList];
  u64 list_weight[kList];
  u64 piece[kMostPieces * kWaves];  // sums of the waves' pieces, in the row's order
  u64 wave_sum[kWaves];
  uint32_t wave_a[kWaves], wave_b[kWaves];
  u64 found_above, found_within;
  uint32_t found, found_count, listed;
  int token;
};

// Element `index` of the row lies in lane (index + shift) / 4 of piece (index + shift) / kPiece, so that
// four neighbours are one aligned load wherever the row starts.
template <typename T>
struct Four;
template <>
struct Four<float> {
  f32x4 w;
  __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const f32x4*>(p); }
  __device__ __forceinline__ void set(int e, float x) { w[e] = x; }
  __device__ __forceinline__ uint32_t key(int e) const { return key_of(w[e]); }
};
template <>
struct Four<bf16> {
  u32x2 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const u32x2*>(p); }
  __device__ __forceinline__ void set(int e, bf16 x) {
    const uint32_t b = __builtin_bit_cast(uint16_t, x);
    w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | b << 16 : b;
  }
  __device__ __forceinline__ uint32_t key(int e) const {
    return key_of(e % 2 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]));
  }
};

template <typename T>
struct Row {
  const T* row;
  int vocab, shift, pieces, tid, lane, wave;
  Shared& sm;

  __device__ __forceinline__ Row(const T* base, int n, Shared& shared)
      : row(base), vocab(n), shift((int)(reinterpret_cast<uintptr_t>(base) / sizeof(T) % 4)),
        pieces((n + shift + kPiece - 1) / kPiece), tid(threadIdx.x), lane(threadIdx.x & 63),
        wave(threadIdx.x >> 6), sm(shared) {}

  __device__ __forceinline__ void load(Four<T>& x, int piece) const {
    const int at = piece * kPiece + 4 * tid - shift;
    if (at >= 0 && at + 4 <= vocab) {
      x.load(row + at);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x.set(e, at + e >= 0 && at + e < vocab ? row[at + e] : static_cast<T>(neg_inf()));
    }
  }
  // f(piece, keys of the lane's four elements), the next pieces in flight meanwhile. The row comes from
  // L2 after the first pass: kept in registers, it leaves too few for the passes (a quarter of it in
  // scratch at 50257 elements), and LDS holds no more than 30000 fp32 elements.
  template <typename F>
  __device__ __forceinline__ void each_piece(F f) {
    constexpr int N = 2;
    Four<T> next[N];
#pragma unroll
    for (int i = 0; i < N; ++i) load(next[i], i);
    for (int at = 0; at < pieces; at += N) {
      Four<T> x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = next[i];
      if (at + N < pieces) {
#pragma unroll
        for (int i = 0; i < N; ++i) load(next[i], at + N + i);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {  // (pieces past the end: all 0)
        const uint32_t k[4] = {x[i].key(0), x[i].key(1), x[i].key(2), x[i].key(3)};
        f(at + i, k);
      }
    }
  }
  __device__ __forceinline__ int index(int piece, int e) const {
    return piece * kPiece + 4 * tid + e - shift;
  }

  // The largest and the smallest of one value from each thread (0 left out of the smallest).
  __device__ __forceinline__ void extremes(uint32_t& most, uint32_t& least) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
      least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    }
    if (lane == 0) sm.wave_a[wave] = most, sm.wave_b[wave] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      most = max(most, sm.wave_a[w]);
      least = min(least, sm.wave_b[w]);
    }
    __syncthreads();
  }

  // The sum of x over the threads before this one, and over all.
  __device__ __forceinline__ u64 before(u64 x, u64& all) {
    const u64 in_wave = wave_scan(x, lane);
    if (lane == 63) sm.wave_sum[wave] = in_wave;
    __syncthreads();
    u64 sum = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) sum = all;
      all += sm.wave_sum[w];
    }
    __syncthreads();
    return sum + in_wave - x;
  }

  // The index at which the sum of measure(key, index) in the row's order reaches `target(sum of all)`,
  // which is above 0 and at most that sum.
  template <typename M, typename G>
  __device__ __forceinline__ int in_order(M measure, G target_of, u64& all) {
    each_piece([&](int i, const uint32_t (&k)[4]) {
      u64 s = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += measure(k[e], index(i, e));
#pragma unroll
      for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d, 64);
      if (lane == 0 && i < pieces) sm.piece[i * kWaves + wave] = s;
    });
    __syncthreads();
    const int n = pieces * kWaves, per = (n + kThreads - 1) / kThreads, first = tid * per;
    u64 mine = 0;
    for (int i = first; i < min(n, first + per); ++i) mine += sm.piece[i];
    u64 at = before(mine, all);
    const u64 target = target_of(all);
    if (at < target && at + mine >= target) {
      int i = first;
      while (at + sm.piece[i] < target) at += sm.piece[i++];
      sm.found = i;
      sm.found_above = at;
    }
    __syncthreads();
    const int hit = sm.found;
    if (wave == hit % kWaves) {  // this wave's piece: its lanes, then the lane's elements
      const int i = hit / kWaves;
      Four<T> x;
      load(x, i);
      const uint32_t k[4] = {x.key(0), x.key(1), x.key(2), x.key(3)};
      u64 w[4], s = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += w[e] = measure(k[e], index(i, e));
      u64 to = sm.found_above + wave_scan(s, lane);
      if (to >= target && to - s < target) {
        to -= s;
        int e = 0;
#pragma unroll
        for (int x = 0; x < 3; ++x)
          if (e == x && to + w[x] < target) to += w[x], ++e;
        sm.token = index(i, e);
      }
    }
    __syncthreads();
    return sm.token;
  }

  // The key at which the sum of measure(key, index), taken in descending order of the keys, reaches
  // target_of(sum of all): above = the sum of the larger keys', `ties` elements have the key itself.
  // measure is 0 for what is left out; lo and hi bound the keys that it is not 0 for, and `width` is
  // the range below hi's logit over which the first histogram is spread.
  template <typename M, typename G>
  __device__ __forceinline__ uint32_t descending(M measure, G target_of, uint32_t lo, uint32_t hi,
                                                 float width, u64& above, uint32_t& ties,
                                                 u64& target) {
    const float top = logit_of(hi), per = (float)kBuckets / width;
    bool by_value = width > 0.f && per < __builtin_inff();
    u64 over = 0;  // what lies above the current range
    target = 0;
    while (true) {
      const uint32_t step = (hi - lo) / kBuckets + 1;
      auto bucket = [&](uint32_t k) {
        if (by_value) return (int)fminf((top - logit_of(k)) * per, (float)(kBuckets - 1));
        return (int)((hi - k) / step);
      };
      sm.weight[tid] = 0;
      sm.count[tid] = 0;
      if (tid == 0) sm.listed = 0;
      __syncthreads();
      each_piece([&](int i, const uint32_t (&k)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k[e] >= lo && k[e] <= hi) {
            const u64 m = measure(k[e], index(i, e));
            if (m != 0) {
              const int b = bucket(k[e]);
              atomicAdd(&sm.weight[b], m);
              atomicAdd(&sm.count[b], 1u);
            }
          }
      });
      __syncthreads();
      u64 all;
      const u64 w = sm.weight[tid], upto = over + before(w, all);
      if (target == 0) target = target_of(all);
      if (upto < target && upto + w >= target) {
        sm.found = tid;
        sm.found_above = upto;
        sm.found_count = sm.count[tid];
      }
      __syncthreads();
      const int b = sm.found;
      over = sm.found_above;
      const uint32_t n = sm.found_count;
      if (n <= kList) {
        each_piece([&](int i, const uint32_t (&k)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] >= lo && k[e] <= hi && bucket(k[e]) == b) {
              const u64 m = measure(k[e], index(i, e));
              if (m != 0) {
                const uint32_t at = atomicAdd(&sm.listed, 1u);
                sm.list[at] = k[e];
                sm.list_weight[at] = m;
              }
            }
        });
        __syncthreads();
        if (tid < n) {
          const uint32_t mine = sm.list[tid];
          u64 more = over, same = 0;
          uint32_t equal = 0;
          for (uint32_t i = 0; i < n; ++i) {
            const uint32_t k = sm.list[i];
            const u64 m = sm.list_weight[i];
            if (k > mine) more += m;
            if (k == mine) same += m, ++equal;
          }
          if (more < target && more + same >= target) {  // (every tie answers the same)
            sm.found = mine;
            sm.found_above = more;
            sm.found_count = equal;
          }
        }
        __syncthreads();
        above = sm.found_above;
        ties = sm.found_count;
        return sm.found;
      }
      // too many: the bucket's own range of keys, in equal steps of keys from here on
      uint32_t most = 0, least = 0xffffffffu;
      each_piece([&](int i, const uint32_t (&k)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k[e] >= lo && k[e] <= hi && bucket(k[e]) == b && measure(k[e], index(i, e)) != 0)
            most = max(most, k[e]), least = min(least, k[e]);
      });
      extremes(most, least);
      hi = most;
      lo = least;
      by_value = false;
      if (lo == hi) {  // all ties
        above = over;
        ties = n;
        return hi;
      }
    }
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(
    int* __restrict__ tokens, float* __restrict__ probs, const T* __restrict__ logits, long long ld,
    int vocab, const SampleSettings set) {
  __shared__ Shared sm;
  const int r = blockIdx.x;
  const T* base = logits + r * ld;
  Row<T> row(base, vocab, sm);

  float temperature = set.temperature == nullptr ? 1.0f : set.temperature[r];
  int k = set.top_k == nullptr ? 0 : set.top_k[r];
  const float p = set.top_p == nullptr ? 1.0f : set.top_p[r];
  const float min_p = set.min_p == nullptr ? 0.0f : set.min_p[r];
  const float given = set.uniforms[r];
  if (!(temperature > 0.f) || min_p > 1.0f) temperature = 1.0f, k = 1;  // the first largest
  if (k <= 0 || k > vocab) k = vocab;

  uint32_t hi = 0, lo = 0xffffffffu;
  row.each_piece([&](int, const uint32_t (&key)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hi = max(hi, key[e]);
      if (key[e] != 0) lo = min(lo, key[e]);
    }
  });
  row.extremes(hi, lo);
  if (hi == 0) {  // nothing to pick
    if (row.tid == 0) {
      tokens[r] = -1;
      if (probs != nullptr) probs[r] = 0.f;
    }
    return;
  }
  if (hi == kInfKey) lo = hi;  // +inf alone counts
  const double top = hi == kInfKey ? 0.0 : (double)logit_of(hi), per = 1.0 / (double)temperature;
  const float range = hi == lo ? 0.f : logit_of(hi) - logit_of(lo);

  // e^z and its multiple of 2^-44
  auto exact = [&](uint32_t key) {
    if (key == hi) return 1.0;
    int n;
    const double e = exp_series(((double)logit_of(key) - top) * per, &n);
    return e * two_to(n);
  };
  auto weigh = [&](uint32_t key) -> u64 {
    int n;
    const double e = exp_series(((double)logit_of(key) - top) * per, &n);
    // (above 2^52 a double is an integer: the sum rounds there, and holds it in its low bits)
    const double s = fma(e, two_to(n + kOne), 0x1p52);
    return key == hi ? 1ull << kOne : (u64)__double_as_longlong(s) & 0xfffffffffffffull;
  };

  // What stays: keys above `cut`, and those equal to it up to index `last`.
  uint32_t cut = lo;
  int last = vocab;
  u64 all;
  auto stays = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= last); };
  // (of the cut's ties that stayed so far, the first `need`)
  auto cut_ties = [&](u64 need, uint32_t ties) {
    if (need >= ties) return;
    last = row.in_order(
        [&](uint32_t key, int i) -> u64 { return key == cut && i <= last ? 1 : 0; },
        [&](u64) { return need; }, all);
  };
  if (k == 1) {
    cut = hi;
    last = row.in_order([&](uint32_t key, int) -> u64 { return key == hi ? 1 : 0; },
                        [](u64) -> u64 { return 1; }, all);
    if (row.tid == 0) {
      tokens[r] = last;
      if (probs != nullptr) probs[r] = 1.0f;
    }
    return;
  }
  if (k < vocab) {
    u64 above, target;
    uint32_t ties;
    const uint32_t old = cut;
    cut = row.descending([&](uint32_t key, int) -> u64 { return key >= old ? 1 : 0; },
                         [&](u64 n) -> u64 { return n < (u64)k ? n : (u64)k; }, lo, hi, range, above,
                         ties, target);
    cut_ties(target - above, ties);
  }
  if (p < 1.0f) {
    u64 above, target;
    uint32_t ties;
    const uint32_t old = cut;
    const int old_last = last;
    cut = row.descending(
        [&](uint32_t key, int i) -> u64 {
          return key > old || (key == old && i <= old_last) ? weigh(key) : 0;
        },
        [&](u64 n) -> u64 {
          const double t = ceil((double)fmaxf(p, 0.f) * (double)n);
          return t < 1.0 ? 1 : (u64)t < n ? (u64)t : n;
        },
        cut, hi, fminf(range, kFaintest * temperature), above, ties, target);
    if (cut != old) last = vocab;
    const u64 w = weigh(cut);
    cut_ties((target - above + w - 1) / w, ties);
  }
  const float floor_p = min_p > 0.f ? min_p : 0.f;
  auto measure = [&](uint32_t key, int i) -> u64 {
    if (!stays(key, i)) return 0;
    if (floor_p > 0.f && exact(key) < (double)floor_p) return 0;
    return weigh(key);
  };
  const float u = given > 0.f ? given : 0.f;
  const int token = row.in_order(
      measure,
      [&](u64 n) -> u64 {  // the first sum above u n
        const u64 t = (u64)((double)u * (double)n) + 1;
        return t < n ? t : n;
      },
      all);
  if (row.tid == 0) {
    tokens[r] = token;
    if (probs != nullptr) {
      const uint32_t key = key_of(static_cast<float>(base[token]));
      probs[r] = (float)(exact(key) * two_to(kOne) / (double)all);
    }
  }
}

template <typename T>
hipError_t launch_sample_t(int* tokens, float* probs, const T* logits, long long ld, int rows,
                           int vocab, const SampleSettings& set, hipStream_t stream) {
  sample_kernel<T><<<rows, kThreads, 0, stream>>>(tokens, probs, logits, ld, vocab, set);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample_bf16(int* tokens, float* probs, const bf16* logits, long long ld, int rows,
                              int vocab, const SampleSettings& settings, hipStream_t stream) {
  return launch_sample_t<bf16>(tokens, probs, logits, ld, rows, vocab, settings, stream);
}
hipError_t launch_sample_f32(int* tokens, float* probs, const float* logits, long long ld, int rows,
                             int vocab, const SampleSettings& settings, hipStream_t stream) {
  return launch_sample_t<float>(tokens, probs, logits, ld, rows, vocab, settings, stream);
}

}  // namespace dadgpt
