// Picking tokens by given random numbers for gfx950: temperature, top-k, top-p, min-p and the draw, one
// workgroup a row and one launch.
//
// The filters all keep a head of the row's descending order, so most of a row need only be compared with
// a bound that no element which stays lies below. In turn: the largest logit; with top-p, the sum Z of all
// weights; the bound (top-k: the k-th largest of the threads' maxima, which k elements reach, or for a
// large k a guess from a sample, checked by counting; top-p: the logit of weight (1 - p) Z / vocab, as all
// elements below it together weigh less than (1 - p) Z; min-p: its own); the elements that reach it, at
// most 8192, into LDS; and there the cuts and the draw, each the search for the element at which a
// running sum (of ones or of weights, by logit or by index) crosses a target: a histogram over 1024
// buckets, the bucket of the crossing, and its few elements compared each with each. Rows with more
// candidates (a huge top-k, flat weights) search over the row itself, and the draw, as that of a row
// without filters, goes by the sums of the row's pieces in order.
//
// A pick must not depend on the order in which weights are added: they are computed in double (relative
// error below 1e-13) and held as multiples of 2^-44 of the largest one, in 64-bit integers, whose sums
// are exact in any order, histogram atomics among them. What that rounds off, 2^-45 a weight at
// random, moves a border by about 1e-11 of the sum for 50257 of them.
//
// Bound by one CU's operations on a row: two or three an element and pass, about 20 for a weight. The
// row (200 KB of fp32 for 50257 logits) comes from L2 after the first pass.
#include "common.hpp"
#include "lanes.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kPiece = 4 * kThreads;        // elements that the workgroup takes at a time, 4 a lane
constexpr int kMostPieces = (1 << 19) / kPiece + 1;
constexpr int kBuckets = kThreads;          // of a histogram: one for each thread to scan
constexpr int kFew = kThreads;              // elements of a bucket that are compared each with each
constexpr int kPerThread = 8, kList = kPerThread * kThreads;  // candidates
constexpr int kMostK = kThreads / 2;        // top-k by the threads' maxima
constexpr int kOne = 44;                    // weights are multiples of 2^-44
constexpr float kFaintest = 31.0f;          // e^-31 < 2^-44.7: weighs nothing
constexpr float kMostFinite = 3.4028234663852886e38f;

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

// Elements in descending order, ties by index: every one has a number of its own.
__device__ __forceinline__ u64 order_of(float x, int index) {
  return (u64)key_of(x) << 32 | (uint32_t)~index;
}

// x of lane l - n of a row of 16, 0 where there is none; of a row's last lane, for the rows after it.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ u64 dpp64(u64 x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
// Sum over the lanes up to and with this one.
__device__ __forceinline__ u64 wave_scan(u64 x) {
  x += dpp64<0x111>(x);  // row_shr:1, 2, 4, 8
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  x += dpp64<0x118>(x);
  x += dpp64<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += dpp64<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, lanes::dpp_u32<lanes::kQuadXor1>(x));
  x = max(x, lanes::dpp_u32<lanes::kQuadXor2>(x));
  x = max(x, lanes::dpp_u32<lanes::kHalfMirror>(x));
  x = max(x, lanes::dpp_u32<lanes::kMirror>(x));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}

struct Shared {
  u64 list[kList];                  // the candidates, as order_of
  u64 few[kFew], few_weight[kFew];  // a bucket's elements
  u64 weight[kBuckets];             // a histogram
  uint32_t count[kBuckets];
  u64 piece[kMostPieces * kWaves];  // sums of the waves' pieces, in the row's order
  double root[64];                  // 2^(i / 64)
  u64 wave_sum[2][kWaves];          // (in turn, so that one barrier a use is enough)
  uint32_t wave_max[2][kWaves];
  u64 found_above, found;
  uint32_t bucket, bucket_count, listed;
  int token;
};

// e^((x - top) / temperature), at most 1, to 1e-13: 2^(k / 64) from the table times a polynomial of the
// rest. As a double, or as a multiple of 2^-44. NaN and -inf weigh nothing.
struct Weigher {
  double top, per;  // per: 64 log2(e) / temperature
  const double* root;
  __device__ __forceinline__ void parts(float x, double& p, double& r, int& n) const {
    constexpr double kMagic = 0x1.8p52, kL = 0.69314718055994530942 / 64;
    const double t = fmax(((double)x - top) * per, -6400.0);
    const double m = t + kMagic, f = t - (m - kMagic);
    const int k = (int)__double_as_longlong(m);
    p = fma(f, kL * kL * kL * kL / 24, kL * kL * kL / 6);
    p = fma(f, p, kL * kL / 2);
    p = fma(f, p, kL);
    p = fma(f, p, 1.0);
    r = root[k & 63];
    n = k >> 6;
  }
  static __device__ __forceinline__ double scaled(double r, int n) {  // r 2^n for r in [1, 2)
    return __longlong_as_double(__double_as_longlong(r) + ((long long)n << 52));
  }
  __device__ __forceinline__ double exact(float x) const {
    double p, r;
    int n;
    parts(x, p, r, n);
    return p * scaled(r, n);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    double p, r;
    int n;
    parts(x, p, r, n);
    // (above 2^52 a double is an integer: the sum rounds there, and holds it in its low bits)
    const double s = fma(p, scaled(r, n + kOne), 0x1p52);
    return (u64)__double_as_longlong(s) & 0xfffffffffffffull;
  }
};

// Four neighbours as they lie in memory.
template <typename T>
struct Four;
template <>
struct Four<float> {
  f32x4 w;
  __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const f32x4*>(p); }
  __device__ __forceinline__ void set(int e, float x) { w[e] = x; }
  __device__ __forceinline__ float get(int e) const { return w[e]; }
};
template <>
struct Four<bf16> {
  u32x2 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const u32x2*>(p); }
  __device__ __forceinline__ void set(int e, bf16 x) {
    const uint32_t b = __builtin_bit_cast(uint16_t, x);
    w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | b << 16 : b;
  }
  __device__ __forceinline__ float get(int e) const {
    return e % 2 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
  }
};

// Element `index` of the row lies in lane (index + shift) / 4 of piece (index + shift) / kPiece, so that
// four neighbours are one aligned load wherever the row starts.
template <typename T>
struct Row {
  const T* row;
  int vocab, shift, pieces, tid, lane, wave;
  bool infinite;  // the largest logit is +inf: those count as 0, all others as -inf
  int turn_max = 0, turn_sum = 0;
  Shared& sm;

  __device__ __forceinline__ Row(const T* base, int n, Shared& shared)
      : row(base), vocab(n), shift((int)(reinterpret_cast<uintptr_t>(base) / sizeof(T) % 4)),
        pieces((n + shift + kPiece - 1) / kPiece), tid(threadIdx.x), lane(threadIdx.x & 63),
        wave(threadIdx.x >> 6), infinite(false), sm(shared) {}

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
  __device__ __forceinline__ float value(const Four<T>& x, int e) const {
    const float v = x.get(e);
    return !infinite ? v : v == __builtin_inff() ? 0.f : neg_inf();
  }
  // f(piece, the lane's four elements), N pieces at a time and the next N in flight meanwhile (a piece
  // past the end: -inf)
  template <int N, typename F>
  __device__ __forceinline__ void each_piece(F f) const {
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
      for (int i = 0; i < N; ++i) {
        const float v[4] = {value(x[i], 0), value(x[i], 1), value(x[i], 2), value(x[i], 3)};
        f(at + i, v);
      }
    }
  }
  __device__ __forceinline__ int index(int piece, int e) const {
    return piece * kPiece + 4 * tid + e - shift;
  }

  // The largest of a value from each thread.
  __device__ __forceinline__ uint32_t largest(uint32_t x) {
    uint32_t* to = sm.wave_max[turn_max ^= 1];
    x = wave_max(x);
    if (lane == 0) to[wave] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x = max(x, to[w]);
    return x;
  }

  // The sum of x over the threads before this one, and over all.
  __device__ __forceinline__ u64 before(u64 x, u64& all) {
    u64* to = sm.wave_sum[turn_sum ^= 1];
    const u64 in_wave = wave_scan(x);
    if (lane == 63) to[wave] = in_wave;
    __syncthreads();
    u64 sum = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) sum = all;
      all += to[w];
    }
    return sum + in_wave - x;
  }

  // The index at which the sum of measure(x, index) in the row's order reaches `target(sum of all)`,
  // which is above 0 and at most that sum.
  template <typename M, typename G>
  __device__ __forceinline__ int in_order(M measure, G target_of, u64& all) {
    each_piece<2>([&](int i, const float (&x)[4]) {
      u64 s = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += measure(x[e], index(i, e));
      s = wave_scan(s);
      if (lane == 63 && i < pieces) sm.piece[i * kWaves + wave] = s;
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
      sm.bucket = i;
      sm.found_above = at;
    }
    __syncthreads();
    const int hit = sm.bucket;
    if (wave == hit % kWaves) {  // this wave's piece: its lanes, then the lane's elements
      const int i = hit / kWaves;
      Four<T> x;
      load(x, i);
      u64 w[4], s = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += w[e] = measure(value(x, e), index(i, e));
      u64 to = sm.found_above + wave_scan(s);
      if (to >= target && to - s < target) {
        to -= s;
        int e = 0;
#pragma unroll
        for (int y = 0; y < 3; ++y)
          if (e == y && to + w[y] < target) to += w[y], ++e;
        sm.token = index(i, e);
      }
    }
    __syncthreads();
    return sm.token;
  }

  // The element at which the sum of weights, taken in descending order of the elements' numbers, reaches
  // target_of(sum of all); 0 where it does not. each(lo, hi, f) calls f(number, weight) for the
  // elements of those numbers that have a weight; no two have the same number.
  template <typename Each, typename G>
  __device__ __forceinline__ u64 search(Each each, u64 lo, u64 hi, G target_of) {
    u64 over = 0, target = 0;  // over: what lies above the current range
    while (true) {
      const float per = (float)kBuckets / ((float)(hi - lo) + 1.0f);
      auto bucket = [&](u64 k) { return min((int)((float)(hi - k) * per), kBuckets - 1); };
      sm.weight[tid] = 0;
      sm.count[tid] = 0;
      if (tid == 0) sm.bucket = kBuckets, sm.listed = 0;
      __syncthreads();
      each(lo, hi, [&](u64 k, u64 w) {
        const int b = bucket(k);
        atomicAdd(&sm.weight[b], w);
        atomicAdd(&sm.count[b], 1u);
      });
      __syncthreads();
      u64 all;
      const u64 w = sm.weight[tid], upto = over + before(w, all);
      if (target == 0) target = target_of(all);
      if (upto < target && upto + w >= target) {
        sm.bucket = tid;
        sm.found_above = upto;
        sm.bucket_count = sm.count[tid];
      }
      __syncthreads();
      const int b = sm.bucket;
      if (b == kBuckets) return 0;
      over = sm.found_above;
      const uint32_t n = sm.bucket_count;
      if (n <= kFew) {
        each(lo, hi, [&](u64 k, u64 weight) {
          if (bucket(k) == b) {
            const uint32_t at = atomicAdd(&sm.listed, 1u);
            sm.few[at] = k;
            sm.few_weight[at] = weight;
          }
        });
        __syncthreads();
        if (tid < n) {
          const u64 mine = sm.few[tid];
          u64 more = over;
          for (uint32_t i = 0; i < n; ++i)
            if (sm.few[i] > mine) more += sm.few_weight[i];
          if (more < target && more + sm.few_weight[tid] >= target) sm.found = mine;
        }
        __syncthreads();
        return sm.found;
      }
      // too many: the bucket's own range, from the largest and smallest of its numbers' halves
      uint32_t a = 0, z = 0;
      each(lo, hi, [&](u64 k, u64) {
        if (bucket(k) == b) a = max(a, (uint32_t)(k >> 32)), z = max(z, (uint32_t)(~k >> 32));
      });
      a = largest(a);
      z = ~largest(z);
      uint32_t c = 0, y = 0;
      each(lo, hi, [&](u64 k, u64) {
        if (bucket(k) == b) {
          if ((uint32_t)(k >> 32) == a) c = max(c, (uint32_t)k);
          if ((uint32_t)(k >> 32) == z) y = max(y, (uint32_t)~k);
        }
      });
      c = largest(c);
      y = ~largest(y);
      hi = (u64)a << 32 | c;
      lo = (u64)z << 32 | y;
    }
  }
};

// search's elements, N of them with every thread.
template <int N>
struct Elements {
  u64 number[N], weight[N];
  template <typename F>
  __device__ __forceinline__ void operator()(u64 lo, u64 hi, F f) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (weight[j] != 0 && number[j] >= lo && number[j] <= hi) f(number[j], weight[j]);
  }
};

// The smallest sum that reaches the share `p` of n, and the smallest above the share `u` of it.
__device__ __forceinline__ u64 reaching(float p, u64 n) {
  const double t = ceil((double)fmaxf(p, 0.f) * (double)n);
  return t < 1.0 ? 1 : (u64)t < n ? (u64)t : n;
}
__device__ __forceinline__ u64 exceeding(float u, u64 n) {
  const u64 t = (u64)((double)u * (double)n) + 1;
  return t < n ? t : n;
}

struct Settings {
  float p, min_p, u, temperature;
  int k;
};
struct Pick {
  int token;
  u64 all;  // the weights' sum that it was drawn from; 0: taken, not drawn
};

// Over the whole row; hi: the largest key.
template <typename T>
__device__ Pick pick_from_row(Row<T>& row, const Settings& s, const Weigher& weigh, uint32_t hi) {
  u64 cut = 1ull << 32;  // what stays: numbers from here on
  const u64 most = (u64)hi << 32 | 0xffffffffu;
  auto each = [&](auto weight) {
    return [&row, weight](u64 lo, u64 hi, auto f) {
      row.template each_piece<2>([&](int i, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 k = order_of(x[e], row.index(i, e));
          if (k >= lo && k <= hi) {
            const u64 w = weight(x[e]);
            if (w != 0) f(k, w);
          }
        }
      });
    };
  };
  if (s.k < row.vocab) {
    const u64 at = row.search(each([](float) { return u64(1); }), cut, most,
                              [&](u64) { return (u64)s.k; });
    cut = max(cut, at);
  }
  if (s.p < 1.0f) {
    const u64 faint = (u64)key_of((float)weigh.top - kFaintest * s.temperature) << 32;
    const u64 at = row.search(each([&](float x) { return weigh(x); }), max(cut, faint), most,
                              [&](u64 all) { return reaching(s.p, all); });
    cut = max(cut, at);
  }
  Pick pick;
  pick.token = row.in_order(
      [&](float x, int i) -> u64 {
        if (order_of(x, i) < cut) return 0;
        if (s.min_p > 0.f && weigh.exact(x) < (double)s.min_p) return 0;
        return weigh(x);
      },
      [&](u64 all) { return exceeding(s.u, all); }, pick.all);
  return pick;
}

// Among the n candidates in sm.list, which hold every element that can stay; z: the weights' sum that
// top-p goes by, 0 for that of the first k.
template <typename T>
__device__ Pick pick_from_list(Row<T>& row, const Settings& s, const Weigher& weigh, uint32_t hi, int n,
                               u64 z) {
  Shared& sm = row.sm;
  Elements<kPerThread> x;
  uint32_t low = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = row.tid + j * kThreads;
    x.number[j] = i < n ? sm.list[i] : 0;
    x.weight[j] = i < n ? 1 : 0;
    if (i < n) low = max(low, (uint32_t)(~x.number[j] >> 32));
  }
  const u64 most = (u64)hi << 32 | 0xffffffffu;
  u64 cut = (u64)~row.largest(low) << 32;
  if (s.k < n) cut = row.search(x, cut, most, [&](u64) { return (u64)s.k; });
  u64 sum = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    if (j * kThreads >= n) break;
    x.weight[j] = x.number[j] >= cut && j * kThreads + row.tid < n ? weigh(logit_of(x.number[j] >> 32)) : 0;
    sum += x.weight[j];
  }
  if (s.p < 1.0f) {
    if (z == 0) row.before(sum, z);
    cut = row.search(x, cut, most, [&](u64) { return reaching(s.p, z); });  // (0: not reached)
  }
  sum = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    if (j * kThreads >= n) break;
    if (x.number[j] < cut ||
        (s.min_p > 0.f && weigh.exact(logit_of(x.number[j] >> 32)) < (double)s.min_p))
      x.weight[j] = 0;
    x.number[j] = (uint32_t)x.number[j];  // ~index: the lowest first
    sum += x.weight[j];
  }
  Pick pick;
  row.before(sum, pick.all);
  const u64 at = row.search(x, (uint32_t)~(row.vocab - 1), 0xffffffffu,
                            [&](u64) { return exceeding(s.u, pick.all); });
  pick.token = (int)~(uint32_t)at;
  return pick;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(
    int* __restrict__ tokens, float* __restrict__ probs, const T* __restrict__ logits, long long ld,
    int vocab, const SampleSettings set) {
  __shared__ Shared sm;
  const int r = blockIdx.x;
  const T* base = logits + r * ld;
  Row<T> row(base, vocab, sm);
  const int tid = row.tid;

  Settings s;
  s.temperature = set.temperature == nullptr ? 1.0f : set.temperature[r];
  s.k = set.top_k == nullptr ? 0 : set.top_k[r];
  s.p = set.top_p == nullptr ? 1.0f : set.top_p[r];
  s.min_p = set.min_p == nullptr ? 0.0f : set.min_p[r];
  s.u = set.uniforms[r];
  s.u = s.u > 0.f ? s.u : 0.f;
  if (!(s.temperature > 0.f) || s.min_p > 1.0f) s.temperature = 1.0f, s.k = 1;  // the first largest
  if (s.k <= 0 || s.k > vocab) s.k = vocab;
  if (!(s.p < 1.0f)) s.p = 1.0f;
  if (!(s.min_p > 0.f)) s.min_p = 0.f;
  if (tid < 64) sm.root[tid] = exp2(tid / 64.0);

  float mine = neg_inf();
  row.template each_piece<4>([&](int, const float (&x)[4]) {
    mine = fmaxf(fmaxf(fmaxf(fmaxf(mine, x[0]), x[1]), x[2]), x[3]);
  });
  uint32_t hi = row.largest(key_of(mine));
  auto answer = [&](int token, float prob) {
    if (tid == 0) {
      tokens[r] = token;
      if (probs != nullptr) probs[r] = prob;
    }
  };
  if (hi == 0) return answer(-1, 0.f);  // nothing to pick
  if (logit_of(hi) == __builtin_inff()) {
    row.infinite = true;
    mine = mine == __builtin_inff() ? 0.f : neg_inf();
    hi = key_of(0.f);
  }
  const float top = logit_of(hi);
  if (s.k == 1) {
    uint32_t first = 0;  // ~index
    if (mine == top)     // (only some threads: their elements once more)
      row.template each_piece<2>([&](int i, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] == top) first = max(first, (uint32_t)~row.index(i, e));
      });
    return answer((int)~row.largest(first), 1.0f);
  }

  const Weigher weigh{top, 64 * 1.4426950408889634074 / (double)s.temperature, sm.root};
  // A logit that every element of weight w or more reaches: that of half of it, and 2^-22 lower, which is
  // more than the logarithm's error and its rounding to fp32.
  auto logit_at = [&](double w) {
    const double x = (double)top + log(0.5 * w) * (double)s.temperature;
    return (float)(x - fabs(x) * 0x1p-22);
  };
  // The bound, as a logit: every element that can stay reaches it.
  const u64 most = (u64)hi << 32 | 0xffffffffu;
  float bound = neg_inf();
  u64 z = 0;
  bool bounded = vocab <= kList;
  if (!bounded && s.k < vocab) {
    if (s.k <= kMostK) {
      // (fewer threads with an element than k: 0, no bound)
      const Elements<1> x{{order_of(mine, tid)}, {mine > neg_inf() ? u64(1) : 0}};
      const uint32_t low = ~row.largest(x.weight[0] != 0 ? ~key_of(mine) : 0u);
      const u64 at = row.search(x, (u64)low << 32, most, [&](u64) { return (u64)s.k; });
      if (at != 0) bound = logit_of((uint32_t)(at >> 32));
      bounded = true;
    } else if (s.k <= kList * 2 / 3) {
      // one piece from the middle: a tenth more of it than k's share, and three standard deviations
      Four<T> four;
      row.load(four, row.pieces / 2);
      Elements<4> x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = row.value(four, e);
        x.number[e] = order_of(v, 4 * tid + e);
        x.weight[e] = v > neg_inf() ? 1 : 0;
      }
      const float share = 1.1f * (float)s.k * (float)kPiece / (float)vocab;
      const u64 at = row.search(x, 0, most, [&](u64) { return (u64)(share + 3.0f * sqrtf(share)); });
      if (at != 0) bound = logit_of((uint32_t)(at >> 32));
      bounded = at != 0;
    }
  } else if (!bounded && s.p < 1.0f) {
    u64 sum = 0;
    row.template each_piece<2>([&](int, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += weigh(x[e]);
    });
    row.before(sum, z);
    bound = logit_at((1.0 - (double)fmaxf(s.p, 0.f)) * (double)z / 0x1p44 / vocab);
    bounded = true;
  }
  // (top-p after top-k goes by the weights of the first k, also of those below min-p; after no top-k by Z,
  // which is known unless everything is a candidate)
  if (s.min_p > 0.f && !(s.p < 1.0f && z == 0)) {
    bound = fmaxf(bound, logit_at(s.min_p));
    bounded = true;
  }
  Pick pick;
  bool picked = false;
  if (bounded) {
    bound = fmaxf(bound, -kMostFinite);
    if (tid == 0) sm.listed = 0;
    __syncthreads();
    row.template each_piece<4>([&](int i, const float (&x)[4]) {
      if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= bound) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] >= bound) {
            const uint32_t at = atomicAdd(&sm.listed, 1u);
            if (at < (uint32_t)kList) sm.list[at] = order_of(x[e], row.index(i, e));
          }
      }
    });
    __syncthreads();
    const int n = (int)sm.listed;
    // (by the sample, k elements at least; otherwise the list holds what stays by its bound)
    if (n <= kList && (n >= s.k || s.k <= kMostK || s.k == vocab || vocab <= kList)) {
      pick = pick_from_list(row, s, weigh, hi, n, z);
      picked = true;
    }
    __syncthreads();
  }
  if (!picked) pick = pick_from_row(row, s, weigh, hi);
  Four<T> x;
  x.set(0, base[pick.token]);
  answer(pick.token, (float)(weigh.exact(row.value(x, 0)) * 0x1p44 / (double)pick.all));
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
