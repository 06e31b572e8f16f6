// Picking tokens by given random numbers for gfx950: temperature, top-k, top-p, min-p and the draw, one
// workgroup a row and one launch.
//
// The filters all keep a head of the row's descending order. In turn: the largest logit; a histogram
// below it of counts (top-k) or counts and weights (top-p), which gives the bucket where the running
// sum crosses the target; the indexes of the elements down to that bucket into LDS; and among those the
// cuts and the draw, each the search for the element at which a running sum (of ones or of weights, by
// logit or by index) crosses its target. Up to 64 elements one wave adds up for each lane what lies above its own; more are
// searched by a finer histogram and the few elements of its bucket. Rows that keep more than 8192
// elements search over the row itself, and the draw there, as that of a row without filters, goes by
// the sums of the waves' stretches of the row.
//
// The histogram has 256 buckets, so that a bucket of a row of usual spread fits the list (with 64 of
// them, flat rows of 50257 had 9000 to 16000 elements in the one that top-p ends in, and needed a second
// histogram of it), and 8 columns, one for every eighth lane: however the logits are spread, eight lanes
// of an atomic meet in a bank at most. (With one column, 785 wave-wide pairs of atomics on 50257 logits of
// a usual spread took 45 us.)
//
// A pick must not depend on the order in which weights are added: they are computed in double (relative
// error below 1e-13) and held as multiples of 2^-44 of the largest one, in 64-bit integers, whose sums
// are exact in any order, histogram atomics among them. What that rounds off, 2^-45 a weight at
// random, moves a border by about 1e-11 of the sum for 50257 of them.
//
// Bound by one CU's operations on a row: two or three an element and pass, about 20 for a weight, and
// between passes by barriers and chains in LDS. The row (200 KB of fp32 for 50257 logits) comes from L2
// after the first pass. 50257 logits, us: one row, top-k of 40, 18 to 19; 32 rows of all kinds 70 to 84; 512
// rows of bf16 with top-p 151 to 159, of fp32 143. 32 rows of one kind: no filter 25, top-k of 40 20, of 5000
// 43, top-p of 0.9 44 (spread of 4) to 95 (of 0.5: 40000 tokens stay), and 320 with all logits equal.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kLevels = 256, kColumns = 8;  // buckets of the row's histogram, copies of each
constexpr int kBuckets = kThreads;          // of a search's: one for each thread to scan
constexpr int kFew = kThreads;              // elements of a bucket that are compared each with each
constexpr int kPerThread = 16, kList = kPerThread * kThreads;  // candidates
constexpr int kOne = 44;                    // weights are multiples of 2^-44
// Where the last bucket by weight begins, in temperatures below the largest logit. e^-31 is 0.61 units of
// 2^-44, which rounds to 1: every logit in a bucket above the last weighs at least a unit, so that counts (of
// those that weigh something) and lists (of all in a bucket) agree. From e^-31.19 on weights round to 0.
constexpr float kFaintest = 31.0f;

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
// Sum over the lanes of its row of 16, and over all, up to and with this one.
__device__ __forceinline__ u64 row_scan(u64 x) {
  x += dpp64<0x111>(x);  // row_shr:1, 2, 4, 8
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  x += dpp64<0x118>(x);
  return x;
}
// The sum over lanes l - 7 to l of a row.
__device__ __forceinline__ u64 sum_of_8(u64 x) {
  x += dpp64<0x111>(x);
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  return x;
}
__device__ __forceinline__ u64 wave_scan(u64 x) {
  x = row_scan(x);
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
  int list[kList];                  // the candidates' indexes
  u64 few[kFew], few_weight[kFew];  // a bucket's elements
  union {
    struct {
      u64 weight[kLevels][kColumns];      // the row's histogram
      uint32_t count[kLevels][kColumns];
    } row;
    struct {
      u64 weight[kBuckets];         // a search's
      uint32_t count[kBuckets];
    } search;
  };
  u64 level_weight[kLevels];
  uint32_t level_count[kLevels];
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
  __device__ __forceinline__ void set(int e, float x) { w[e] = x; }  // (in the order of e)
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

// The row in stretches, one for each wave, in order; a wave goes through its own in pieces of 256
// elements, four neighbours a lane. Element `index` is number index + shift of them, so that four
// neighbours are one aligned load wherever the row starts. NP > 0: a row of at most NP pieces a wave,
// which stays in registers for the passes over all of it; 0: they read it again (from L2).
template <typename T, int NP>
struct Row {
  const T* row;
  Four<T> kept[NP > 0 ? NP : 1];
  int vocab, shift, pieces, first, tid, lane, wave;
  bool infinite;  // the largest logit is +inf: those count as 0, all others as -inf
  int turn_max = 0, turn_sum = 0;
  Shared& sm;

  __device__ __forceinline__ Row(const T* base, int n, Shared& shared)
      : row(base), vocab(n), shift((int)(reinterpret_cast<uintptr_t>(base) / sizeof(T) % 4)),
        pieces((n + shift + 256 * kWaves - 1) / (256 * kWaves)), tid(threadIdx.x),
        lane(threadIdx.x & 63), wave(threadIdx.x >> 6), infinite(false), sm(shared) {
    first = wave * pieces * 256 + 4 * lane - shift;
#pragma unroll
    for (int i = 0; i < NP; ++i) load(kept[i], i);
  }

  __device__ __forceinline__ void load(Four<T>& x, int piece) const {
    const int at = index(piece, 0);
    if (piece < pieces && at >= 0 && at + 4 <= vocab) {
      x.load(row + at);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x.set(e, piece < pieces && at + e >= 0 && at + e < vocab ? row[at + e]
                                                                : static_cast<T>(neg_inf()));
    }
  }
  __device__ __forceinline__ int index(int piece, int e) const { return first + piece * 256 + e; }
  __device__ __forceinline__ float value(const Four<T>& x, int e) const {
    const float v = x.get(e);
    return !infinite ? v : only_inf(v);
  }
  static __device__ __forceinline__ float only_inf(float v) {
    return v == __builtin_inff() ? 0.f : neg_inf();
  }
  __device__ __forceinline__ void set_infinite() {
    infinite = true;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Four<T> x = kept[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) kept[i].set(e, static_cast<T>(only_inf(x.get(e))));
    }
  }
  // f(piece, the lane's four elements), N pieces at a time and the next N in flight meanwhile
  template <int N, typename F>
  __device__ __forceinline__ void each_again(F f) const {
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
  // (pieces past the end, there for the sake of whole Ns, are all -inf.) AGAIN: from memory, where the
  // registers are needed for other things
  template <bool AGAIN, typename F>
  __device__ __forceinline__ void each_piece(F f) const {
    if constexpr (NP > 0 && !AGAIN) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float v[4] = {kept[i].get(0), kept[i].get(1), kept[i].get(2), kept[i].get(3)};
        f(i, v);
      }
    } else {
      each_again<4>(f);
    }
  }

  // The number (order_of) of a listed element.
  __device__ __forceinline__ u64 number_of(int i) const {
    Four<T> x;
    x.set(0, row[i]);
    return order_of(value(x, 0), i);
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
  template <bool AGAIN, typename M, typename G>
  __device__ __forceinline__ int in_order(M measure, G target_of, u64& all) {
    u64 mine = 0;
    each_piece<AGAIN>([&](int i, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += measure(x[e], index(i, e));
    });
    u64* to = sm.wave_sum[turn_sum ^= 1];
    const u64 stretch = wave_scan(mine);
    if (lane == 63) to[wave] = stretch;
    __syncthreads();
    u64 at = 0, sum = 0, my_sum = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) at = all, my_sum = to[w];
      all += to[w];
    }
    sum = at + my_sum;
    const u64 target = target_of(all);
    if (at < target && sum >= target) {  // this wave's stretch: its pieces, lanes, the lane's elements
      for (int i = 0; i < pieces; ++i) {
        Four<T> x;
        load(x, i);
        u64 w[4], s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s += w[e] = measure(value(x, e), index(i, e));
        const u64 upto = at + wave_scan(s);
        if (__builtin_amdgcn_ballot_w64(upto >= target) == 0) {
          at = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(upto >> 32), 63) << 32 |
               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)upto, 63);
          continue;
        }
        if (upto >= target && upto - s < target) {
          u64 x = upto - s;
          int e = 0;
#pragma unroll
          for (int y = 0; y < 3; ++y)
            if (e == y && x + w[y] < target) x += w[y], ++e;
          sm.token = index(i, e);
        }
        break;
      }
    }
    __syncthreads();
    return sm.token;
  }

  // A histogram over buckets bucket_of(x) (kLevels: none), descending, of counts and measure(x, index)
  // (0: not counted). The bucket at which the sum of measures (and `over`) reaches target_of(sum of
  // all): its number (kLevels: nowhere), the elements in it and down to its end, and the sums of all
  // and of what lies above it.
  struct Level {
    int bucket;
    uint32_t own, count;
    u64 all, over;
  };
  __device__ __forceinline__ static u64 lane_of(u64 x, int i) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, i);
  }
  template <bool WEIGHTS, bool AGAIN, typename B, typename M, typename G>
  __device__ __forceinline__ Level histogram(B bucket_of, M measure, G target_of, u64 over = 0) {
    for (int i = tid; i < kLevels * kColumns; i += kThreads) {
      sm.row.count[0][i] = 0;
      if constexpr (WEIGHTS) sm.row.weight[0][i] = 0;
    }
    __syncthreads();
    const int column = lane % kColumns;
    each_piece<AGAIN>([&](int i, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int b = bucket_of(x[e]);
        if (b >= kLevels) continue;
        const u64 w = measure(x[e], index(i, e));
        if (w == 0) continue;
        atomicAdd(&sm.row.count[b][column], 1u);
        if constexpr (WEIGHTS) atomicAdd(&sm.row.weight[b][column], w);
      }
    });
    __syncthreads();
    for (int i = tid; i < kLevels * kColumns; i += kThreads) {
      const u64 n = sum_of_8((u64)sm.row.count[0][i]);
      const u64 w = WEIGHTS ? sum_of_8(sm.row.weight[0][i]) : n;
      if (lane % kColumns == kColumns - 1)
        sm.level_count[i / kColumns] = (uint32_t)n, sm.level_weight[i / kColumns] = w;
    }
    __syncthreads();
    // (every wave for itself)
    static_assert(kLevels == 4 * 64 && kColumns == 8, "four buckets a lane, eight lanes a bucket's copies");
    u64 w[4], n[4], sum = 0, number = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum += w[e] = sm.level_weight[4 * lane + e];
      number += n[e] = sm.level_count[4 * lane + e];
    }
    const u64 upto = wave_scan(sum) + over;
    Level r;
    r.all = lane_of(upto, 63);
    const u64 target = target_of(r.all);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(upto - sum < target && upto >= target);
    const int at = hit != 0 ? __builtin_ctzll(hit) : 63;
    // (each lane as if it were the one)
    u64 above = upto - sum, count = wave_scan(number) - number + n[0], own = n[0];
    int e = 0;
#pragma unroll
    for (int y = 0; y < 3; ++y)
      if (e == y && above + w[y] < target) above += w[y], own = n[y + 1], count += own, ++e;
    r.bucket = hit != 0 ? 4 * at + __builtin_amdgcn_readlane(e, at) : kLevels;
    r.own = (uint32_t)lane_of(own, at);
    r.count = (uint32_t)lane_of(count, at);
    r.over = lane_of(above, at);
    return r;
  }

  // Appends the elements with good(x) to sm.list; their number (those past kList are not held).
  template <bool AGAIN, typename P>
  __device__ __forceinline__ int collect(P good) {
    if (tid == 0) sm.listed = 0;
    __syncthreads();
    each_piece<AGAIN>([&](int i, const float (&x)[4]) {
      uint64_t in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = __builtin_amdgcn_ballot_w64(good(x[e]));
      if ((in[0] | in[1] | in[2] | in[3]) == 0) return;  // wave-uniform
      uint32_t at = 0;
      if (lane == 0)
        at = atomicAdd(&sm.listed, (uint32_t)(__builtin_popcountll(in[0]) + __builtin_popcountll(in[1]) +
                                              __builtin_popcountll(in[2]) + __builtin_popcountll(in[3])));
      at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32),
                                                           __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0));
        if ((in[e] >> lane & 1) != 0 && to < (uint32_t)kList) sm.list[to] = index(i, e);
        at += __builtin_popcountll(in[e]);
      }
    });
    __syncthreads();
    const int n = (int)sm.listed;
    __syncthreads();  // (the next collect or search begins by setting it to 0)
    return n;
  }

  // The element at which the sum of weights, taken in descending order of the elements' numbers, reaches
  // target_of(sum of all); 0 where it does not. each(lo, hi, f) calls f(number, weight) for the
  // elements of those numbers that have a weight; no two have the same number.
  // (`over`: the sum of weights above hi)
  template <typename Each, typename G>
  __device__ __forceinline__ u64 search(const Each& each, u64 lo, u64 hi, G target_of, u64 over = 0) {
    u64 target = 0;
    while (true) {
      const float per = (float)kBuckets / ((float)(hi - lo) + 1.0f);
      auto bucket = [&](u64 k) { return min((int)((float)(hi - k) * per), kBuckets - 1); };
      sm.search.weight[tid] = 0;
      sm.search.count[tid] = 0;
      if (tid == 0) sm.bucket = kBuckets, sm.listed = 0;
      __syncthreads();
      each(lo, hi, [&](u64 k, u64 w) {
        const int b = bucket(k);
        atomicAdd(&sm.search.weight[b], w);
        atomicAdd(&sm.search.count[b], 1u);
      });
      __syncthreads();
      u64 all;
      const u64 w = sm.search.weight[tid], upto = over + before(w, all);
      if (target == 0) target = target_of(all);
      if (upto < target && upto + w >= target) {
        sm.bucket = tid;
        sm.found_above = upto;
        sm.bucket_count = sm.search.count[tid];
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

// Buckets of equal width below `top`, the last one with all that lies lower; and those of one bucket, in
// kLevels equal parts of it.
struct Levels {
  float top, per;
  __device__ __forceinline__ int operator()(float x) const {
    return x > neg_inf() ? (int)fminf((top - x) * per, (float)(kLevels - 1)) : kLevels;
  }
};
struct Parts {
  Levels levels;
  int bucket;
  __device__ __forceinline__ int operator()(float x) const {
    // Every use of this has to give an element the same part: Levels says whether it is in the bucket at
    // all, and the difference is rounded after the product, not once with it in some uses.
#pragma clang fp contract(off)
    const float t = (levels.top - x) * levels.per - (float)bucket;
    return levels(x) == bucket ? min(max((int)(t * (float)kLevels), 0), kLevels - 1) : kLevels;
  }
};

// The listed elements, kPerThread of them with every thread, each of weight 1.
template <typename T, int NP>
__device__ __forceinline__ Elements<kPerThread> listed(const Row<T, NP>& row, int n) {
  Elements<kPerThread> x;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = row.tid + j * kThreads;
    x.number[j] = i < n ? row.number_of(row.sm.list[i]) : 0;
    x.weight[j] = i < n ? 1 : 0;
  }
  return x;
}

// Over the whole row, where more stays than the list holds; hi: the largest key, `first`: the row's
// histogram for the first filter.
template <typename T, int NP>
__device__ __forceinline__ Pick pick_from_row(Row<T, NP>& row, const Settings& s, const Weigher& weigh,
                                              uint32_t hi, float per_k, float per_p,
                                              const typename Row<T, NP>::Level& first) {
  u64 cut = 1ull << 32;  // what stays: numbers from here on
  const u64 most = (u64)hi << 32 | 0xffffffffu;
  const float top = (float)weigh.top;
  // The number at which the sum of weigh_of(x, number) reaches its target: by the row's histogram and the
  // elements of its bucket, or, if they are too many (ties), in the row.
  auto cut_at = [&](auto by_weight, float per, auto target_of, bool known) {
    auto weight = [&](float x, u64 k) -> u64 {
      if constexpr (by_weight())
        return weigh(x) & (k >= cut ? ~u64(0) : 0);
      else
        return 1;
    };
    auto measure = [&](float x, int i) { return weight(x, order_of(x, i)); };
    const Levels levels{top, per};
    auto at = known ? first : row.template histogram<by_weight(), true>(levels, measure, target_of);
    const u64 target = target_of(at.all);
    auto among = [&](auto bucket_of) -> u64 {  // (the elements that weigh nothing are not in `own`)
      const int n =
          row.template collect<true>([&](float x) { return bucket_of(x) == at.bucket; });
      if (n > kList) return 0;
      Elements<kPerThread> x = listed(row, n);
      uint32_t low = 0;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j)
        if (x.weight[j] != 0) {
          low = max(low, (uint32_t)(~x.number[j] >> 32));
          x.weight[j] = weight(logit_of((uint32_t)(x.number[j] >> 32)), x.number[j]);
        }
      const uint32_t least = ~row.largest(low);
      return row.search(x, (u64)least << 32, most, [&](u64) { return target; }, at.over);
    };
    u64 found = 0;
    if (at.own <= (uint32_t)kList) {
      found = among(levels);
    } else if (at.bucket < kLevels - 1) {
      const Parts parts{levels, at.bucket};
      at = row.template histogram<by_weight(), true>(parts, measure, [&](u64) { return target; }, at.over);
      if (at.own <= (uint32_t)kList) found = among(parts);
    }
    if (found != 0) return found;
    auto each = [&](u64 lo, u64 hi, auto f) {
      row.template each_again<2>([&](int i, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 k = order_of(x[e], row.index(i, e));
          if (k >= lo && k <= hi) {
            const u64 w = weight(x[e], k);
            if (w != 0) f(k, w);
          }
        }
      });
    };
    return row.search(each, cut, most, [&](u64) { return target; });
  };
  if (s.k < row.vocab)
    cut = max(cut, cut_at(std::false_type{}, per_k, [&](u64) { return (u64)s.k; }, true));
  if (s.p < 1.0f)
    cut = max(cut, cut_at(std::true_type{}, per_p, [&](u64 all) { return reaching(s.p, all); },
                          s.k == row.vocab));
  Pick pick;
  pick.token = row.template in_order<true>(
      [&](float x, int i) -> u64 {
        // (no branch: one would leave each weight's latency bare)
        const u64 w = weigh(x) & (order_of(x, i) >= cut ? ~u64(0) : 0);
        return s.min_p > 0.f && weigh.exact(x) < (double)s.min_p ? 0 : w;
      },
      [&](u64 all) { return exceeding(s.u, all); }, pick.all);
  return pick;
}

// Of a number and a weight a lane (0: none; no two numbers are the same): the sum of the weights of the
// lanes with larger numbers.
__device__ __forceinline__ u64 above_in_wave(u64 number, u64 weight, int n) {
  u64 sum = 0;
  for (int i = 0; i < n; ++i) {
    const u64 k = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(number >> 32), i) << 32 |
                  (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)number, i);
    const u64 w = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(weight >> 32), i) << 32 |
                  (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)weight, i);
    sum += k > number ? w : 0;
  }
  return sum;
}
__device__ __forceinline__ u64 wave_total(u64 x) {
  x = wave_scan(x);
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
}

// pick_from_list for up to 64 candidates, in one wave; the answer is in every lane.
__device__ __forceinline__ Pick pick_in_wave(const Settings& s, const Weigher& weigh, u64 number, int n,
                                             u64 z, int lane) {
  u64 w = 0;
  if (lane < n) {
    w = weigh(logit_of((uint32_t)(number >> 32)));
    if (s.min_p > 0.f && !(s.p < 1.0f) && weigh.exact(logit_of((uint32_t)(number >> 32))) < (double)s.min_p)
      w = 0;
  }
  if (s.k < n && above_in_wave(number, lane < n ? 1 : 0, n) >= (u64)s.k) w = 0;
  if (s.p < 1.0f) {
    const u64 all = z != 0 ? z : wave_total(w);
    if (above_in_wave(number, w, n) >= reaching(s.p, all)) w = 0;
    if (s.min_p > 0.f && w != 0 &&
        weigh.exact(logit_of((uint32_t)(number >> 32))) < (double)s.min_p)
      w = 0;
  }
  Pick pick;
  pick.all = wave_total(w);
  const u64 at = (uint32_t)number, before = above_in_wave(at, w, n);  // ~index: the lowest first
  const u64 target = exceeding(s.u, pick.all);
  const uint64_t hit = __builtin_amdgcn_ballot_w64(w != 0 && before < target && before + w >= target);
  pick.token = (int)~(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)number, __builtin_ctzll(hit));
  return pick;
}

// Among the n candidates in sm.list, which hold every element that can stay; z: the weights' sum that
// top-p goes by, 0 for that of the first k.
template <typename T, int NP>
__device__ __forceinline__ Pick pick_from_list(Row<T, NP>& row, const Settings& s,
                                               const Weigher& weigh, uint32_t hi, int n, u64 z) {
  Elements<kPerThread> x = listed(row, n);
  uint32_t low = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j)
    if (x.weight[j] != 0) low = max(low, (uint32_t)(~x.number[j] >> 32));
  const u64 most = (u64)hi << 32 | 0xffffffffu;
  u64 cut = (u64)~row.largest(low) << 32;
  if (s.k < n) cut = row.search(x, cut, most, [&](u64) { return (u64)s.k; });
  u64 sum = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j)
    if (j * kThreads < n) {
      x.weight[j] = j * kThreads + row.tid < n && x.number[j] >= cut
                        ? weigh(logit_of((uint32_t)(x.number[j] >> 32)))
                        : 0;
      sum += x.weight[j];
    }
  if (s.p < 1.0f) {
    if (z == 0) row.before(sum, z);
    cut = row.search(x, cut, most, [&](u64) { return reaching(s.p, z); });
  }
  sum = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j)
    if (j * kThreads < n) {
      if (x.number[j] < cut ||
          (s.min_p > 0.f &&
           weigh.exact(logit_of((uint32_t)(x.number[j] >> 32))) < (double)s.min_p))
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

template <typename T, int NP>
__global__ __launch_bounds__(kThreads, NP == 0 ? 4 : 2) void sample_kernel(
    int* __restrict__ tokens, float* __restrict__ probs, const T* __restrict__ logits, long long ld,
    int vocab, const SampleSettings set) {
  __shared__ Shared sm;
  const int r = blockIdx.x;
  const T* base = logits + r * ld;
  Row<T, NP> row(base, vocab, sm);
  const int tid = row.tid;

  Settings s;
  s.temperature = set.temperature == nullptr ? 1.0f : set.temperature[r];
  s.k = set.top_k == nullptr ? 0 : set.top_k[r];
  s.p = set.top_p == nullptr ? 1.0f : set.top_p[r];
  s.min_p = set.min_p == nullptr ? 0.0f : set.min_p[r];
  s.u = set.uniforms[r];
  s.u = s.u > 0.f ? fminf(s.u, 1.0f) : 0.f;
  if (!(s.temperature > 0.f) || s.min_p > 1.0f) s.temperature = 1.0f, s.k = 1;  // the first largest
  if (s.k <= 0 || s.k > vocab) s.k = vocab;
  if (!(s.p < 1.0f)) s.p = 1.0f;
  if (!(s.min_p > 0.f)) s.min_p = 0.f;
  if (tid < 64) sm.root[tid] = exp2(tid / 64.0);

  float mine = neg_inf();
  row.template each_piece<false>([&](int, const float (&x)[4]) {
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
    row.set_infinite();
    mine = mine == __builtin_inff() ? 0.f : neg_inf();
    hi = key_of(0.f);
  }
  const float top = logit_of(hi);
  if (s.k == 1) {
    uint32_t first = 0;  // ~index
    if (mine == top)     // (only some threads: their elements once more)
      row.template each_again<4>([&](int i, const float (&x)[4]) {
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
  auto finish = [&](const Pick& pick) {
    Four<T> x;
    x.set(0, base[pick.token]);
    answer(pick.token, (float)(weigh.exact(row.value(x, 0)) * 0x1p44 / (double)pick.all));
  };
  int n = kList + 1;  // candidates
  typename Row<T, NP>::Level at{};
  u64 z = 0;
  // buckets a unit of logit: for top-k down to the smallest maximum of a thread, which that many elements
  // reach if every thread has one, and further for a larger k; for top-p down to what weighs nothing
  float per_k = 0.f, per_p = (float)(kLevels - 1) / (kFaintest * s.temperature);
  if (!(per_p < 0x1p100f)) per_p = 0x1p100f;
  if (s.k < vocab) {
    const uint32_t low = ~row.largest(~key_of(mine));
    const float range = low != 0 ? 1.02f * (top - logit_of(low)) : kFaintest;
    per_k = (float)(kLevels - 1) / (s.k <= kThreads ? range : 2.0f * range);
    if (!(per_k < 0x1p100f)) per_k = 0x1p100f;
  }
  bool by_bound = false;  // the candidates are the logits from `bound` on
  float bound = -3.4028234663852886e38f;
  if (vocab <= kList && (s.k < vocab || s.p < 1.0f)) {
    by_bound = true;
  } else if (s.k < vocab || s.p < 1.0f) {
    const bool by_k = s.k < vocab;
    const Levels levels{top, by_k ? per_k : per_p};
    if (by_k)
      at = row.template histogram<false, false>(levels, [](float, int) { return u64(1); },
                                         [&](u64) { return (u64)s.k; });
    else
      at = row.template histogram<true, false>(levels, [&](float x, int) { return weigh(x); },
                                        [&](u64 all) { return reaching(s.p, all); });
    if (!by_k) z = at.all;
    if (at.count <= (uint32_t)kList) {
      // (the last bucket's lower end is the lowest logit, also where the distance overflows)
      by_bound = at.bucket >= kLevels - 1;
      const float end = (float)(at.bucket + 1);
      if (!by_bound) n = row.template collect<false>([&](float x) { return (top - x) * levels.per < end; });
    }
  } else if (s.min_p > 0.f) {
    by_bound = true;
    bound = fmaxf(logit_at(s.min_p), bound);
  }
  if (by_bound) n = row.template collect<false>([&](float x) { return x >= bound; });
  if (s.k == vocab && s.p == 1.0f && s.min_p == 0.f) {
    Pick pick;
    pick.token = row.template in_order<false>(
        [&](float x, int) { return weigh(x); }, [&](u64 all) { return exceeding(s.u, all); }, pick.all);
    return finish(pick);
  }
  if (n <= 64) {
    if (row.wave == 0) {
      const u64 number = row.lane < n ? row.number_of(sm.list[row.lane]) : 0;
      finish(pick_in_wave(s, weigh, number, n, z, row.lane));
    }
    return;
  }
  finish(n <= kList ? pick_from_list(row, s, weigh, hi, n, z)
                    : pick_from_row(row, s, weigh, hi, per_k, per_p, at));
}

template <typename T>
hipError_t launch_sample_t(int* tokens, float* probs, const T* logits, long long ld, int rows,
                           int vocab, const SampleSettings& set, hipStream_t stream) {
  auto run = [&](auto np) {
    sample_kernel<T, np()><<<rows, kThreads, 0, stream>>>(tokens, probs, logits, ld, vocab, set);
    return hipGetLastError();
  };
  // Pieces of 256 elements for each of the 8 waves; up to 25 of them stay in registers (100 for fp32), as many
  // as the others leave room for: larger vocabularies are read again. A row with fewer pieces than its kernel
  // walks empty ones, so up to 8 have a kernel of their own. 32 rows in fp32, top-k of 40 / top-p of 0.9 / no
  // filter, us (bf16 within 3.5 of it):
  //   vocabulary   8 pieces           25                 read again
  //         4000   20.4  26.7   7.6   23.4  29.3  14.6   20.3  26.6   6.7
  //        16000   13.0  55.7  10.0   18.2  62.1  17.0   16.0  56.8  11.6
  //        25000                      19.5  74.1  19.8   22.2  72.9  19.2
  //        32000                      19.0  71.8  20.7   21.1  70.2  19.9
  //        40000                      19.8  68.0  22.6   24.0  68.6  24.1
  //        50257                      20.1  73.4  24.9   28.6  78.1  30.8
  //       131072                                         48.5   178  64.6
  // With more rows than CUs, two workgroups on a CU, in 128 registers each and with the row from L2, hide
  // more than that saves (512 rows of 50257 in bf16: 153 us, 203 with the rows in registers).
  const int pieces = (vocab + 3 + 256 * kWaves - 1) / (256 * kWaves);
  if (rows > (device_cus() > 0 ? device_cus() : 256)) return run(std::integral_constant<int, 0>{});
  if (pieces <= 8) return run(std::integral_constant<int, 8>{});
  if (pieces <= 25) return run(std::integral_constant<int, 25>{});
  return run(std::integral_constant<int, 0>{});
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
