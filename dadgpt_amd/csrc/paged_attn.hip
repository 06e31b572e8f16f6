// Attention of each sequence's new tokens over its pages, for gfx950: chunks of prompts, single tokens,
// and both in one call.
//
// Work. The queries that share a KV head are rows of one product: row r of a (sequence, KV head) is
// query head r % G of its group for new token r / G, so that K and V are read once for the group. A
// workgroup owns 128 of these rows, and `chunk` keys of those that they see; the chunks of one tile
// leave fp32 partials, which the last workgroup to arrive merges (as decode.hip, whose header says why
// relaxed agent-scope accesses order that).
//
// The keys are walked in tiles of 64. A tile is four groups of 16 tokens, each within a page (a page
// holds 16 at least): a wave stages one group of K and V by direct global -> LDS loads from wherever
// the block table puts it, tile t + 1 in flight while tile t is multiplied. Scores, softmax and P V are
// those of the bf16 forward (attn_fwd_bf16.hip): S^T = K Q^T with Q in registers, a lane a row,
// P straight from the score registers into O^T += V^T P^T, and a running maximum that moves only when
// weights would reach 2^64.
//
// Where a tile has fewer rows than 128, two or four waves share 32 rows and take every second or fourth
// 32 keys; their results are merged at the end.
//
// fp32: the same walk with the products of x3.hpp (six bf16 products for an fp32 one), tiles loaded
// into registers and split into three bf16 planes as they are stored, maxima in natural-log units.
#include "common.hpp"
#include "decode.hpp"
#include "lanes.hpp"
#include "paged.hpp"
#include "serving.hpp"
#include "tiles.hpp"
#include "x3.hpp"

namespace dadgpt {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 32 * kWaves;  // rows of a workgroup
constexpr float kMaxP = 0x1p64f;    // weights that reach it move the running maximum

template <typename T>
struct TileArgs {
  T* out;
  const T *q, *k_pages, *v_pages;
  long long ld_out, ld_q;
  PagedStep p;
  int group, page_log2;
  int chunk, n_chunk;   // keys of a workgroup, chunks of the longest cache
  int part_rows;        // rows that a partial has room for
  bool one_tile;        // every sequence has one tile at most
  float scale;          // fp32: as it is; bf16: |scale| log2 e
  bool negate;          // scale < 0 (bf16)
  float* part;          // [tile][KV head][chunk][part_rows][D + 2]: maximum, sum, unnormalised output
  unsigned* counter;    // [tile][KV head]
};

// What a workgroup does: tile `tile` of the step's list (every sequence's tiles one after the other),
// KV head `head`, keys key0 .. key1 - 1.
struct Work {
  int seq, row0, rows;            // first row of the tile in the sequence's rows x heads, rows in it
  int first, token, key0, key1;   // row of the step of the sequence's first token, that token's number
  int chunks;                     // of the tile
  __device__ __forceinline__ bool none() const { return rows <= 0; }
};

template <typename T>
__device__ __forceinline__ Work find_work(const TileArgs<T>& a, int lane) {
  int seq = blockIdx.y, tile = 0;
  if (!a.one_tile) {
    // the sequence whose tiles hold this one: 64 sequences at a time, their tiles summed up over lanes
    int left = blockIdx.y;
    seq = a.p.n_seq;
    for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
      int n = 0;
      if (s0 + lane < a.p.n_seq) {
        const paged::NewRows r(a.p, s0 + lane);
        n = (int)(((long long)r.count * a.group + kTile - 1) / kTile);
      }
      int upto = n;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(upto, d, 64);
        if (lane >= d) upto += y;
      }
      const uint64_t reach = __builtin_amdgcn_ballot_w64(upto > left);
      if (reach != 0) {
        const int at = __builtin_ctzll(reach);
        seq = s0 + at;
        tile = left - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
        break;
      }
      left -= __builtin_amdgcn_readlane(upto, 63);
    }
  }
  Work w{};
  if (seq >= a.p.n_seq) return w;
  w.seq = seq;
  const paged::NewRows r(a.p, seq);
  w.row0 = tile * kTile;
  w.rows = (int)min((long long)kTile, (long long)r.count * a.group - w.row0);
  if (w.none()) return w;
  w.first = r.first;
  w.token = r.token;
  const int seen = r.token + (w.row0 + w.rows - 1) / a.group + 1;  // by the tile's last row
  w.chunks = seen > a.chunk ? (seen + a.chunk - 1) / a.chunk : 1;
  if ((int)blockIdx.z >= w.chunks) w.rows = 0;
  w.key0 = blockIdx.z * a.chunk;
  w.key1 = min(seen, w.key0 + a.chunk);
  return w;
}

// Row `r` of a workgroup's rows: its new token, and where its elements lie in a row of q or out.
struct RowPlace {
  int t, col;
};
template <int D>
__device__ __forceinline__ RowPlace row_place(const Work& w, int group, int r) {
  const uint32_t x = w.row0 + r, t = x / (uint32_t)group;
  return RowPlace{(int)t, (int)((blockIdx.x * group + (x - t * group)) * D)};
}

// ------------------------------------------------------------------------ merging

__device__ __forceinline__ void st_agent2(float* p, float a, float b) {
  const uint64_t w = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// e^x or, in the bf16 kernel, whose maxima are in log2 units, 2^x; 0 at -inf.
template <typename T>
__device__ __forceinline__ float weight_of(float x) {
  if constexpr (sizeof(T) == 2)
    return fast_exp2(x);
  else
    return x == neg_inf() ? 0.f : exp_acc(x);
}

// Parts of one row's sums: maximum, weights, weighted values. A part whose scores are all -inf weighs
// nothing.
template <typename T>
struct Merged {
  float m = neg_inf(), l = 0.f, o = 0.f;
  __device__ __forceinline__ void add(float m1, float l1, float o1) {
    const float mn = fmaxf(m, m1), base = mn == neg_inf() ? 0.f : mn;
    const float f0 = weight_of<T>(m - base), f1 = weight_of<T>(m1 - base);
    m = mn;
    l = l * f0 + l1 * f1;
    o = o * f0 + o1 * f1;
  }
  __device__ __forceinline__ float value() const { return l == 0.f ? 0.f : o / l; }
};
// The partials of chunks c0 .. c1 - 1 of one element (`at`: its row's first partial, `col`), eight
// loaded before any is used.
template <typename T>
__device__ __forceinline__ Merged<T> merge_chunks_of(const float* at, size_t pitch, int col, int c0,
                                                     int c1) {
  constexpr int N = 8;
  Merged<T> r;
  for (int c = c0; c < c1; c += N) {
    float m[N], l[N], o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float* x = at + min(c + j, c1 - 1) * pitch;
      m[j] = ld_agent(x);
      l[j] = ld_agent(x + 1);
      o[j] = ld_agent(x + 2 + col);
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j < c1) r.add(m[j], l[j], o[j]);
  }
  return r;
}

// The last workgroup of a tile to arrive: every chunk's partial is written. `lds`: kFew * D * kWaves * 3
// floats. Few rows: a wave takes every element for a quarter of the chunks.
constexpr int kFew = 8;
template <typename T, int D>
__device__ __forceinline__ void merge_tile(const TileArgs<T>& a, const Work& w, const float* part,
                                           float* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t pitch = (size_t)a.part_rows * (D + 2);
  auto store = [&](int e, float x) {
    const RowPlace at = row_place<D>(w, a.group, e / D);
    a.out[(w.first + at.t) * a.ld_out + at.col + e % D] = Elem<T>::from(x);
  };
  const int n = w.rows * D;
  if (w.rows > kFew) {
    for (int e = tid; e < n; e += kThreads)
      store(e, merge_chunks_of<T>(part + (e / D) * (D + 2), pitch, e % D, 0, w.chunks).value());
    return;
  }
  Merged<T>* all = reinterpret_cast<Merged<T>*>(lds);
  const int c0 = w.chunks * wave / kWaves, c1 = w.chunks * (wave + 1) / kWaves;
  for (int e = lane; e < n; e += 64)
    all[wave * kFew * D + e] = merge_chunks_of<T>(part + (e / D) * (D + 2), pitch, e % D, c0, c1);
  __syncthreads();
  for (int e = tid; e < n; e += kThreads) {
    Merged<T> r = all[e];
#pragma unroll
    for (int x = 1; x < kWaves; ++x) {
      const Merged<T>& y = all[x * kFew * D + e];
      r.add(y.m, y.l, y.o);
    }
    store(e, r.value());
  }
}

// Counts this workgroup's partial (written by the relaxed agent-scope stores before) in; true in the
// last workgroup of the tile, which leaves the counter at zero.
__device__ __forceinline__ bool last_to_arrive(unsigned* counter, int chunks, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned before =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = before == (unsigned)(chunks - 1);
    if (before == (unsigned)(chunks - 1))  // no one else of this call comes
      __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *flag != 0;
}

// ------------------------------------------------------------------------ rows and waves

// Who of a workgroup does what: `ks` waves to 32 rows, wave `sub` of them for rows q0 .. q0 + 31, lane l
// and l + 32 for row q0 + l % 32 (rows past the tile's last repeat it).
template <int D>
struct WaveRows {
  int ks, groups, grp, sub, q0;
  bool active;
  RowPlace mine;
  int after;               // the last key that the lane's row sees,
  int all_see, some_see;   // that all and that some of the wave's rows do
  __device__ __forceinline__ WaveRows(const Work& w, int group, int wave, int l32) {
    ks = w.rows <= 32 ? 4 : w.rows <= 64 ? 2 : 1;
    groups = kWaves / ks;
    grp = wave % groups;
    sub = wave / groups;
    q0 = 32 * grp;
    active = q0 < w.rows;
    mine = row_place<D>(w, group, min(q0 + l32, w.rows - 1));
    after = w.token + mine.t;
    all_see = w.token + (w.row0 + q0) / group;
    some_see = w.token + (w.row0 + min(q0 + 31, w.rows - 1)) / group;
  }
  __device__ __forceinline__ bool owner() const { return sub == 0 && active; }
};

// Adds up the waves that share rows, rescaled to the larger maximum, in order, into the owners'. The
// workgroup's reads of `lds` are done before and after.
template <typename T, int D>
__device__ __forceinline__ void join_waves(const WaveRows<D>& r, f32x16 (&o)[D / 32], float& m,
                                           float& l, void* lds, float (*ml)[2][64], int lane) {
  if (r.ks == 1) return;
  AccLds* slots = reinterpret_cast<AccLds*>(lds);
  const int slot = (r.sub - 1) * r.groups + r.grp;
  if (r.sub > 0) {
    put_acc(o, slots + slot * (D / 32), lane);
    ml[slot][0][lane] = m;
    ml[slot][1][lane] = l;
  }
  __syncthreads();
  if (r.sub == 0)
    for (int x = 0; x < r.ks - 1; ++x) {
      const int from = x * r.groups + r.grp;
      const float m1 = ml[from][0][lane], mn = fmaxf(m, m1);
      const float base = mn == neg_inf() ? 0.f : mn;
      const float f0 = weight_of<T>(m - base), f1 = weight_of<T>(m1 - base);
      m = mn;
      l = l * f0 + ml[from][1][lane] * f1;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] *= f0;
      add_acc(o, slots + from * (D / 32), lane, f1);
    }
  __syncthreads();
}

// A tile of several chunks: leaves this one's partial, and in the last workgroup to arrive merges all.
template <typename T, int D>
__device__ __forceinline__ void leave_partial(const TileArgs<T>& a, const Work& w,
                                              const WaveRows<D>& r, const f32x16 (&o)[D / 32], float m,
                                              float l, float* lds, int* flag, int lane) {
  const int l32 = lane & 31, hi = lane >> 5;
  const size_t unit = (size_t)blockIdx.y * a.p.Hkv + blockIdx.x;
  float* part = a.part + unit * a.n_chunk * a.part_rows * (D + 2);
  if (r.owner() && r.q0 + l32 < w.rows) {
    float* row = part + ((size_t)blockIdx.z * a.part_rows + r.q0 + l32) * (D + 2);
    if (hi == 0) st_agent2(row, m, l);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float* to = row + 2 + 32 * db + 8 * g + 4 * hi;
        st_agent2(to, o[db][4 * g], o[db][4 * g + 1]);
        st_agent2(to + 2, o[db][4 * g + 2], o[db][4 * g + 3]);
      }
  }
  if (last_to_arrive(a.counter + unit, w.chunks, flag)) merge_tile<T, D>(a, w, part, lds);
}

// The pages of a tile's four groups of 16 tokens, the first of them token `key`.
struct Pages {
  int id[4];
};
template <typename T>
__device__ __forceinline__ Pages pages_at(const TileArgs<T>& a, const Work& w, int key) {
  const int* table = a.p.table + (size_t)w.seq * a.p.max_pages;
  Pages g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    g.id[i] = table[min((key + 16 * i) >> a.page_log2, a.p.max_pages - 1)];
  return g;
}

// ------------------------------------------------------------------------ bf16

// Weights exp2(s c - m) as bf16 operands of the next product; their fp32 sum.
__device__ __forceinline__ float weights_bf16(bf16x8 (&p)[2], const f32x16& s, float c, float m) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 8 * j + 2 * e;
      const float p0 = fast_exp2(fmaf(s[r], c, -m)), p1 = fast_exp2(fmaf(s[r + 1], c, -m));
      w[e] = pack_bf16x2(p0, p1);
      sum = r == 0 ? p0 + p1 : sum + (p0 + p1);
    }
    p[j] = as_bf16x8(w);
  }
  return sum;
}

// A wave's 16 tokens of a tile of K or V: `rows` of them exist (the others take the last one's place;
// they are masked, and must be finite where the last one is), `id` names their page; nothing to read: zeros.
template <int D>
struct Stage {
  static constexpr int C = D / 8, PER = 16 * C / 64;  // pieces a row, instructions a wave
  uint32_t off[PER];
  __device__ __forceinline__ explicit Stage(int lane) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int row = (n * 64 + lane) / C, c = (n * 64 + lane) % C;
      off[n] = (uint32_t)(row * D + (c ^ swz<D>(row)) * 8) * 2u;
    }
  }
  __device__ __forceinline__ void operator()(bf16* tile, const bf16* src, int rows, bool there,
                                             int wave, int lane) const {
    bf16* to = tile + wave * 16 * D;
    if (!there) {
#pragma unroll
      for (int n = 0; n < PER; ++n)
        *reinterpret_cast<u32x4*>(to + (n * 64 + lane) * 8) = u32x4{0u, 0u, 0u, 0u};
      return;
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      uint32_t o = off[n];
      if (rows < 16) {
        const int r = (n * 64 + lane) / C;
        if (r >= rows) o -= (uint32_t)((r - rows + 1) * D * 2);
      }
      dma_lds16_sbase(src, o, to + n * 64 * 8);
    }
  }
};

template <int D>
__global__ __launch_bounds__(kThreads, 3) void paged_bf16_kernel(const TileArgs<bf16> a) {
  constexpr int DS = D / 16, DB = D / 32;
  // two tiles of K, two of V; in the end the waves' partials, output rows or merged chunks
  __shared__ __attribute__((aligned(16))) bf16 lds[4 * kTileRows * D];
  bf16 *const sk[2] = {lds, lds + kTileRows * D};
  bf16 *const sv[2] = {lds + 2 * kTileRows * D, lds + 3 * kTileRows * D};
  __shared__ float sm_ml[kWaves - 1][2][64];
  __shared__ int flag;
  static_assert(sizeof(lds) >= (kWaves - 1) * DB * sizeof(AccLds), "waves' partials fit");
  static_assert(sizeof(lds) >= kWaves * 32 * D * sizeof(bf16), "output rows fit");
  static_assert(sizeof(lds) >= kFew * D * kWaves * sizeof(Merged<bf16>), "merged chunks fit");

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_work(a, lane);
  if (w.none()) return;
  const WaveRows<D> r(w, a.group, wave, l32);

  // the lane's query, columns 16 ds + 8 hi + 0 .. 7 (rows past the last repeat it)
  const bf16* qrow = a.q + (w.first + r.mine.t) * a.ld_q + r.mine.col + 8 * hi;
  bf16x8 qop[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qop[ds] = ld_g128(qrow + 16 * ds);
  const int head = blockIdx.x, n_tiles = w.key1 > w.key0 ? (w.key1 - w.key0 + 63) / 64 : 0;
  const Stage<D> stage(lane);
  auto load = [&](int t, const Pages& g, bf16* tk, bf16* tv) {
    const int key = w.key0 + 64 * t + 16 * wave, left = w.key1 - key;
    const int id = wave == 0 ? g.id[0] : wave == 1 ? g.id[1] : wave == 2 ? g.id[2] : g.id[3];
    const bool there = left > 0 && paged::is_page(a.p, id);
    const size_t at = there ? paged::page_row(a.p, id, head, key & (a.p.page - 1)) : 0;
    stage(tk, a.k_pages + at, left, there, wave, lane);
    stage(tv, a.v_pages + at, left, there, wave, lane);
  };

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  float m = neg_inf(), l = 0.f;

  Pages now{}, next{};
  if (n_tiles > 0) {
    now = pages_at(a, w, w.key0);
    load(0, now, sk[0], sv[0]);
    if (n_tiles > 1) next = pages_at(a, w, w.key0 + 64);
  }
  wait_vm_lds<0>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) {
    asm volatile("" : "+v"(qop[ds]));
    if (a.negate) qop[ds] = neg_bf16x8(qop[ds]);
  }

  auto tile = [&](int t, const bf16* ck, const bf16* cv, bf16* nk, bf16* nv) {
    const int k0 = w.key0 + 64 * t;
    Pages after_next = next;
    if (t + 1 < n_tiles) {
      load(t + 1, next, nk, nv);
      if (t + 2 < n_tiles) after_next = pages_at(a, w, k0 + 128);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c0 = k0 + 32 * i;
      if (!r.active || ((2 * t + i) & (r.ks - 1)) != r.sub || c0 > r.some_see || c0 >= w.key1)
        continue;
      const bool bad0 = !paged::is_page(a.p, now.id[2 * i]);
      const bool bad1 = !paged::is_page(a.p, now.id[2 * i + 1]);
      f32x16 s{};
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
        s = mfma32(lds_op(ck, rm_off<D>(32 * i + sigma32(l32), 2 * ds + hi)), qop[ds], s);
      if (c0 + 31 > r.all_see || bad0 || bad1) {
        const int last = r.after - c0 - 8 * hi;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (reg_row(x, 0) > last || (x < 8 ? bad0 : bad1)) s[x] = neg_inf();
      }
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 va[DB][2], p[2];
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 2; ++j) va[db][j] = lds_tr_op<D>(cv, 32 * i + 16 * j, 32 * db, lane);
      float sum = weights_bf16(p, s, a.scale, m);
      // 2^64 or more, inf, or NaN (a row's first keys: m is -inf), compared on the bits; both halves of
      // a row take the row's decision, and no other row's bits depend on it
      const bool need = __float_as_uint(sum) >= __float_as_uint(kMaxP);
      if (__builtin_amdgcn_ballot_w64(need) != 0) {
        float mx = s[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) mx = fmaxf(mx, s[x]);
        mx = max_halves(mx) * a.scale;
        const float mn = or_halves(need) ? fmaxf(m, mx) : m;
        const float base = mn == neg_inf() ? 0.f : mn;  // no key seen yet weighs anything
        const float f = fast_exp2(m - base);
        m = mn;
        l *= f;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= f;
        sum = weights_bf16(p, s, a.scale, base);
      }
      l += sum;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 2; ++j) o[db] = mfma32(va[db][j], p[j], o[db]);
    }
    now = next;
    next = after_next;
    wait_vm_lds<0>();
    __builtin_amdgcn_s_barrier();
  };
  for (int t = 0; t < n_tiles; t += 2) {
    tile(t, sk[0], sv[0], sk[1], sv[1]);
    if (t + 1 < n_tiles) tile(t + 1, sk[1], sv[1], sk[0], sv[0]);
  }
  l = sum_halves(l);

  join_waves<bf16, D>(r, o, m, l, lds, sm_ml, lane);
  if (w.chunks == 1) {
    if (!r.owner()) return;
    // rows through the wave's own stretch of LDS, so that a store instruction covers whole heads
    constexpr int C = D / 8;
    bf16* rows = lds + r.grp * 32 * D;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 4 * db + g;
        u32x2 x;
        x[0] = pack_bf16x2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv);
        x[1] = pack_bf16x2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
        *reinterpret_cast<u32x2*>(rows + l32 * D + ((c ^ (l32 % C)) << 3) + 4 * hi) = x;
      }
#pragma unroll
    for (int n = 0; n < 32 * C / 64; ++n) {
      const int i = (n * 64 + lane) / C, c = (n * 64 + lane) % C;
      const u32x4 x = *reinterpret_cast<const u32x4*>(rows + i * D + ((c ^ (i % C)) << 3));
      if (r.q0 + i < w.rows) {
        const RowPlace at = row_place<D>(w, a.group, r.q0 + i);
        *reinterpret_cast<u32x4*>(a.out + (w.first + at.t) * a.ld_out + at.col + 8 * c) = x;
      }
    }
    return;
  }
  leave_partial<bf16, D>(a, w, r, o, m, l, reinterpret_cast<float*>(lds), &flag, lane);
}

// ------------------------------------------------------------------------ fp32

// A tile's K or V on its way through registers: D / 16 pieces of 16 bytes a thread; tokens that do not
// exist are zeros.
template <int D>
struct PageTile {
  static constexpr int kPieces = D / 16, kThreads = 64 * kWaves;
  f32x4 r[kPieces];
  __device__ __forceinline__ void load(const TileArgs<float>& a, const float* pages, const Pages& g,
                                       int head, int key0, int key1) {
    const int row0 = threadIdx.x / (D / 4), col = 4 * (threadIdx.x % (D / 4));
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      constexpr int kStep = kThreads / (D / 4);  // rows of a piece of the workgroup: 16 or 32
      const int key = key0 + row0 + kStep * i;
      int id = g.id[kStep / 16 * i];
      if constexpr (kStep == 32) id = row0 < 16 ? id : g.id[2 * i + 1];
      const bool there = key < key1 && paged::is_page(a.p, id);
      r[i] = there ? *reinterpret_cast<const f32x4*>(
                         pages + paged::page_row(a.p, id, head, key & (a.p.page - 1)) + col)
                   : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  __device__ __forceinline__ f32x4 piece(int i) const { return r[i]; }
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void paged_f32_kernel(const TileArgs<float> a) {
  constexpr int DB = D / 32, kPlane = 3 * kTileRows * D, kPitch = D + 4;
  // K and V as three bf16 planes each; in the end the waves' partials, output rows or merged chunks
  __shared__ __attribute__((aligned(16))) bf16 planes[2 * kPlane];
  __shared__ float sm_ml[kWaves - 1][2][64];
  __shared__ int flag;
  static_assert(sizeof(planes) >= (kWaves - 1) * DB * sizeof(AccLds), "waves' partials fit");
  static_assert(sizeof(planes) >= kWaves * 32 * kPitch * sizeof(float), "output rows fit");
  static_assert(sizeof(planes) >= kFew * D * kWaves * sizeof(Merged<float>), "merged chunks fit");

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_work(a, lane);
  if (w.none()) return;
  const WaveRows<D> r(w, a.group, wave, l32);

  X3 q[D / 16];  // the lane's query, split
  load_split_row<D>(q, a.q + (w.first + r.mine.t) * a.ld_q + r.mine.col, hi);
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  float m = neg_inf(), l = 0.f;

  const int head = blockIdx.x, n_tiles = w.key1 > w.key0 ? (w.key1 - w.key0 + 63) / 64 : 0;
  Pages now{}, next{};
  PageTile<D> tk, tv;
  if (n_tiles > 0) {
    now = pages_at(a, w, w.key0);
    tk.load(a, a.k_pages, now, head, w.key0, w.key1);
    tv.load(a, a.v_pages, now, head, w.key0, w.key1);
    if (n_tiles > 1) next = pages_at(a, w, w.key0 + 64);
  }
  for (int t = 0; t < n_tiles; ++t) {
    const int k0 = w.key0 + 64 * t;
    __syncthreads();  // the last tile's reads are done
    store_x3<D, kTileRows>(tk, planes);
    store_x3<D, kTileRows>(tv, planes + kPlane);
    Pages after_next = next;
    if (t + 1 < n_tiles) {
      tk.load(a, a.k_pages, next, head, k0 + 64, w.key1);
      tv.load(a, a.v_pages, next, head, k0 + 64, w.key1);
      if (t + 2 < n_tiles) after_next = pages_at(a, w, k0 + 128);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c0 = k0 + 32 * i;
      if (!r.active || ((2 * t + i) & (r.ks - 1)) != r.sub || c0 > r.some_see || c0 >= w.key1)
        continue;
      const bool bad0 = !paged::is_page(a.p, now.id[2 * i]);
      const bool bad1 = !paged::is_page(a.p, now.id[2 * i + 1]);
      const bool partly = c0 + 31 > r.all_see || bad0 || bad1;
      const int last = r.after - c0 - 8 * hi;
      auto hidden = [&](int x) { return reg_row(x, 0) > last || (x < 8 ? bad0 : bad1); };
      f32x16 s = score_tile_p<D, kTileRows>(planes, 32 * i, q, lane);
      float sum;
      f32x16 p;
      auto weights = [&]() {
#pragma unroll
        for (int x = 0; x < 16; ++x) p[x] = exp_acc(fmaf(s[x], a.scale, -m));
        if (partly) {
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (hidden(x)) p[x] = 0.f;
        }
        sum = p[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) sum += p[x];
      };
      weights();
      // as in the bf16 kernel; a row that needs it sees a key of these
      const bool need = __float_as_uint(sum) >= __float_as_uint(kMaxW);
      if (__builtin_amdgcn_ballot_w64(need) != 0) {
        float mx = neg_inf();
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (!(partly && hidden(x))) mx = fmaxf(mx, s[x] * a.scale);
        mx = max_halves(mx);
        const float mn = or_halves(need) ? fmaxf(m, mx) : m;
        const float f = m == neg_inf() ? 0.f : exp_acc(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= f;
        weights();
      }
      l += sum;
      accumulate_t_p<D, kTileRows>(o, planes + kPlane, 32 * i, p, lane);
    }
    now = next;
    next = after_next;
  }
  l = sum_halves(l);
  __syncthreads();  // the tiles are read: partials and output rows go there
  join_waves<float, D>(r, o, m, l, planes, sm_ml, lane);
  if (w.chunks == 1) {
    if (!r.owner()) return;
    float* rows = reinterpret_cast<float*>(planes) + r.grp * 32 * kPitch;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(rows + l32 * kPitch + 32 * db + 8 * g + 4 * hi) =
            f32x4{o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv,
                  o[db][4 * g + 3] * inv};
#pragma unroll
    for (int n = 0; n < 32 * D / 4 / 64; ++n) {
      const int i = (n * 64 + lane) / (D / 4), c = (n * 64 + lane) % (D / 4);
      const f32x4 x = *reinterpret_cast<const f32x4*>(rows + i * kPitch + 4 * c);
      if (r.q0 + i < w.rows) {
        const RowPlace at = row_place<D>(w, a.group, r.q0 + i);
        *reinterpret_cast<f32x4*>(a.out + (w.first + at.t) * a.ld_out + at.col + 4 * c) = x;
      }
    }
    return;
  }
  leave_partial<float, D>(a, w, r, o, m, l, reinterpret_cast<float*>(planes), &flag, lane);
}

// ------------------------------------------------------------------------ host

struct Plan {
  int tiles, chunk, n_chunk, part_rows;
  size_t counters, partials;  // bytes
};

// Workgroups that a step is cut into where it has fewer tiles: about eight a CU.
long long wanted() { return 8LL * (device_cus() > 0 ? device_cus() : 256); }
constexpr int kLeastKeys = 256;  // of a chunk

long long tiles_of(int n_seq, long long group, int rows, int max_rows) {
  const long long per_seq = (max_rows * group + kTile - 1) / kTile;
  return std::min(n_seq * per_seq, n_seq + rows * group / kTile);
}

// Tiles of the step's list, keys of a workgroup, and what the workspace holds. The lengths are on the
// device: the grid has room for every sequence at its longest.
Plan plan_of(const PagedStep& s) {
  const long long group = s.H / s.Hkv, max_len = (long long)s.max_pages * s.page;
  Plan p{};
  p.tiles = (int)tiles_of(s.n_seq, group, s.rows, s.max_rows);
  p.part_rows = (int)std::min(s.max_rows * group, (long long)kTile);
  const long long units = (long long)p.tiles * s.Hkv;
  const long long want = (wanted() + units - 1) / units;
  const long long chunk = std::max<long long>(kLeastKeys, (max_len + want - 1) / want);
  p.chunk = (int)((chunk + 63) / 64 * 64);
  p.n_chunk = (int)((max_len + p.chunk - 1) / p.chunk);
  if (p.n_chunk > 1) {
    p.counters = counter_bytes(p.tiles, s.Hkv);
    p.partials = sizeof(float) * units * p.n_chunk * p.part_rows * (s.D + 2);
  }
  return p;
}

template <typename T, typename F>
hipError_t launch_paged_t(T* out, long long ld_out, const T* q, long long ld_q, const T* k_pages,
                          const T* v_pages, const PagedStep& s, float scale, void* workspace,
                          size_t workspace_bytes, F launch) {
  const Plan plan = plan_of(s);
  TileArgs<T> a{};
  a.out = out, a.q = q, a.k_pages = k_pages, a.v_pages = v_pages;
  a.ld_out = ld_out, a.ld_q = ld_q, a.p = s;
  a.group = s.H / s.Hkv;
  a.page_log2 = __builtin_ctz((unsigned)s.page);
  a.chunk = plan.chunk, a.n_chunk = plan.n_chunk, a.part_rows = plan.part_rows;
  a.one_tile = (long long)s.max_rows * a.group <= kTile;
  // bf16: masked scores are -inf before they are scaled, so the factor is kept above 0: at 1e-30 every score
  // weighs the same, as at a scale of 0 (as attn_fwd_bf16.hip).
  a.scale = sizeof(T) == 2 ? fmaxf(fabsf(scale) * kLog2e, 1e-30f) : scale;
  a.negate = scale < 0.f;
  if (plan.n_chunk > 1) {
    // the caller checked workspace_bytes >= paged_workspace_needed(); partials against its end
    const size_t at = (workspace_bytes - plan.partials) & ~(size_t)15;
    a.counter = static_cast<unsigned*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
  }
  launch(a, dim3(s.Hkv, plan.tiles, plan.n_chunk));
  return hipGetLastError();
}

}  // namespace

size_t paged_workspace_needed(const PagedStep& step) {
  const Plan p = plan_of(step);
  return p.n_chunk > 1 ? p.counters + p.partials + 16 : 0;
}

// Of n tiles x KV heads, n < wanted(), a plan makes at most ceil(max_len / kLeastKeys) chunks each and
// wanted() + n workgroups in all; more than that are not cut. The bound grows with every argument.
size_t paged_workspace_bytes(const PagedStep& s) {
  const long long group = s.H / s.Hkv, max_len = (long long)s.max_pages * s.page;
  const long long chunks = (max_len + kLeastKeys - 1) / kLeastKeys;
  if (chunks <= 1) return 0;
  const long long units =
      std::min(tiles_of(s.n_seq, group, s.rows, s.max_rows) * s.Hkv, wanted());
  const long long parts = std::min(units * chunks, wanted() + units);
  const long long part_rows = std::min(s.max_rows * group, (long long)kTile);
  return counter_bytes((int)units, 1) + sizeof(float) * parts * part_rows * (s.D + 2) + 16;
}

hipError_t launch_paged_attention_bf16(bf16* out, long long ld_out, const bf16* q, long long ld_q,
                                       const bf16* k_pages, const bf16* v_pages,
                                       const PagedStep& step, float scale, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  return launch_paged_t<bf16>(
      out, ld_out, q, ld_q, k_pages, v_pages, step, scale, workspace, workspace_bytes,
      [&](const TileArgs<bf16>& a, dim3 grid) {
        if (step.D == 64)
          paged_bf16_kernel<64><<<grid, kThreads, 0, stream>>>(a);
        else
          paged_bf16_kernel<32><<<grid, kThreads, 0, stream>>>(a);
      });
}

hipError_t launch_paged_attention_f32(float* out, long long ld_out, const float* q, long long ld_q,
                                      const float* k_pages, const float* v_pages,
                                      const PagedStep& step, float scale, void* workspace,
                                      size_t workspace_bytes, hipStream_t stream) {
  return launch_paged_t<float>(
      out, ld_out, q, ld_q, k_pages, v_pages, step, scale, workspace, workspace_bytes,
      [&](const TileArgs<float>& a, dim3 grid) {
        if (step.D == 64)
          paged_f32_kernel<64><<<grid, kThreads, 0, stream>>>(a);
        else
          paged_f32_kernel<32><<<grid, kThreads, 0, stream>>>(a);
      });
}

}  // namespace dadgpt
