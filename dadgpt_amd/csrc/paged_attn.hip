// Attention of each sequence's new tokens over its pages, for gfx950: chunks of prompts, single tokens,
// and both in one call.
//
// Work. The queries that share a KV head are rows of one product: row r of a (sequence, KV head) is
// query head r % G of its group for new token r / G, so that K and V are read once for the group. A few
// rows are one tile, 128 a tile otherwise; a workgroup owns a tile's rows for a chunk of the keys that
// they see. The chunks of one tile leave fp32 partials, which the last workgroup to arrive merges (as
// decode.hip, whose header says why relaxed agent-scope accesses order that).
//
// Three kernels, by the rows (path_of): paged_rows_kernel on the VALU, paged_mid_bf16_kernel in 16-row
// matrix tiles, and the tiles below. The first two are bound by HBM and by the chain row_start, lens ->
// page -> keys -> merge, and have all of a workgroup's loads in flight at once: 32 sequences of 1 to 1024
// tokens, 12 heads of 64 in bf16, 14 us (50 MB, 3.6 TB/s), 8 of 1 to 32768 with three rows for each of 4 KV
// heads 34 to 43 us (134 MB, 3.1 to 3.9 TB/s).
//
// Tiles (bf16). The keys are walked in tiles of 64. A tile is four groups of 16 tokens, each within a page
// (a page holds 16 at least): a wave stages one group of K and V by direct global -> LDS loads from
// wherever the block table puts it, tile t + 1 in flight while tile t is multiplied. Scores, softmax and
// P V are those of the bf16 forward (attn_fwd_bf16.hip): S^T = K Q^T with Q in registers, a lane a row,
// P straight from the score registers into O^T += V^T P^T, rounded to bf16 there as in the forward, and a
// running maximum that moves only when weights would reach 2^64. Where a tile has fewer rows than 128, two
// or four waves share 32 rows and take every second or fourth 32 keys; their results are merged at the end.
// Bound by VALU and matrix pipe, in waves that depend on themselves: 8 prompts' chunks of up to 512 rows
// over up to 8192 tokens, 12 heads, 54 to 67 us (25 GFLOP, up to 460 TFLOP/s); 512 rows over 32768 tokens
// 48 us (540 TFLOP/s). A third buffer, four workgroups a CU (spills) and neighbouring tiles on one XCD
// were no faster.
//
// fp32: the same walk with the products of x3.hpp (six bf16 products for an fp32 one), tiles loaded
// into registers and split into three bf16 planes as they are stored, maxima in natural-log units. 8 prompts'
// chunks as above over up to 4096 tokens: 124 to 136 us (12 GFLOP, 89 to 97 TFLOP/s of the 154 of a library
// product).
//
// Which kernel and how a tile's keys are cut follow from the step (the rows of a sequence at most, all tiles'
// keys): a sequence's results have the same bits in every equal step, and in another one, alone for instance,
// the same within their roundings.
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
  int chunk, n_chunk;   // a few rows: keys of a workgroup, chunks of the longest cache
  int slots;            // tiles: partials of a KV head that there is room for
  int rows, part_pitch; // the most of a tile; floats of its partial of a chunk
  float scale;          // fp32: as it is; bf16: |scale| log2 e
  bool negate;          // scale < 0 (bf16)
  float* part;          // partials: maximum, sum, unnormalised output of every row
  unsigned* counter;    // one for each partial; a tile uses its first chunk's
};

// What a workgroup does: the rows of a tile, KV head `head`, keys key0 .. key1 - 1 of chunk `chunk`.
struct Work {
  int head, chunk, chunks;        // (of the tile)
  int seq, row0, rows;            // first row of the tile in the sequence's rows x heads, rows in it
  int first, token, key0, key1;   // row of the step of the sequence's first token, that token's number
  int part0, part_step;           // the partial of its chunk 0, and how far apart those of its chunks are
  __device__ __forceinline__ bool none() const { return rows <= 0; }
  // rows from row0 on, chunk `chunk` of `keys` keys each; a cache of `whole` tokens or fewer stays in one
  template <typename T>
  __device__ __forceinline__ void take(const TileArgs<T>& a, const paged::NewRows& r, int keys,
                                       int whole) {
    rows = (int)min((long long)kTile, (long long)r.count * a.group - row0);
    if (none()) return;
    first = r.first;
    token = r.token;
    const int seen = token + (row0 + rows - 1) / a.group + 1;  // by the tile's last row
    chunks = seen > keys && r.len > whole ? (seen + keys - 1) / keys : 1;
    if (chunk >= chunks) rows = 0;
    key0 = chunk * keys;
    key1 = chunks == 1 ? seen : min(seen, key0 + keys);
  }
};

// A few rows: a sequence is one tile, in chunks of a.chunk keys; the grid is (KV head, sequence, chunk).
template <typename T>
__device__ __forceinline__ Work find_few(const TileArgs<T>& a) {
  Work w{};
  w.head = blockIdx.x, w.seq = blockIdx.y, w.chunk = blockIdx.z;
  w.part0 = (w.seq * a.p.Hkv + w.head) * a.n_chunk;
  w.part_step = 1;
  w.take(a, paged::NewRows::of<true>(a.p, w.seq), a.chunk, a.chunk);
  return w;
}

// Tiles of 128 rows: the grid is (KV head, place in a list). The list is every sequence's tiles, once for
// each chunk of its keys. How long a chunk is follows from the lengths, which only the device has: all the
// tiles' keys, shared out evenly over kShares workgroups, three a CU; longer where there are more tiles
// than that, which even each other out. So a cache that is far from its room still fills the machine, and
// one long sequence among short ones is cut. Merging chunks costs about 6 us of waiting, as much as a few
// tiles: a chunk has kLeastKeys at least, and in bf16 a sequence that is not twice as long stays whole.
// In bf16, 12 heads of 64, against equal parts of the longest cache: chunks of up to 512 rows of 8 prompts
// of up to 8192 tokens 67 us (75), 64 sequences of up to 1024 tokens with up to 256 rows 28 (29), one of
// 32768 with 512 rows 48 (55).
constexpr int kShares = 768;
template <typename T>
constexpr int kLeastKeys = sizeof(T) == 2 ? 512 : 256;
template <typename T>
constexpr int kWhole = sizeof(T) == 2 ? 2 : 1;  // chunks
template <typename T>
__device__ __forceinline__ Work find_tile(const TileArgs<T>& a, int lane) {
  // tiles and tokens of sequence s0 + lane
  auto count = [&](int s, int& tiles, int& len, uint64_t& keys) {
    tiles = 0, len = 0, keys = 0;
    if (s >= a.p.n_seq) return;
    const auto r = paged::NewRows::of<false>(a.p, s);
    tiles = (int)(((long long)r.count * a.group + kTile - 1) / kTile);
    len = max(r.token + r.count, 0);
    keys = (uint64_t)tiles * max(len - r.count / 2, (len + 1) / 2);  // about those that the rows see
  };
  int tiles, len;
  unsigned all_tiles = 0;
  uint64_t keys, all_keys = 0;
  for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
    count(s0 + lane, tiles, len, keys);
    all_tiles += tiles, all_keys += keys;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    all_tiles += __shfl_xor(all_tiles, d, 64);
    all_keys += __shfl_xor((unsigned long long)all_keys, d, 64);
  }
  const float share = (float)all_keys * a.p.Hkv * (1.0f / kShares) *
                      fmaxf(1.0f, (float)all_tiles * a.p.Hkv * (1.0f / kShares));
  const int chunk = max(kLeastKeys<T>, ((int)fminf(share, (float)(1 << 24)) + 64) / 64 * 64);

  Work w{};
  w.head = blockIdx.x;
  w.seq = -1;
  // the sequence whose places in the list hold this one: 64 sequences at a time, summed up over lanes
  int left = blockIdx.y, parts_before = 0, n_tiles = 0;
  for (int s0 = 0; s0 < a.p.n_seq; s0 += 64) {
    if (a.p.n_seq > 64) count(s0 + lane, tiles, len, keys);
    const int cuts = len > kWhole<T> * chunk ? (len + chunk - 1) / chunk : 1;
    const int places = tiles * cuts, parts = cuts > 1 ? places : 0;
    int upto = places, parts_upto = parts;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d, 64), y = __shfl_up(parts_upto, d, 64);
      if (lane >= d) upto += x, parts_upto += y;
    }
    const uint64_t reach = __builtin_amdgcn_ballot_w64(upto > left);
    if (reach != 0) {
      const int at = __builtin_ctzll(reach);
      w.seq = s0 + at;
      n_tiles = __builtin_amdgcn_readlane(tiles, at);
      left -= __builtin_amdgcn_readlane(upto - places, at);
      parts_before += __builtin_amdgcn_readlane(parts_upto - parts, at);
      // (a list that the arrays make longer than the step has room for: its tiles there are left out)
      if (parts_before + __builtin_amdgcn_readlane(parts, at) > a.slots) return w;
      break;
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
    parts_before += __builtin_amdgcn_readlane(parts_upto, 63);
  }
  if (w.seq < 0) return w;
  w.chunk = __builtin_amdgcn_readfirstlane(left / n_tiles);
  const int tile = n_tiles - 1 - (left - w.chunk * n_tiles);  // the last rows, which see most, first
  w.row0 = __builtin_amdgcn_readfirstlane(tile * kTile);
  w.part0 = (parts_before + tile) * a.p.Hkv + w.head;
  w.part_step = n_tiles * a.p.Hkv;
  const int keys_each = __builtin_amdgcn_readfirstlane(chunk);
  w.take(a, paged::NewRows::of<true>(a.p, w.seq), keys_each, kWhole<T> * keys_each);
  return w;
}

// Row `r` of a workgroup's rows: its new token, and where its elements lie in a row of q or out.
struct RowPlace {
  int t, col;
};
template <int D>
__device__ __forceinline__ RowPlace row_place(const Work& w, int group, int r) {
  const uint32_t x = w.row0 + r, t = x / (uint32_t)group;
  return RowPlace{(int)t, (int)((w.head * group + (x - t * group)) * D)};
}

// ------------------------------------------------------------------------ merging

// The partial of chunk `c` of the workgroup's tile.
template <typename T>
__device__ __forceinline__ float* partial(const TileArgs<T>& a, const Work& w, int c) {
  return a.part + (w.part0 + c * (size_t)w.part_step) * a.part_pitch;
}

__device__ __forceinline__ void st_agent2(float* p, float a, float b) {
  const uint64_t w = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// 2^x where the maxima are in log2 units, e^x where they are in natural-log ones (the fp32 tiles); 0 at
// -inf.
template <bool LOG2>
__device__ __forceinline__ float weight_of(float x) {
  if constexpr (LOG2)
    return fast_exp2(x);
  else
    return x == neg_inf() ? 0.f : exp_acc(x);
}

__device__ __forceinline__ void ld_agent2(const float* p, float& a, float& b) {
  const uint64_t w = __hip_atomic_load(const_cast<uint64_t*>(reinterpret_cast<const uint64_t*>(p)),
                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  a = __uint_as_float((uint32_t)w);
  b = __uint_as_float((uint32_t)(w >> 32));
}

// Parts of one row's sums: maximum, weights, weighted values. A part whose scores are all -inf weighs
// nothing.
template <bool LOG2>
struct Merged {
  float m = neg_inf(), l = 0.f, o = 0.f;
  __device__ __forceinline__ void add(float m1, float l1, float o1) {
    const float mn = fmaxf(m, m1), base = mn == neg_inf() ? 0.f : mn;
    const float f0 = weight_of<LOG2>(m - base), f1 = weight_of<LOG2>(m1 - base);
    m = mn;
    l = l * f0 + l1 * f1;
    o = o * f0 + o1 * f1;
  }
  __device__ __forceinline__ float value() const { return l == 0.f ? 0.f : o / l; }
};
// The partials of chunks c0 .. c1 - 1 of one element (`at`: its row's first partial, `col`), eight
// loaded before any is used.
template <bool LOG2>
__device__ __forceinline__ Merged<LOG2> merge_chunks_of(const float* at, size_t pitch, int col, int c0,
                                                     int c1) {
  constexpr int N = 8;
  Merged<LOG2> r;
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

// The last workgroup of a tile to arrive: every chunk's partial is written. Up to FEW rows, a wave takes
// every element for its share of the chunks; `lds` has room for FEW * D * WAVES Merged.
constexpr int kFew = 8;
template <bool LOG2, int WAVES, int FEW, typename T, int D>
__device__ __forceinline__ void merge_tile(const TileArgs<T>& a, const Work& w, const float* part,
                                           void* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t pitch = a.part_pitch;
  auto store = [&](int e, float x) {
    const RowPlace at = row_place<D>(w, a.group, e / D);
    a.out[(w.first + at.t) * a.ld_out + at.col + e % D] = Elem<T>::from(x);
  };
  auto merge = [&](int e, int c0, int c1) {
    return merge_chunks_of<LOG2>(part + (e / D) * (D + 2), pitch, e % D, c0, c1);
  };
  const int n = w.rows * D;
  if (w.rows > FEW) {
    for (int e = tid; e < n; e += 64 * WAVES) store(e, merge(e, 0, w.chunks).value());
    return;
  }
  Merged<LOG2>* all = reinterpret_cast<Merged<LOG2>*>(lds);
  const int c0 = w.chunks * wave / WAVES, c1 = w.chunks * (wave + 1) / WAVES;
  for (int e = lane; e < n; e += 64) all[wave * FEW * D + e] = merge(e, c0, c1);
  __syncthreads();
  for (int e = tid; e < n; e += 64 * WAVES) {
    Merged<LOG2> r = all[e];
#pragma unroll
    for (int x = 1; x < WAVES; ++x) {
      const Merged<LOG2>& y = all[x * FEW * D + e];
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
      const float f0 = weight_of<sizeof(T) == 2>(m - base), f1 = weight_of<sizeof(T) == 2>(m1 - base);
      m = mn;
      l = l * f0 + ml[from][1][lane] * f1;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] *= f0;
      add_acc(o, slots + from * (D / 32), lane, f1);
    }
  __syncthreads();
}

// A row's running state in a wave: maximum and sum of its weights, O^T.
template <int D>
struct Running {
  f32x16 o[D / 32];
  float m = neg_inf(), l = 0.f;
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
  }
};

// A tile of several chunks: the owners leave their sums as the lanes hold them, so that every store of a
// wave is 512 bytes in a row; in the last workgroup to arrive the waves that share rows take every chunk in
// turn and are joined again, and true is returned.
__host__ __device__ constexpr int group_floats(int D) { return 64 * (2 + D / 2); }  // of 32 rows
template <typename T, int D>
__device__ __forceinline__ bool merge_chunks(const TileArgs<T>& a, const Work& w,
                                             const WaveRows<D>& r, Running<D>& x, void* lds,
                                             float (*ml)[2][64], int* flag, int lane) {
  constexpr int N = D / 2;  // of O^T in a lane
  const int place = r.grp * group_floats(D) + 2 * lane;
  if (r.owner()) {
    float* to = partial(a, w, w.chunk) + place;
    st_agent2(to, x.m, x.l);
#pragma unroll
    for (int i = 0; i < N; i += 2) st_agent2(to + 64 * (2 + i), x.o[i / 16][i % 16], x.o[i / 16][i % 16 + 1]);
  }
  if (!last_to_arrive(a.counter + w.part0, w.chunks, flag)) return false;
  x = Running<D>();
  if (r.active) {
    float m[2], l[2], o[2][N];
    auto load = [&](int b, int c) {
      const float* at = partial(a, w, min(c, w.chunks - 1)) + place;
      ld_agent2(at, m[b], l[b]);
#pragma unroll
      for (int i = 0; i < N; i += 2) ld_agent2(at + 64 * (2 + i), o[b][i], o[b][i + 1]);
    };
    auto add = [&](int b, int c) {
      if (c >= w.chunks) return;
      const float mn = fmaxf(x.m, m[b]), base = mn == neg_inf() ? 0.f : mn;
      const float f0 = weight_of<sizeof(T) == 2>(x.m - base), f1 = weight_of<sizeof(T) == 2>(m[b] - base);
      x.m = mn;
      x.l = x.l * f0 + l[b] * f1;
#pragma unroll
      for (int i = 0; i < N; ++i) x.o[i / 16][i % 16] = x.o[i / 16][i % 16] * f0 + o[b][i] * f1;
    };
    load(0, r.sub);
    for (int c = r.sub; c < w.chunks; c += 2 * r.ks) {
      load(1, c + r.ks);
      add(0, c);
      if (c + 2 * r.ks < w.chunks) load(0, c + 2 * r.ks);
      add(1, c + r.ks);
    }
  }
  join_waves<T, D>(r, x.o, x.m, x.l, lds, ml, lane);
  return true;
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
    g.id[i] = paged::ld_uniform(table + min((key + 16 * i) >> a.page_log2, a.p.max_pages - 1));
  return g;
}

// Merges the waves' results in LDS into the output, or into the chunk's partial; true in the last
// workgroup of a tile of several chunks.
template <bool LOG2, int W, int ROWS, typename T, int D>
__device__ __forceinline__ bool merge_waves(const TileArgs<T>& a, const Work& w,
                                            const float (&o)[W][ROWS][D], const float (&m)[W][ROWS],
                                            const float (&l)[W][ROWS], int* flag) {
  for (int e = threadIdx.x; e < w.rows * D; e += 64 * W) {
    const int r = e / D, col = e % D;
    Merged<LOG2> x;
#pragma unroll
    for (int i = 0; i < W; ++i) x.add(m[i][r], l[i][r], o[i][r][col]);
    if (w.chunks == 1) {
      const RowPlace p = row_place<D>(w, a.group, r);
      a.out[(w.first + p.t) * a.ld_out + p.col + col] = Elem<T>::from(x.value());
    } else {
      float* to = partial(a, w, w.chunk) + (size_t)r * (D + 2);
      st_agent(to + 2 + col, x.o);
      if (col == 0) st_agent2(to, x.m, x.l);
    }
  }
  return w.chunks > 1 &&
         last_to_arrive(a.counter + w.part0, w.chunks, flag);
}

// ------------------------------------------------------------------------ a few rows

// NR rows (1 to most_rows(): a token of as many query heads, or a few tokens): products on the VALU, as
// decode.hip's. Every 16-byte load of a wave covers whole rows of a page, all of a wave's loads are in flight
// before any arithmetic, and nothing passes through LDS before the waves are merged. A chunk is one round of
// loads of eight waves: `chunk` is few_keys().
constexpr int kRowWaves = 8, kRowLoads = 8;
template <typename T, int D>
__host__ __device__ constexpr int few_keys() {
  return kRowWaves * kRowLoads * 64 / (D / Elem<T>::kPer16B);
}

template <typename T, int D, int NR>
__global__ __launch_bounds__(64 * kRowWaves) void paged_rows_kernel(const TileArgs<T> a) {
  constexpr int EPL = Elem<T>::kPer16B, LPR = D / EPL, KPL = 64 / LPR, NLD = kRowLoads;
  constexpr int KW = NLD * KPL, W = kRowWaves;
  static_assert(KPL <= 16, "the rows of a load lie in one page");
  struct Waves {
    float o[W][NR][D], m[W][NR], l[W][NR];
  };
  // the waves' results; in the end merged chunks
  __shared__ __attribute__((aligned(16))) char lds[W * NR * D * sizeof(Merged<true>)];
  static_assert(sizeof(lds) >= sizeof(Waves), "the waves' results fit");
  Waves& sm = *reinterpret_cast<Waves*>(lds);
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, sub = lane % LPR, grp = lane / LPR;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_few(a);
  if (w.none()) return;
  const int head = w.head, key0 = w.key0 + wave * KW;

  float m[NR], l[NR], o[NR][EPL];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r] = neg_inf();
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[r][e] = 0.f;
  }
  if (key0 < w.key1) {  // wave-uniform
    // Rows past the end take the place of the last one, loads past it of the wave's first: in a page, and
    // masked below.
    const int* table = a.p.table + (size_t)w.seq * a.p.max_pages;
    bool bad[NLD], any_bad = false;
    size_t at[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int ki = key0 + i * KPL, k = ki < w.key1 ? ki : key0;
      const int id = paged::ld_uniform(table + (k >> a.page_log2));
      bad[i] = !paged::is_page(a.p, id);
      any_bad = any_bad || bad[i];
      at[i] = paged::page_row(a.p, bad[i] ? 0 : id, head, k & (a.p.page - 1));  // (there is a page 0)
    }
    u32x4 q[NR];
    int after[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const RowPlace p = row_place<D>(w, a.group, min(r, w.rows - 1));
      after[r] = w.token + p.t;
      q[r] = ld_g128u(a.q + (w.first + p.t) * a.ld_q + p.col + sub * EPL);
    }
    u32x4 kr[NLD], vr[NLD];
    auto row = [&](int i) {
      const int left = w.key1 - 1 - (key0 + i * KPL);  // below 0: the wave's first row
      return (size_t)max(min(grp, left), 0) * D + sub * EPL;
    };
#pragma unroll
    for (int i = 0; i < NLD; ++i) kr[i] = ld_stream(a.k_pages + at[i] + row(i));
#pragma unroll
    for (int i = 0; i < NLD; ++i) vr[i] = ld_stream(a.v_pages + at[i] + row(i));
    __builtin_amdgcn_sched_barrier(0);  // all of them stay in flight
    if (any_bad) {
#pragma unroll
      for (int i = 0; i < NLD; ++i)
        if (bad[i]) kr[i] = u32x4{0u, 0u, 0u, 0u}, vr[i] = u32x4{0u, 0u, 0u, 0u};
    }
    float s[NR][NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int key = key0 + i * KPL + grp;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float x = lanes::group_sum<LPR>(Elem<T>::dot(q[r], kr[i])) * a.scale;
        const bool seen = key < w.key1 && !bad[i] && (NR == 1 || key <= after[r]);
        s[r][i] = seen ? x : neg_inf();
        m[r] = fmaxf(m[r], s[r][i]);
      }
    }
    float base[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = lanes::wave_max_of_groups<LPR>(m[r]);
      base[r] = m[r] == neg_inf() ? 0.f : m[r];
    }
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      float v[EPL];
      Elem<T>::unpack(vr[i], v);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float p = fast_exp2(s[r][i] - base[r]);
        l[r] += p;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] = fmaf(p, v[e], o[r][e]);
      }
    }
    // over the row groups: lanes with the same columns
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if constexpr (LPR < 8) {
        l[r] += __shfl_xor(l[r], LPR, 64);
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] += __shfl_xor(o[r][e], LPR, 64);
      }
      constexpr int K0 = LPR < 8 ? 8 : LPR;
      l[r] = lanes::sum_across<K0>(l[r]);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] = lanes::sum_across<K0>(o[r][e]);
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (grp == 0) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) sm.o[wave][r][sub * EPL + e] = o[r][e];
    }
    if (lane == 0) sm.m[wave][r] = m[r], sm.l[wave][r] = l[r];
  }
  __syncthreads();
  if (merge_waves<true, W, NR, T, D>(a, w, sm.o, sm.m, sm.l, &flag))
    merge_tile<true, W, NR, T, D>(a, w, partial(a, w, 0), lds);
}

// ------------------------------------------------------------------------ bf16

// Weights exp2(s c - m) as bf16 operands of the next product, rounded once as the bf16 forward's; their fp32
// sum. (Weights in two parts, as the kernel for up to 32 rows has them, would take the error from 1.25 to 1.4
// times that of the result's rounding to 1.0, and 8 chunks of 256 rows over up to 8192 tokens, 12 heads of 64,
// from 47 to 54 us, 512 rows over 32768 from 75 to 94; in two parts for tiles of up to 32 rows alone, 52 and 85.)
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

// A wave's 16 tokens of a tile of K or V; nothing to read: zeros.
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
  // `rows` of the 16 exist: the others take the last one's place (they are masked, and must be finite where
  // the last one is)
  __device__ __forceinline__ void clip(int rows, int lane) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int r = (n * 64 + lane) / C;
      if (r >= rows) off[n] -= (uint32_t)((r - rows + 1) * D * 2);
    }
  }
  __device__ __forceinline__ void operator()(bf16* tile, const bf16* src, bool there, int wave,
                                             int lane) const {
    bf16* to = tile + wave * 16 * D;
    if (!there) {
#pragma unroll
      for (int n = 0; n < PER; ++n)
        *reinterpret_cast<u32x4*>(to + (n * 64 + lane) * 8) = u32x4{0u, 0u, 0u, 0u};
      return;
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) dma_lds16_sbase(src, off[n], to + n * 64 * 8);
  }
};

// Where a workgroup's groups of 16 tokens lie: lane i knows it of group i of 64, 16 tiles, so that a tile
// costs a wave two v_readlane. (As scalar lookups and products for each tile, these were half of the scalar
// instructions, which were as many as the vector ones.)
struct Groups {
  uint32_t lo, hi;       // the first element
  uint64_t there, bad;   // has tokens of the workgroup and a page; has no page
  int next;              // page of group 64 + lane
  template <typename T>
  __device__ __forceinline__ Groups(const TileArgs<T>& a, const Work& w, int lane) {
    next = look(a, w, lane);
    advance(a, w, 0, lane);
  }
  template <typename T>
  __device__ __forceinline__ static int look(const TileArgs<T>& a, const Work& w, int group) {
    const int page = (w.key0 + 16 * group) >> a.page_log2;
    return a.p.table[(size_t)w.seq * a.p.max_pages + min(page, a.p.max_pages - 1)];
  }
  // to groups 64 b .. 64 b + 63
  template <typename T>
  __device__ __forceinline__ void advance(const TileArgs<T>& a, const Work& w, int b, int lane) {
    const int key = w.key0 + 16 * (64 * b + lane);
    const bool page = paged::is_page(a.p, next);
    const size_t at = paged::page_row(a.p, page ? next : 0, w.head, key & (a.p.page - 1));
    lo = (uint32_t)at, hi = (uint32_t)(at >> 32);
    there = __builtin_amdgcn_ballot_w64(page && key < w.key1);
    bad = __builtin_amdgcn_ballot_w64(!page);
    next = look(a, w, 64 * (b + 1) + lane);
  }
  __device__ __forceinline__ size_t at(int i) const {
    return (size_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, i) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)lo, i);
  }
};

// 32 keys, the first of them token c0: rows 32 i .. of the tiles ck and cv. `bad`: bits 0 and 1, their first
// and second 16 have no page; mask: that, or some of the rows do not see them all.
template <int D>
__device__ __forceinline__ void keys32(Running<D>& x, const bf16* ck, const bf16* cv, int i, int c0,
                                       bool mask, uint32_t bad, const WaveRows<D>& r,
                                       const bf16x8 (&q)[D / 16], float scale, int lane) {
  constexpr int DB = D / 32;
  const int l32 = lane & 31, hi = lane >> 5;
  f32x16 s{};
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds)
    s = mfma32(lds_op(ck, rm_off<D>(32 * i + sigma32(l32), 2 * ds + hi)), q[ds], s);
  if (mask) {
    const bool bad0 = (bad & 1) != 0, bad1 = (bad & 2) != 0;
    const int last = r.after - c0 - 8 * hi;
#pragma unroll
    for (int y = 0; y < 16; ++y)
      if (reg_row(y, 0) > last || (y < 8 ? bad0 : bad1)) s[y] = neg_inf();
  }
  __builtin_amdgcn_sched_barrier(0);
  bf16x8 va[DB][2], p[2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 2; ++j) va[db][j] = lds_tr_op<D>(cv, 32 * i + 16 * j, 32 * db, lane);
  float sum = weights_bf16(p, s, scale, x.m);
  // 2^64 or more, inf, or NaN (a row's first keys: m is -inf), compared on the bits; both halves of a
  // row take the row's decision, and no other row's bits depend on it
  const bool need = __float_as_uint(sum) >= __float_as_uint(kMaxP);
  if (__builtin_amdgcn_ballot_w64(need) != 0) {
    float mx = s[0];
#pragma unroll
    for (int y = 1; y < 16; ++y) mx = fmaxf(mx, s[y]);
    mx = max_halves(mx) * scale;
    const float mn = or_halves(need) ? fmaxf(x.m, mx) : x.m;
    const float base = mn == neg_inf() ? 0.f : mn;  // no key seen yet weighs anything
    const float f = fast_exp2(x.m - base);
    x.m = mn;
    x.l *= f;
#pragma unroll
    for (int db = 0; db < DB; ++db) x.o[db] *= f;
    sum = weights_bf16(p, s, scale, base);
  }
  x.l += sum;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 2; ++j) x.o[db] = mfma32(va[db][j], p[j], x.o[db]);
}

// The owners' rows into the output, through the wave's own stretch of LDS, so that a store instruction
// covers whole heads.
template <int D>
__device__ __forceinline__ void store_rows(const TileArgs<bf16>& a, const Work& w,
                                           const WaveRows<D>& r, const Running<D>& x, bf16* lds,
                                           int lane) {
  constexpr int C = D / 8;
  if (!r.owner()) return;
  const int l32 = lane & 31, hi = lane >> 5;
  bf16* rows = lds + r.grp * 32 * D;
  const float inv = x.l == 0.f ? 0.f : 1.0f / x.l;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 4 * db + g;
      u32x2 y;
      y[0] = pack_bf16x2(x.o[db][4 * g] * inv, x.o[db][4 * g + 1] * inv);
      y[1] = pack_bf16x2(x.o[db][4 * g + 2] * inv, x.o[db][4 * g + 3] * inv);
      *reinterpret_cast<u32x2*>(rows + l32 * D + ((c ^ (l32 % C)) << 3) + 4 * hi) = y;
    }
#pragma unroll
  for (int n = 0; n < 32 * C / 64; ++n) {
    const int i = (n * 64 + lane) / C, c = (n * 64 + lane) % C;
    const u32x4 y = *reinterpret_cast<const u32x4*>(rows + i * D + ((c ^ (i % C)) << 3));
    if (r.q0 + i < w.rows) {
      const RowPlace at = row_place<D>(w, a.group, r.q0 + i);
      *reinterpret_cast<u32x4*>(a.out + (w.first + at.t) * a.ld_out + at.col + 8 * c) = y;
    }
  }
}

// The lane's query, columns 16 ds + 8 hi + 0 .. 7.
template <int D>
__device__ __forceinline__ void load_query(bf16x8 (&q)[D / 16], const TileArgs<bf16>& a,
                                           const Work& w, const WaveRows<D>& r, int hi) {
  const bf16* row = a.q + (w.first + r.mine.t) * a.ld_q + r.mine.col + 8 * hi;
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) q[ds] = ld_g128(row + 16 * ds);
}
// (once the direct loads' wait is over: the compiler, which does not see those, has none to add then)
template <int D>
__device__ __forceinline__ void take_query(bf16x8 (&q)[D / 16], bool negate) {
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    asm volatile("" : "+v"(q[ds]));
    if (negate) q[ds] = neg_bf16x8(q[ds]);
  }
}

// Up to 16 NB rows, a chunk of 512 keys (1024 at D = 32) for eight waves: a wave takes 64 (128) keys in one
// round, K straight into registers and V through its own stretch of LDS, everything in flight at once and
// no barrier until the waves are merged. (The kernel below, with a tile of 64 keys in flight for the
// workgroup, is a chain of as many memory latencies as a chunk has tiles.) On v_mfma_f32_16x16x32_bf16:
//   S^T[16 keys][16 rows] = K Q^T   A = K as it lies in memory: lane l holds key l % 16, columns 8 (l / 16)
//                                   .. + 7 of each 32
//   O^T[16 columns][16 rows] += V^T P^T over 32 keys, V^T by ds_read_b64_tr_b16
// Of 32 keys, the two tiles of scores take 8 g + r and 8 g + 4 + r as their rows 4 g + r (r < 4): the
// lanes l / 16 = g then hold the weights of keys 8 g .. + 7, the other product's operand. Weights are the sum
// of two bf16 numbers, good to 2^-15, so that a decode step's results are as exact whichever of the kernels for
// a few rows it takes; one number, as in the tiles, costs 0.6 us less of 43 (8 sequences of 4096 to 32768
// tokens, three rows for each of 4 KV heads). The first is cut off, and the second a 2^-20 of the weight
// larger than the rest: neither is 0 or of another sign than the weight, so an infinite value's products are
// the infinity.
typedef __attribute__((ext_vector_type(4))) float acc16;
__device__ __forceinline__ acc16 mfma16(const bf16x8& a, const bf16x8& b, const acc16& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t cut_pair(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float rest_of(float p) {
  return fmaf(p, 1.0f + 0x1p-20f, -__uint_as_float(__float_as_uint(p) & 0xffff0000u));
}
constexpr int kMidWaves = 8;
template <int D>
__host__ __device__ constexpr int mid_wave_keys() {
  return 64 * 64 / D;
}

template <int D, int NB>
__global__ __launch_bounds__(64 * kMidWaves, 4) void paged_mid_bf16_kernel(const TileArgs<bf16> a) {
  constexpr int KW = mid_wave_keys<D>(), NJ = KW / 32, NG = KW / 16, DS = D / 32, DB = D / 16;
  constexpr int W = kMidWaves, ROWS = 16 * NB;
  struct Waves {
    float o[W][ROWS][D], m[W][ROWS], l[W][ROWS];
  };
  constexpr size_t kV = sizeof(bf16) * W * KW * D, kFewBytes = sizeof(Merged<true>) * W * kFew * D;
  constexpr size_t kBytes = kV > sizeof(Waves) ? kV : sizeof(Waves);
  // V; then the waves' results; in the end merged chunks
  __shared__ __attribute__((aligned(16))) char lds[kBytes > kFewBytes ? kBytes : kFewBytes];
  __shared__ int flag;
  Waves& sm = *reinterpret_cast<Waves*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_few(a);
  if (w.none()) return;
  const int head = w.head, key0 = w.key0 + wave * KW;

  float m[NB], l[NB];
  acc16 o[NB][DB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b] = neg_inf();
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[b][d] = acc16{0.f, 0.f, 0.f, 0.f};
  }
  if (key0 < w.key1) {  // wave-uniform
    // The pages of the wave's groups of 16 tokens. What has none is read from the wave's first page, or
    // from page 0, and masked; V has zeros in its place.
    const int* table = a.p.table + (size_t)w.seq * a.p.max_pages;
    bool there[NG], bad[NG];
    size_t at[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int k = key0 + 16 * i < w.key1 ? key0 + 16 * i : key0;
      const int id = paged::ld_uniform(table + (k >> a.page_log2));
      bad[i] = !paged::is_page(a.p, id);
      there[i] = key0 + 16 * i < w.key1 && !bad[i];
      at[i] = paged::page_row(a.p, bad[i] ? 0 : id, head, k & (a.p.page - 1));
    }
    bf16x8 q[NB][DS], kr[NJ][2][DS];
    int after[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const RowPlace p = row_place<D>(w, a.group, min(16 * b + l16, w.rows - 1));
      after[b] = w.token + p.t;
      const bf16* row = a.q + (w.first + p.t) * a.ld_q + p.col + 8 * g4;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) q[b][ds] = ld_g128(row + 32 * ds);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // row l16 of the tile: token 8 (l16 / 4) + 4 t + l16 % 4 of the 32, in group 2 j or 2 j + 1
        const int k = 8 * (l16 >> 2) + 4 * t + (l16 & 3), i = 2 * j + (l16 >> 3);
        const int left = w.key1 - 1 - (key0 + 16 * i);  // below 0: the wave's first row
        const size_t more = at[2 * j + 1] - at[2 * j], base = at[2 * j] + (l16 >> 3 ? more : 0);
        const bf16* row = a.k_pages + base + (size_t)max(min(k & 15, left), 0) * D + 8 * g4;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
          kr[j][t][ds] = as_bf16x8(ld_stream(row + 32 * ds));
      }
    Stage<D> stage(lane);
    bf16* v = reinterpret_cast<bf16*>(lds) + wave * KW * D;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int left = w.key1 - key0 - 16 * i;
      if (there[i] && left < 16) stage.clip(left, lane);  // (the last group that is there)
      stage(v, a.v_pages + at[i], there[i], i, lane);
    }
    wait_vm_lds<0>();
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        asm volatile("" : "+v"(q[b][ds]));
        if (a.negate) q[b][ds] = neg_bf16x8(q[b][ds]);
      }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      acc16 s[NJ][2];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[j][t] = acc16{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) s[j][t] = mfma16(kr[j][t][ds], q[b][ds], s[j][t]);
          // register r: key 8 g4 + 4 t + r of these 32, of group 2 j or 2 j + 1
          const int last = min(after[b], w.key1 - 1) - (key0 + 32 * j + 8 * g4 + 4 * t);
          const bool none = (bad[2 * j] && g4 < 2) || (bad[2 * j + 1] && g4 >= 2);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r > last || none) s[j][t][r] = neg_inf();
            m[b] = fmaxf(m[b], s[j][t][r]);
          }
        }
      m[b] = lanes::max_xor32(lanes::max_xor16(m[b])) * a.scale;
      const float base = m[b] == neg_inf() ? 0.f : m[b];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        u32x4 p, rest;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const float p0 = fast_exp2(fmaf(s[j][t][r], a.scale, -base));
            const float p1 = fast_exp2(fmaf(s[j][t][r + 1], a.scale, -base));
            l[b] += p0 + p1;
            p[2 * t + r / 2] = cut_pair(p0, p1);
            rest[2 * t + r / 2] = pack_bf16x2(rest_of(p0), rest_of(p1));
          }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          s16x4 x[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int row = 32 * j + 8 * g4 + 4 * half + (l16 >> 2), col = 16 * d + 4 * (l16 & 3);
            const lds_bf16* at = (const lds_bf16*)v + row * D + (((col >> 3) ^ swz<D>(row)) << 3) +
                                 (col & 7);
            x[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
          }
          const bf16x8 vt = __builtin_bit_cast(
              bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
          o[b][d] = mfma16(vt, as_bf16x8(rest), o[b][d]);
          o[b][d] = mfma16(vt, as_bf16x8(p), o[b][d]);
        }
      }
      l[b] = lanes::sum_xor32(lanes::sum_xor16(l[b]));
    }
  }
  __syncthreads();  // every wave is done with V
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int row = 16 * b + l16;
    if (row >= w.rows) continue;
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *reinterpret_cast<f32x4*>(&sm.o[wave][row][16 * d + 4 * g4]) =
          f32x4{o[b][d][0], o[b][d][1], o[b][d][2], o[b][d][3]};
    if (g4 == 0) sm.m[wave][row] = m[b], sm.l[wave][row] = l[b];
  }
  __syncthreads();
  if (merge_waves<true, W, ROWS, bf16, D>(a, w, sm.o, sm.m, sm.l, &flag))
    merge_tile<true, W, kFew, bf16, D>(a, w, partial(a, w, 0), lds);
}

template <int D>
__global__ __launch_bounds__(kThreads, 3) void paged_bf16_kernel(const TileArgs<bf16> a) {
  constexpr int DB = D / 32;
  // two tiles of K, two of V; in the end the waves' partials, output rows or merged chunks
  __shared__ __attribute__((aligned(16))) bf16 lds[4 * kTileRows * D];
  bf16 *const sk[2] = {lds, lds + kTileRows * D};
  bf16 *const sv[2] = {lds + 2 * kTileRows * D, lds + 3 * kTileRows * D};
  __shared__ float sm_ml[kWaves - 1][2][64];
  __shared__ int flag;
  static_assert(sizeof(lds) >= (kWaves - 1) * DB * sizeof(AccLds), "waves' partials fit");
  static_assert(sizeof(lds) >= kWaves * 32 * D * sizeof(bf16), "output rows fit");

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_tile(a, lane);
  if (w.none()) return;
  const WaveRows<D> r(w, a.group, wave, l32);

  bf16x8 q[D / 16];
  load_query<D>(q, a, w, r, hi);

  const int n_tiles = w.key1 > w.key0 ? (w.key1 - w.key0 + 63) / 64 : 0;
  Stage<D> stage(lane);
  Groups g(a, w, lane);
  auto load = [&](int t, bf16* tk, bf16* tv) {
    if (t % 16 == 0 && t > 0) g.advance(a, w, t / 16, lane);
    const int i = 4 * (t % 16) + wave;
    const bool there = (g.there >> i & 1) != 0;
    const size_t at = g.at(i);
    const int left = w.key1 - (w.key0 + 64 * t + 16 * wave);
    if (there && left < 16) stage.clip(left, lane);
    stage(tk, a.k_pages + at, there, wave, lane);
    stage(tv, a.v_pages + at, there, wave, lane);
  };

  Running<D> x;
  if (n_tiles > 0) load(0, sk[0], sv[0]);
  wait_vm_lds<0>();
  __builtin_amdgcn_s_barrier();
  take_query<D>(q, a.negate);

  // blocks of 32 keys that some of the wave's rows see, and that all of them do
  const int some = !r.active ? 0 : (min(r.some_see + 1, w.key1) - w.key0 + 31) / 32;
  const int all = (r.all_see + 1 - w.key0) / 32;
  auto tile = [&](int t, const bf16* ck, const bf16* cv, bf16* nk, bf16* nv) {
    const uint32_t bad = (uint32_t)(g.bad >> 4 * (t % 16)) & 15;
    if (t + 1 < n_tiles) load(t + 1, nk, nv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int block = 2 * t + i;
      if (((block & (r.ks - 1)) == r.sub) & (block < some))
        keys32<D>(x, ck, cv, i, w.key0 + 32 * block, (block >= all) | (bad != 0), bad >> 2 * i, r, q,
                  a.scale, lane);
    }
    wait_vm_lds<0>();
    __builtin_amdgcn_s_barrier();
  };
  for (int t = 0; t < n_tiles; t += 2) {
    tile(t, sk[0], sv[0], sk[1], sv[1]);
    if (t + 1 < n_tiles) tile(t + 1, sk[1], sv[1], sk[0], sv[0]);
  }
  x.l = sum_halves(x.l);
  join_waves<bf16, D>(r, x.o, x.m, x.l, lds, sm_ml, lane);
  if (w.chunks > 1 && !merge_chunks<bf16, D>(a, w, r, x, lds, sm_ml, &flag, lane)) return;
  store_rows<D>(a, w, r, x, lds, lane);
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

// The three planes of a product of x3.hpp leave NaN of an infinity (inf - inf in the split, or cross terms of
// unlike signs): what the first planes' product makes infinite is infinite, and counts as that. (An element
// that rounds to an infinity in bf16, above 3.39e38, is taken for one.)
template <int D>
__device__ __forceinline__ void infinite_scores(f32x16& s, const bf16* planes, int row0,
                                                const X3 (&q)[D / 16], int lane) {
  bool odd = false;
#pragma unroll
  for (int x = 0; x < 16; ++x) odd = odd || !(fabsf(s[x]) < __builtin_inff());
  if (__builtin_amdgcn_ballot_w64(odd) == 0) return;
  const int krow = row0 + sigma32(lane & 31), hi = lane >> 5;
  f32x16 first = zero16();
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds)
    first = mfma32(lds_op(planes, rm_off<D>(krow, 2 * ds + hi)), q[ds].v[0], first);
#pragma unroll
  for (int x = 0; x < 16; ++x)
    if (fabsf(first[x]) == __builtin_inff()) s[x] = first[x];
}

// accumulate_t_p, with such values in the product of the first planes alone.
template <int D>
__device__ __forceinline__ void accumulate_infinite(f32x16 (&acc)[D / 32], const bf16* planes, int row0,
                                                    const f32x16& p, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[8 * j + e];
    const X3 pb = split3(x);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      u32x4 a[3];
#pragma unroll
      for (int pl = 0; pl < 3; ++pl)
        a[pl] = as_u32x4(lds_tr_op<D>(planes + pl * kTileRows * D, row0 + 16 * j, 32 * db, lane));
      const bf16x8 all = as_bf16x8(a[0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = (a[0][e] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
        const uint32_t hi = (a[0][e] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
#pragma unroll
        for (int pl = 0; pl < 3; ++pl) a[pl][e] &= ~(lo | hi);
      }
      const X3 v{{as_bf16x8(a[0]), as_bf16x8(a[1]), as_bf16x8(a[2])}};
      acc[db] = mfma32(v.v[1], pb.v[1], acc[db]);  // (in mfma_x6's order)
      acc[db] = mfma32(v.v[2], pb.v[0], acc[db]);
      acc[db] = mfma32(v.v[0], pb.v[2], acc[db]);
      acc[db] = mfma32(v.v[1], pb.v[0], acc[db]);
      acc[db] = mfma32(v.v[0], pb.v[1], acc[db]);
      acc[db] = mfma32(all, pb.v[0], acc[db]);
    }
  }
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void paged_f32_kernel(const TileArgs<float> a) {
  constexpr int DB = D / 32, kPlane = 3 * kTileRows * D, kPitch = D + 4;
  // K and V as three bf16 planes each; in the end the waves' partials, output rows or merged chunks
  __shared__ __attribute__((aligned(16))) bf16 planes[2 * kPlane];
  __shared__ float sm_ml[kWaves - 1][2][64];
  __shared__ int flag;
  static_assert(sizeof(planes) >= (kWaves - 1) * DB * sizeof(AccLds), "waves' partials fit");
  static_assert(sizeof(planes) >= kWaves * 32 * kPitch * sizeof(float), "output rows fit");

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = find_tile(a, lane);
  if (w.none()) return;
  const WaveRows<D> r(w, a.group, wave, l32);

  X3 q[D / 16];  // the lane's query, split
  load_split_row<D>(q, a.q + (w.first + r.mine.t) * a.ld_q + r.mine.col, hi);
  Running<D> x;
  f32x16(&o)[DB] = x.o;
  float &m = x.m, &l = x.l;

  const int head = w.head, n_tiles = w.key1 > w.key0 ? (w.key1 - w.key0 + 63) / 64 : 0;
  // The walk over the tiles. INFINITE: for scores and values that are infinite, which become NaN otherwise.
  auto walk = [&](auto infinite) {
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
        if constexpr (infinite()) infinite_scores<D>(s, planes, 32 * i, q, lane);
        float sum;
        f32x16 p;
        auto weights = [&](float base) {
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const float y = fmaf(s[x], a.scale, -base);
            p[x] = exp_acc(y);
            if constexpr (infinite()) p[x] = y == neg_inf() ? 0.f : p[x];  // (exp_acc's is NaN)
          }
          if (partly) {
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (hidden(x)) p[x] = 0.f;
          }
          sum = p[0];
#pragma unroll
          for (int x = 1; x < 16; ++x) sum += p[x];
        };
        weights(m);
        // as in the bf16 kernel; a row that needs it sees a key of these
        const bool need = __float_as_uint(sum) >= __float_as_uint(kMaxW);
        if (__builtin_amdgcn_ballot_w64(need) != 0) {
          float mx = neg_inf();
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (!(partly && hidden(x))) mx = fmaxf(mx, s[x] * a.scale);
          mx = max_halves(mx);
          const float mn = or_halves(need) ? fmaxf(m, mx) : m;
          const float base = mn == neg_inf() ? 0.f : mn;  // no key seen yet weighs anything
          const float f = weight_of<false>(m - base);
          m = mn;
          l *= f;
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] *= f;
          weights(base);
        }
        l += sum;
        if constexpr (infinite())
          accumulate_infinite<D>(o, planes + kPlane, 32 * i, p, lane);
        else
          accumulate_t_p<D, kTileRows>(o, planes + kPlane, 32 * i, p, lane);
      }
      now = next;
      next = after_next;
    }
    __syncthreads();  // the tiles are read
  };
  if (tid == 0) flag = 0;
  walk(std::false_type{});
  // (a NaN in a sum stays, so that one look at the end is enough, and costs no tile anything)
  bool nan = !(l == l);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) nan = nan || !(o[db][i] == o[db][i]);
  if (nan) flag = 1;
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(flag) != 0) {
    x = Running<D>();
    walk(std::true_type{});
  }
  l = sum_halves(l);
  join_waves<float, D>(r, o, m, l, planes, sm_ml, lane);
  if (w.chunks > 1 &&
      !merge_chunks<float, D>(a, w, r, x, planes, sm_ml, &flag, lane))
    return;
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
}

// ------------------------------------------------------------------------ host

// The kernel of a step, by the rows of a (sequence, KV head): the VALU's up to 2 (fp32: 4); bf16 up to 32: a
// wave for itself; tiles of 128. At 8 sequences of 1 to 32768 tokens, 4 KV heads of 64, in bf16, the first two
// take 31 and 40 us with one row, 41 and 41 with 2, 47 and 42 with 3; the tiles 49 with 3, where the second
// still takes 49 with 8 and 57 with 16.
enum Path { kRows, kMid, kTiles };
constexpr int kMostMid = 32;
constexpr int most_rows(int elem) { return elem == 2 ? 2 : 4; }
Path path_of(const PagedStep& s, int elem) {
  const long long rows = (long long)s.max_rows * (s.H / s.Hkv);
  return rows <= most_rows(elem) ? kRows : elem == 2 && rows <= kMostMid ? kMid : kTiles;
}

struct Plan {
  Path path;
  int tiles, chunk, n_chunk, slots, rows, part_pitch;
  size_t counters, partials;  // bytes
};

long long tiles_of(const PagedStep& s) {
  const long long group = s.H / s.Hkv, per_seq = (s.max_rows * group + kTile - 1) / kTile;
  return std::min(s.n_seq * per_seq, s.n_seq + s.rows * group / kTile);
}
// Of find_tile()'s list: with T the sum that it shares out, the tiles' lengths add up to 2 T at most, and a
// chunk has T Hkv / kShares keys at least, so a KV head has no more than 2 kShares / Hkv chunks besides the
// first ones; and no more than twice that of tiles that are cut.
long long places_of(const PagedStep& s) { return tiles_of(s) + 2 * kShares / s.Hkv + 1; }
long long slots_of(const PagedStep& s) {
  const long long most = ((long long)s.max_pages * s.page + 255) / 256;  // (a chunk has 256 keys at least)
  return most <= 1 ? 0
                   : std::min({places_of(s), 4LL * kShares / s.Hkv + 1, tiles_of(s) * most});
}
int mid_keys_of(int D) { return kMidWaves * (D == 64 ? mid_wave_keys<64>() : mid_wave_keys<32>()); }
int few_keys_of(int elem, int D) {
  return elem == 2 ? (D == 64 ? few_keys<bf16, 64>() : few_keys<bf16, 32>())
                   : (D == 64 ? few_keys<float, 64>() : few_keys<float, 32>());
}

// The lengths are on the device: there is room for every sequence at its longest.
Plan plan_of(const PagedStep& s, int elem) {
  const long long group = s.H / s.Hkv, max_len = (long long)s.max_pages * s.page;
  Plan p{};
  p.path = path_of(s, elem);
  p.rows = (int)std::min(s.max_rows * group, (long long)kTile);
  long long parts = 0;
  if (p.path == kTiles) {
    p.part_pitch = (p.rows + 31) / 32 * group_floats(s.D);
    p.slots = (int)slots_of(s);
    parts = (long long)p.slots * s.Hkv;
  } else {
    p.part_pitch = p.rows * (s.D + 2);
    p.chunk = p.path == kRows ? few_keys_of(elem, s.D) : mid_keys_of(s.D);
    p.n_chunk = (int)((max_len + p.chunk - 1) / p.chunk);
    if (p.n_chunk > 1) parts = (long long)s.n_seq * s.Hkv * p.n_chunk;
  }
  p.counters = parts * sizeof(unsigned);
  p.partials = parts * p.part_pitch * sizeof(float);
  return p;
}

template <typename T, typename F>
hipError_t launch_paged_t(T* out, long long ld_out, const T* q, long long ld_q, const T* k_pages,
                          const T* v_pages, const PagedStep& s, float scale, void* workspace,
                          size_t workspace_bytes, F launch) {
  const Plan plan = plan_of(s, sizeof(T));
  TileArgs<T> a{};
  a.out = out, a.q = q, a.k_pages = k_pages, a.v_pages = v_pages;
  a.ld_out = ld_out, a.ld_q = ld_q, a.p = s;
  a.group = s.H / s.Hkv;
  a.page_log2 = __builtin_ctz((unsigned)s.page);
  a.chunk = plan.chunk, a.n_chunk = plan.n_chunk, a.slots = plan.slots;
  a.rows = plan.rows, a.part_pitch = plan.part_pitch;
  // bf16: masked scores are -inf before they are scaled, so the factor is kept above 0: at 1e-30 every score
  // weighs the same, as at a scale of 0 (as attn_fwd_bf16.hip).
  a.scale = sizeof(T) == 2 ? fmaxf(fabsf(scale) * kLog2e, 1e-30f) : scale;
  a.negate = scale < 0.f;
  if (plan.path == kRows) a.scale = scale * kLog2e;  // (masked after it)
  if (plan.partials > 0) {
    // the caller checked workspace_bytes >= paged_workspace_needed(); partials against its end
    const size_t at = (workspace_bytes - plan.partials) & ~(size_t)15;
    a.counter = static_cast<unsigned*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
  }
  const dim3 grid = plan.path == kTiles ? dim3(s.Hkv, (unsigned)places_of(s))
                                        : dim3(s.Hkv, s.n_seq, plan.n_chunk);
  launch(a, grid, plan.path);
  return hipGetLastError();
}

template <typename T>
void launch_rows(const TileArgs<T>& a, dim3 grid, hipStream_t stream) {
  auto run = [&](auto d) {
    auto rows = [&](auto nr) { paged_rows_kernel<T, d(), nr()><<<grid, 64 * kRowWaves, 0, stream>>>(a); };
    if (a.rows == 1) return rows(std::integral_constant<int, 1>{});
    if constexpr (most_rows(sizeof(T)) > 2) {
      if (a.rows == 4) return rows(std::integral_constant<int, 4>{});
      if (a.rows == 3) return rows(std::integral_constant<int, 3>{});
    }
    rows(std::integral_constant<int, 2>{});
  };
  if (a.p.D == 64)
    run(std::integral_constant<int, 64>{});
  else
    run(std::integral_constant<int, 32>{});
}

}  // namespace

bool paged_fits(const PagedStep& step, int elem) {
  return path_of(step, elem) != kTiles || places_of(step) <= 65535;  // (of n_seq: the caller's check)
}

size_t paged_workspace_needed(const PagedStep& step, int elem) {
  const Plan p = plan_of(step, elem);
  return p.partials > 0 ? p.counters + p.partials + 16 : 0;
}

// The most counters and the most partials, of tiles or of a few rows, each of which grows with every argument:
// counters lie at the front and partials at the end, so that a step's partials never reach another's counters,
// which stay at zero between calls.
size_t paged_workspace_bytes(const PagedStep& s) {
  const long long group = s.H / s.Hkv, max_len = (long long)s.max_pages * s.page;
  const long long tile_rows = std::min((s.max_rows * group + 31) / 32 * 32, (long long)kTile);
  long long counters = slots_of(s) * s.Hkv, floats = counters * tile_rows * (s.D + 4);
  if (group <= kMostMid) {
    const int keys = std::min({few_keys_of(2, s.D), few_keys_of(4, s.D), mid_keys_of(s.D)});
    const long long n_chunk = (max_len + keys - 1) / keys;
    const long long parts = n_chunk > 1 ? s.n_seq * s.Hkv * n_chunk : 0;
    counters = std::max(counters, parts);
    floats = std::max(floats, parts * std::min<long long>(s.max_rows * group, kMostMid) * (s.D + 2));
  }
  return counters > 0 ? counters * sizeof(unsigned) + floats * sizeof(float) + 16 : 0;
}

hipError_t launch_paged_attention_bf16(bf16* out, long long ld_out, const bf16* q, long long ld_q,
                                       const bf16* k_pages, const bf16* v_pages,
                                       const PagedStep& step, float scale, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  return launch_paged_t<bf16>(
      out, ld_out, q, ld_q, k_pages, v_pages, step, scale, workspace, workspace_bytes,
      [&](const TileArgs<bf16>& a, dim3 grid, Path path) {
        if (path == kRows) {
          launch_rows(a, grid, stream);
        } else if (path == kMid) {
          auto run = [&](auto d, auto nb) {
            paged_mid_bf16_kernel<d(), nb()><<<grid, 64 * kMidWaves, 0, stream>>>(a);
          };
          constexpr std::integral_constant<int, 64> d64;
          constexpr std::integral_constant<int, 32> d32;
          constexpr std::integral_constant<int, 1> one;
          constexpr std::integral_constant<int, 2> two;
          if (step.D == 64)
            a.rows <= 16 ? run(d64, one) : run(d64, two);
          else
            a.rows <= 16 ? run(d32, one) : run(d32, two);
        } else if (step.D == 64)
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
      [&](const TileArgs<float>& a, dim3 grid, Path path) {
        if (path == kRows)
          launch_rows(a, grid, stream);
        else if (step.D == 64)
          paged_f32_kernel<64><<<grid, kThreads, 0, stream>>>(a);
        else
          paged_f32_kernel<32><<<grid, kThreads, 0, stream>>>(a);
      });
}

}  // namespace dadgpt
