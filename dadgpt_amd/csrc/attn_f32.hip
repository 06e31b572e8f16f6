// fp32 causal flash attention at fp32 accuracy on gfx950. This is the reference's precision
// (cuda/attention.cu:1): forward with online softmax and a saved natural-log logsumexp, backward
// recomputing the probabilities from it. Every fp32 product runs on the bf16 matrix cores,
// each float split into three bf16 values and each product formed from the six cross terms
// that matter (see X3 below: as accurate as the fp32 MFMA, in 37% of its matrix time, and
// beside the VALU, which the fp32 MFMA of gfx950 does not run beside). The softmax
// exponentials are exp_acc (below: 1.24 ulp in six VALU operations, the library expf 0.85 in
// thirteen) and the logsumexp's logarithm is logf; results match float64 to ~1e-6 (O, lse)
// and the fp32 CPU path within its own rounding. The forward moves its running maximum lazily
// (as the bf16 forward does) and masking runs only where a chunk needs it.
//
// Work decomposition (every product a 32 x 32 MFMA tile, one wave per 32 rows):
//  forward  a wave owns 32 queries (lane l holds query l % 32): S^T = K Q^T over each 32-key
//           chunk with Q in registers (split once), the online softmax per lane, O^T += V^T P^T
//           with P split from the score registers (the K rows are read through sigma32, so
//           score registers 8j..8j+7 of lane half h are the MFMA k-slice of that half: no lane
//           exchange). K and V tiles are split once per workgroup as they are staged, into
//           three bf16 planes each in the bf16 kernels' swizzled layout, read with
//           ds_read_b128 (K rows) and ds_read_b64_tr_b16 (V^T);
//  dK/dV    a wave owns 32 keys (lane l holds key l % 32) and walks the later query chunks:
//           S = Q K^T and dP = dO V^T with K and V split once (in registers; at d_head 64 V's two
//           lower planes in LDS), Q and dO as bf16 planes, P and dS in registers, dV^T += dO^T P
//           and dK^T += Q^T dS (no atomics);
//  dQ       a wave owns 32 queries again: S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T, with
//           Q and dO split once and K, V as bf16 planes;
//  delta    rowsum(dO * O), computed by the backward's workgroups or, for long rows, by a pass of
//           its own.
// dK/dV and dQ are workgroups of one launch. One or two waves share a row group's chunks, by the
// size of the grid (fwd_waves_per_group, bwd_waves_per_group).
// The next tile is loaded while the current one is on the matrix cores and split into planes as
// it is stored: through registers in the forward; in dK/dV and dQ by direct loads into LDS,
// which leaves the registers to the split operands (splitting dO, K and V once instead of at
// each use: B16 H12 S1024 backward 606 -> 528 us, bit-identical).
//
// The DROP instantiations apply attention-probability dropout with the keep bits of
// dropout.hpp: the forward and dQ hold keys along registers (keep_words16), dK/dV holds queries
// along registers (keep_col16).
#include <type_traits>

#include "common.hpp"
#include "dropout.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "tiles.hpp"
#include "window.hpp"
#include "x3.hpp"

namespace dadgpt {
namespace {

// A workgroup is KG x KS waves: KG row groups of 32 rows (queries, or keys in dK/dV) it owns,
// and KS waves per group that share its chunks of the other dimension. The staged tile has
// 32 KS rows; wave (g, s) of a workgroup computes group g against the tile's chunk s, and the KS
// partial results are merged through LDS at the end.
constexpr int kGroups = 4;
constexpr int kRows = 32 * kGroups;  // rows a workgroup owns
// At most 256 registers a lane (two waves per SIMD; one runs the backward ~15% slower).
constexpr int wgs_per_cu(int ks) { return 2 / ks; }
// The windowed kernels also have KG = 2 with KS = 2, for grids that leave CUs idle: at D = 64 its
// tiles leave a CU room for one such workgroup.
constexpr int wgs_per_cu(int ks, int kg, int d) {
  return kg == kGroups ? wgs_per_cu(ks) : d == 64 ? 1 : 2;
}

constexpr int kPitchPad = 4;  // epilogues stage rows of D floats at a pitch of D + 4

// A TR-row fp32 tile and its register prefetch by NT threads, TR*D/(4 NT) 16-byte pieces each;
// rows at or past S read as zeros.
template <int D, int TR, int NT>
struct Tile {
  static constexpr int kPieces = TR * D / 4 / NT;
  static constexpr int kThreads = NT;
  f32x4 r[kPieces];

  __device__ __forceinline__ void load(const float* src, int row0, int S) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int u = threadIdx.x + NT * i, row = u / (D / 4), c = u % (D / 4);
      r[i] = row0 + row < S ? *reinterpret_cast<const f32x4*>(src + (size_t)(row0 + row) * D +
                                                              4 * c)
                            : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  __device__ __forceinline__ f32x4 piece(int i) const { return r[i]; }
};

// The same tile prefetched through LDS instead of registers: each lane's pieces travel by direct
// global -> LDS loads into the lane's own 16-byte slots, so a wave reads back only what it
// loaded itself and needs no barrier, just its own wait. Rows at or past S read row S-1.
template <int D, int TR, int NT>
struct RawTile {
  static constexpr int kPieces = TR * D / 4 / NT;
  static constexpr int kThreads = NT;
  const float* src;
  float* lds;  // TR * D floats
  int S, wave, lane;
  __device__ __forceinline__ void issue(int row0) const {
    const int left = S - 1 - row0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int u = NT * i + 64 * wave + lane, row = u / (D / 4), c = u % (D / 4);
      dma_lds16_sbase(src + (size_t)row0 * D, (uint32_t)(min(row, left) * D + 4 * c) * 4u,
                      lds + 4 * (NT * i + 64 * wave));
    }
  }
  __device__ __forceinline__ f32x4 piece(int i) const {
    return *reinterpret_cast<const f32x4*>(lds + 4 * (NT * i + 64 * wave + lane));
  }
};

// score_tile_p and accumulate_t_p at the start of `planes`, with the addresses from
// LaneLds (tiles.hpp): the dK/dV kernel's register relief. At D = 64 the kernel uses all 256: the
// one-wave instances without dropout and the two-wave ones with it keep one or two registers in
// scratch, the others none.
template <int D, int TR>
__device__ __forceinline__ f32x16 score_tile_px(const bf16* planes, const X3 (&b)[D / 16],
                                                const LaneLds& lo) {
  uint32_t ra[D / 16];
  row_addr_xor<D>(ra, lo.ro);
  f32x16 acc = zero16();
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    X3 a;
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) a.v[pl] = lds_row_at(planes + pl * TR * D, ra[ds]);
    acc = mfma_x6(a, b[ds], acc);
  }
  return acc;
}
// score_tile_px with the lower planes of the B operand in LDS (`blo`, by lane).
template <int D, int TR>
__device__ __forceinline__ f32x16 score_tile_pxl(const bf16* planes, const bf16x8 (&b0)[D / 16],
                                                 const bf16x8 (*blo)[2][64], int lane,
                                                 const LaneLds& lo) {
  uint32_t ra[D / 16];
  row_addr_xor<D>(ra, lo.ro);
  f32x16 acc = zero16();
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    X3 a;
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) a.v[pl] = lds_row_at(planes + pl * TR * D, ra[ds]);
    acc = mfma_x6(a, X3{{b0[ds], blo[ds][0][lane], blo[ds][1][lane]}}, acc);
  }
  return acc;
}
template <int D, int TR>
__device__ __forceinline__ void accumulate_t_px(f32x16 (&acc)[D / 32], const bf16* planes,
                                                const f32x16& p, const LaneLds& lo) {
  uint32_t ta[2][D / 32];
  tr_addr_xor<D>(ta, lo.tr);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[8 * j + e];
    const X3 pb = split3(x);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      X3 a;
#pragma unroll
      for (int pl = 0; pl < 3; ++pl)
        a.v[pl] = lds_tr_at(planes + pl * TR * D + 16 * j * D, ta[0][db], ta[1][db]);
      acc[db] = mfma_x6(a, pb, acc[db]);
    }
  }
}

// Writes a wave's transposed accumulators (element r of lane (l32, h), block db: row l32 of
// the wave, column 32 db + c32_row(r, h)) as 32 contiguous rows of D floats through the wave's
// LDS slot `stage` (32 x (D + 4) floats), times `mul` (per lane).
template <int D>
__device__ __forceinline__ void store_rows_t(float* dst, int row0, int S,
                                             const f32x16 (&acc)[D / 32], float mul,
                                             float* stage, int lane) {
  const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      stage[l32 * (D + kPitchPad) + 32 * db + c32_row(r, h)] = acc[db][r] * mul;
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own LDS writes are done
  __builtin_amdgcn_wave_barrier();
  constexpr int kPieces = 32 * D / 4 / 64;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int u = lane + 64 * i, row = u / (D / 4), c = u % (D / 4);
    if (row0 + row < S)
      *reinterpret_cast<f32x4*>(dst + (size_t)(row0 + row) * D + 4 * c) =
          *reinterpret_cast<const f32x4*>(stage + row * (D + kPitchPad) + 4 * c);
  }
}

// ------------------------------------------------------------------------------ forward

// ONCE: the conversions of Q's and the weights' splits forced to happen once (pack_once).
// WIN: sliding window and sinks, as in the bf16 forward.
template <int D, bool DROP, int KS, bool ONCE, bool WIN = false, int KG = kGroups>
__global__ __launch_bounds__(64 * KG * KS, wgs_per_cu(KS, KG, D)) void fwd_f32_kernel(
    float* __restrict__ out, float* __restrict__ lse, const float* __restrict__ q,
    const float* __restrict__ k, const float* __restrict__ v, int S, float scale,
    const DropParams dr, const WindowArg<WIN> win) {
  constexpr int NT = 64 * KG * KS, TR = 64, CPT = 2 / KS;  // chunks per tile and wave
  // K and V tiles as three bf16 planes each; after the tile loop they hold the second waves'
  // partial results, then the epilogue's fp32 staging rows. With two waves per group there are
  // two sets (one workgroup has the CU's LDS to itself), see the tile loop.
  constexpr int kPlane = 3 * TR * D;
  __shared__ __attribute__((aligned(16))) bf16 planes[KS * 2 * kPlane];
  constexpr int kPart = (D / 32) * 1024 + 128;  // a partial: O, m and l (floats)
  constexpr int kStage = 32 * (D + kPitchPad);  // a wave's staged rows (floats)
  static_assert(4 * kPlane >= 4 * KG * (KS > 1 && kPart > kStage ? kPart : kStage),
                "partials and staging fit");
  const int bh = blockIdx.x;
  const int blk = gridDim.y - 1 - blockIdx.y;  // longest query blocks first
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform: scalar
  const int grp = wave % KG, sub = wave / KG;
  const size_t base = (size_t)bh * S * D;
  const int row0 = blk * 32 * KG;          // the workgroup's first query
  const int q0 = row0 + 32 * grp;           // the wave's first query
  const int qi = q0 + l32;                // this lane's query
  const int last = min(S, row0 + 32 * KG) - 1;  // the workgroup's last query
  const KeyTiles<WIN, TR> keys(row0, last, win);
  const int n_tiles = keys.count();

  X3 qb[D / 16];  // the lane's query row, split
  load_split_row<D, ONCE>(qb, q + base + (size_t)min(qi, S - 1) * D, h);
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) o[db] = zero16();
  float m = neg_inf(), lh = 0.f;  // running maximum; this lane half's sum of weights

  Tile<D, TR, NT> tk, tv;
  tk.load(k + base, keys.row(0), S);
  tv.load(v + base, keys.row(0), S);
  // Splits the loaded tile t into `to` and loads tile t + 1.
  auto stage = [&](int t, bf16* to) {
    store_x3<D, TR>(tk, to);
    store_x3<D, TR>(tv, to + kPlane);
    if (t + 1 < n_tiles) {
      tk.load(k + base, keys.row(t + 1), S);
      tv.load(v + base, keys.row(t + 1), S);
    }
  };
  auto compute = [&](int t, const bf16* skp) {
    const bf16* svp = skp + kPlane;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = KS == 1 ? i : sub;
      const int key0 = keys.row(t) + 32 * c;
      if (key0 > q0 + 31) continue;  // wave-uniform: the whole chunk is in the future
      if constexpr (WIN)
        if (!chunk_visible(key0, q0, win)) continue;
      f32x16 s = score_tile_p<D, TR>(skp, 32 * c, qb, lane);
      // only the chunk whose first key is the wave's first query holds keys after a query
      // (or past S); waves are 32-query aligned, so it is the one with key0 == q0
      bool diag = key0 == q0;
      if constexpr (WIN) diag = !chunk_whole(key0, q0, win);
      auto hidden = [&](int u) {
        if constexpr (WIN)
          return HiddenKeys(key0 + 8 * h, qi, win)(reg_row(u, 0));
        else
          return key0 + reg_row(u, h) > qi;
      };
      // weights against the running maximum m as it stands (natural-log units)
      float w[16], ps;
      auto weights = [&](float mref) {
#pragma unroll
        for (int u = 0; u < 16; ++u) w[u] = exp_acc(fmaf(s[u], scale, -mref));
        if (diag) {
#pragma unroll
          for (int u = 0; u < 16; ++u)
            if (hidden(u)) w[u] = 0.f;
        }
        ps = w[0];  // (0 + w[0] could not be folded: it maps -0 to +0)
#pragma unroll
        for (int u = 1; u < 16; ++u) ps += w[u];
      };
      // The maximum moves only when a row's weights would reach 2^64 (or are inf/NaN: m is
      // -inf before a row's first chunk), compared on the bits (ps is +0, positive or NaN).
      // Both lane halves of a row take the row's decision, and only the rows that need it
      // move: the others rescale by exp(0) = 1 and recompute the same weights, so no row's
      // bits depend on another row.
      auto move = [&](bool need) {
        float cm = neg_inf();
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (!(diag && hidden(u))) cm = fmaxf(cm, s[u] * scale);
        // a row that needs it has a visible key in the chunk: its maximum is finite
        const float mn = or_halves(need) ? fmaxf(m, max_halves(cm)) : m;
        // 0 on a row's first chunk (exp_acc has no -inf input path)
        const float alpha = m == neg_inf() ? 0.f : exp_acc(m - mn);
        m = mn;
        lh *= alpha;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      };
      if constexpr (WIN) {
        // with few chunks a row, the first one's weights are not tried against -inf
        const bool none = m == neg_inf();
        if (__builtin_amdgcn_ballot_w64(none) != 0) move(none);  // (wave-uniform)
      }
      weights(m);
      const bool need = __float_as_uint(ps) >= __float_as_uint(kMaxW);
      if (__builtin_amdgcn_ballot_w64(need) != 0) {  // wave-uniform
        move(need);
        weights(m);
      }
      lh += ps;
      KeepWords16 keep = {};
      if constexpr (DROP) keep = keep_words16(dr, (uint64_t)bh * S + qi, key0, h);
#pragma unroll
      for (int u = 0; u < 16; ++u) s[u] = DROP ? w[u] * keep_factor(keep, u, dr) : w[u];
      accumulate_t_p<D, TR, ONCE>(o, svp, 32 * c, s, lane);
    }
  };
  if constexpr (KS == 1) {
    for (int t = 0; t < n_tiles; ++t) {
      __syncthreads();  // the previous tile's reads are done
      stage(t, planes);
      __syncthreads();
      compute(t, planes);
    }
  } else {
    // One barrier per tile: tile t is computed from one set while t + 1 is split into the other.
    // A SIMD holds one wave of each half, and the halves do the two in opposite order: in step,
    // both would be on the matrix cores and then both on the VALU.
    bf16 *set0 = planes, *set1 = planes + 2 * kPlane;
    stage(0, set0);
    __syncthreads();
    auto tile = [&](int t, bf16* cur, bf16* next) {
      if (sub == 1 && t + 1 < n_tiles) stage(t + 1, next);
      compute(t, cur);
      if (sub == 0 && t + 1 < n_tiles) stage(t + 1, next);
      __syncthreads();
    };
    for (int t = 0; t < n_tiles; t += 2) {
      tile(t, set0, set1);
      if (t + 1 < n_tiles) tile(t + 1, set1, set0);
    }
  }
  __syncthreads();  // every wave is done with the tiles: they hold partials and staging now
  constexpr int kSlot = KS > 1 && kPart > kStage ? kPart : kStage;
  float* slot = reinterpret_cast<float*>(planes) + grp * kSlot;
  if constexpr (KS == 2) {
    // (m, l, O) of the group's second wave: rescaled to the larger maximum and added. A wave
    // that saw no chunk has m = -inf and zeros, which get weight 0.
    float* ml = slot + (D / 32) * 1024;
    if (sub == 1) {
      put_acc(o, reinterpret_cast<AccLds*>(slot), lane);
      ml[lane] = m;
      ml[64 + lane] = lh;
    }
    __syncthreads();
    if (sub == 1) return;
    const float m1 = ml[lane], mn = fmaxf(m, m1);
    const float a0 = m == neg_inf() ? 0.f : exp_acc(m - mn);
    const float a1 = m1 == neg_inf() ? 0.f : exp_acc(m1 - mn);
    m = mn;
    lh = lh * a0 + ml[64 + lane] * a1;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= a0;
    add_acc(o, reinterpret_cast<const AccLds*>(slot), lane, a1);
    __builtin_amdgcn_wave_barrier();
  }
  const float l = sum_halves(lh);
  if (h == 0 && qi < S) lse[(size_t)bh * S + qi] = m + logf(l);
  store_rows_t<D>(out + base, q0, S, o, 1.0f / l, slot, lane);
}

// ----------------------------------------------------------------------------- backward

// delta[row] = sum_d dout[row][d] * out[row][d]: D/4 lanes per row, one 16-byte piece each;
// a grid-stride loop over rows (the lanes of a row share every trip, so the row's shuffles
// always see all of its lanes).
template <int D>
__global__ __launch_bounds__(256) void delta_f32_kernel(float* __restrict__ delta,
                                                        const float* __restrict__ dout,
                                                        const float* __restrict__ out,
                                                        long long rows) {
  constexpr int LPR = D / 4;
  const int c = threadIdx.x % LPR;
  const long long stride = (long long)gridDim.x * (256 / LPR);
  for (long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / LPR; row < rows;
       row += stride) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(dout + row * D + 4 * c);
    const f32x4 b = *reinterpret_cast<const f32x4*>(out + row * D + 4 * c);
    float acc = a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
    acc = lanes::group_sum<LPR>(acc);
    if (c == 0) delta[row] = acc;
  }
}

// LDS of the backward kernels (bytes): two streamed tiles of 32 KS rows as three bf16 planes
// each, and raw; afterwards the partials and staging of the epilogue (`acc` accumulators a wave).
template <int D, int KS>
struct BwdLds {
  static constexpr int TR = 32 * KS, kPlane = 3 * TR * D;
  static constexpr int kBytes = 2 * kPlane * 2 + 2 * TR * D * 4;
  static constexpr int slot_floats(int acc) {
    const int stage = 32 * (D + kPitchPad), part = acc * 1024;
    return KS > 1 && part > stage ? part : stage;
  }
};

// What a backward kernel works on.
struct F32BwdArgs {
  float *dq, *dk, *dv, *delta;
  const float *q, *k, *v, *dout, *out, *lse;
  int S;
  float scale;
  DropParams dr;
};
// LDS of a workgroup: the tiles, and per query row of a dK/dV tile lse and delta * scale.
template <int D, int KS, int KG = kGroups>
struct F32BwdShared {
  __attribute__((aligned(16))) char tiles[BwdLds<D, KS>::kBytes];
  __attribute__((aligned(16))) float sl[32 * KS], sd[32 * KS];
  // dK/dV at D = 64: the lower planes of the groups' V rows, by lane
  bf16x8 vlo[KG][D == 64 ? D / 16 : 1][2][64];
};

// delta of rows row0 .. S-1 into LDS, by the whole workgroup: D/4 lanes per row, one 16-byte
// piece each, four groups of rows in flight.
template <int D, int NT>
__device__ __forceinline__ void delta_rows(float* delta, const float* dout, const float* out,
                                           int row0, int S) {
  constexpr int LPR = D / 4, ROWS = NT / LPR, N = 4;
  const int c = threadIdx.x % LPR, lr = threadIdx.x / LPR;
  for (int b0 = row0; b0 < S; b0 += N * ROWS) {
    f32x4 g[N], o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const size_t r = min(b0 + i * ROWS + lr, S - 1);
      g[i] = *reinterpret_cast<const f32x4*>(dout + r * D + 4 * c);
      o[i] = *reinterpret_cast<const f32x4*>(out + r * D + 4 * c);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float acc = g[i][0] * o[i][0] + g[i][1] * o[i][1] + g[i][2] * o[i][2] + g[i][3] * o[i][3];
      acc = lanes::group_sum<LPR>(acc);
      const int r = b0 + i * ROWS + lr;
      if (c == 0 && r < S) delta[r - row0] = acc;
    }
  }
}

// The windowed backward's arguments. A dK/dV workgroup walks the queries up to its key block's
// window (block_end, in rows); a sink key's later queries are up to `pieces` pieces of piece_rows
// rows, and the sums of all lie in `partial`, [BH][block's own, piece 1, ..][dK, dV][sink rows,
// whole 32s][D]. Without pieces a block with sink keys walks all of them.
struct F32WindowBwdArgs : Window {
  int piece_rows, pieces;
  float* partial;
  // of the block of `rows` keys from row0 on; where it holds sink keys, of the 128 keys around it
  __device__ __forceinline__ int block_end(int row0, int rows, int S) const {
    if (row0 < sinks) {
      if (pieces == 0) return S;
      row0 = row0 / kRows * kRows, rows = kRows;
    }
    return min(S, (row0 + rows + window - 2) / 64 * 64 + 64);
  }
  // pieces of a sink key's later queries
  __device__ __forceinline__ int far_pieces(int key, int S) const {
    return (S - block_end(key, 1, S) + piece_rows - 1) / max(piece_rows, 1);
  }
};
template <bool WIN>
struct F32WindowBwdArg {};
template <>
struct F32WindowBwdArg<true> : F32WindowBwdArgs {};

// One workgroup's dK and dV. OWN_DELTA: delta is computed here, into own_delta (a float for each
// row from the first tile on); otherwise it is read from a.delta. WIN: the queries of a key block
// end with its last key's window (piece 0), and what later ones add to a block's sink keys is other
// workgroups' (piece 1, 2, ..): their sums and the block's own sink rows go to the partials, which
// window_join_f32_kernel adds up.
template <int D, bool DROP, int KS, bool OWN_DELTA, bool WIN = false, int KG = kGroups>
__device__ __forceinline__ void dkdv_f32_workgroup(const F32BwdArgs& a, int bh, int blk,
                                                   F32BwdShared<D, KS, KG>& sm, float* own_delta,
                                                   const F32WindowBwdArg<WIN>& win = {},
                                                   int piece = 0) {
  // Q and dO tiles: planes and raw
  using Lds = BwdLds<D, KS>;
  constexpr int TR = Lds::TR, NT = 64 * KG * KS;
  char* smem = sm.tiles;
  bf16 *sqp = reinterpret_cast<bf16*>(smem), *sgp = sqp + Lds::kPlane;
  float* raw = reinterpret_cast<float*>(sgp + Lds::kPlane);
  constexpr int kSlot = Lds::slot_floats(2 * (D / 32));
  static_assert(KG * kSlot * 4 <= Lds::kBytes, "partials and staging fit");
  float *sl = sm.sl, *sd = sm.sd;
  const float *q = a.q, *k = a.k, *v = a.v, *dout = a.dout, *lse = a.lse, *delta = a.delta;
  float *dk = a.dk, *dv = a.dv;
  const int S = a.S;
  const float scale = a.scale;
  const DropParams& dr = a.dr;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform: scalar
  const int grp = wave % KG, sub = wave / KG;
  const size_t base = (size_t)bh * S * D;
  const int row0 = blk * 32 * KG;         // the workgroup's first key
  const int k0 = row0 + 32 * grp;         // the wave's first key
  const int kj = k0 + l32;                // this lane's key
  int t0 = row0 / TR;  // first query tile with a query >= the first key
  int n_tiles = (S + TR - 1) / TR;
  if constexpr (WIN) {
    const int end = win.block_end(row0, 32 * KG, S);
    if (piece > 0) t0 = (end + (piece - 1) * win.piece_rows) / TR;
    n_tiles = (min(S, piece > 0 ? t0 * TR + win.piece_rows : end) + TR - 1) / TR;
    if (t0 >= n_tiles) return;
  }

  // The lane's K and V rows (score-product B layout), split. At D = 64 V's lower planes go to LDS,
  // which the two waves of a group share (published by the first barrier): with all six planes
  // in registers (96 of 256) the loop spilled and the compiler could not move the softmax under
  // the dP products (B16 H12 S1024 513 -> 498 us, with dropout B4 180 -> 153; at D = 32, where
  // they fit, the LDS reads cost 4%).
  constexpr bool kVLds = D == 64;
  X3 kb[D / 16], vb[D / 16];
  load_split_row<D>(kb, k + base + (size_t)min(kj, S - 1) * D, h);
  load_split_row<D>(vb, v + base + (size_t)min(kj, S - 1) * D, h);
  bf16x8 vb0[D / 16];
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    vb0[ds] = vb[ds].v[0];
    if constexpr (kVLds) {
      if (sub == 0) sm.vlo[grp][ds][0][lane] = vb[ds].v[1], sm.vlo[grp][ds][1][lane] = vb[ds].v[2];
      asm volatile("" : "+v"(vb0[ds]));
    }
    // not to be split again inside the loop
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) {
      asm volatile("" : "+v"(kb[ds].v[pl]));
      if constexpr (!kVLds) asm volatile("" : "+v"(vb[ds].v[pl]));
    }
  }
  f32x16 da[2 * (D / 32)];  // dV^T, then dK^T
  f32x16(&dva)[D / 32] = reinterpret_cast<f32x16(&)[D / 32]>(da[0]);
  f32x16(&dka)[D / 32] = reinterpret_cast<f32x16(&)[D / 32]>(da[D / 32]);
#pragma unroll
  for (int i = 0; i < 2 * (D / 32); ++i) da[i] = zero16();

  const LaneLds lo = lane_lds<D>(lane);
  const RawTile<D, TR, NT> tq{q + base, raw, S, wave, lane},
      tg{dout + base, raw + TR * D, S, wave, lane};
  float pl = 0.f, pd = 0.f;
  auto load_stats = [&](int row0) {
    const int r = row0 + (threadIdx.x & (TR - 1));
    pl = r < S ? lse[(size_t)bh * S + r] : 0.f;
    if constexpr (OWN_DELTA)
      pd = 0.f;  // read from own_delta as the tile is staged
    else
      pd = r < S ? delta[(size_t)bh * S + r] : 0.f;
  };
  tq.issue(t0 * TR);
  tg.issue(t0 * TR);
  load_stats(t0 * TR);
  if constexpr (OWN_DELTA)
    delta_rows<D, NT>(own_delta, dout + base, a.out + base, t0 * TR,
                      WIN ? min(S, n_tiles * TR) : S);
  for (int t = t0; t < n_tiles; ++t) {
    wait_vm_lds<0>();  // this wave's pieces of the tile
    __syncthreads();   // every wave is done with the previous tile's planes
    store_x3<D, TR>(tq, sqp);
    store_x3<D, TR>(tg, sgp);
    if (threadIdx.x < TR) {
      if constexpr (OWN_DELTA) pd = own_delta[min(t * TR + (int)threadIdx.x, S - 1) - t0 * TR];
      sl[threadIdx.x] = pl, sd[threadIdx.x] = pd * scale;
    }
    __syncthreads();
    if (t + 1 < n_tiles) {
      tq.issue((t + 1) * TR);
      tg.issue((t + 1) * TR);
      load_stats((t + 1) * TR);
    }
    const int qrow0 = t * TR + 32 * sub;
    // wave-uniform: every query of the chunk precedes every key, or lies past S
    if (qrow0 + 31 < k0 || (KS > 1 && qrow0 >= S)) continue;
    if constexpr (WIN)
      if (!chunk_visible(k0, qrow0, win)) continue;
    const bf16 *qc = sqp + 32 * sub * D, *gc = sgp + 32 * sub * D;
    // lane (l32, h), register u: query qrow0 + reg_row(u, h), key kj
    f32x16 s = score_tile_px<D, TR>(qc, kb, lo);   // Q K^T
    f32x16 dp;  // dO V^T
    if constexpr (kVLds)
      dp = score_tile_pxl<D, TR>(gc, vb0, sm.vlo[grp], lane, lo);
    else
      dp = score_tile_px<D, TR>(gc, vb, lo);
    uint32_t keep = 0;
    if constexpr (DROP) keep = keep_col16(dr, (uint64_t)bh * S + qrow0, k0, lane);
    // P in place of S, under the dP products: registers 8j..8j+7 are the 8 consecutive rows
    // 32 sub + 16j + 8h .., their statistics two 16-byte LDS reads each
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const f32x4 ls =
          *reinterpret_cast<const f32x4*>(sl + 32 * sub + 16 * (g4 >> 1) + 8 * h + 4 * (g4 & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g4 + e] = exp_acc(fmaf(s[4 * g4 + e], scale, -ls[e]));
    }
    // keys after a query, or rows past S, only where the chunk reaches the wave's first
    // keys or S (wave-uniform)
    bool mask = qrow0 < k0 + 31 || qrow0 + 31 >= S;
    int end = S;
    if constexpr (WIN) {
      mask = qrow0 + 31 >= S || !chunk_whole(k0, qrow0, win);
      if (kj >= win.sinks) end = min(S, kj + win.window);
    }
    if (mask) {
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int qrow = qrow0 + reg_row(u, h);
        s[u] = kj <= qrow && qrow < end ? s[u] : 0.f;
      }
    }
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const f32x4 ds =
          *reinterpret_cast<const f32x4*>(sd + 32 * sub + 16 * (g4 >> 1) + 8 * h + 4 * (g4 & 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = 4 * g4 + e;
        const float p = s[u];
        float g = dp[u];
        if constexpr (DROP) {
          const float f = keep_factor(keep, u, dr.scale);
          g *= f;
          s[u] = p * f;  // the probability that multiplied V
        }
        dp[u] = p * fmaf(g, scale, -ds[e]);  // P (dP - delta) scale
      }
    }
    accumulate_t_px<D, TR>(dva, gc, s, lo);   // dV^T += dO^T P
    accumulate_t_px<D, TR>(dka, qc, dp, lo);  // dK^T += Q^T dS
  }
  __syncthreads();
  float* slot = reinterpret_cast<float*>(smem) + grp * kSlot;
  if constexpr (KS == 2) {
    if (sub == 1) put_acc(da, reinterpret_cast<AccLds*>(slot), lane);
    __syncthreads();
    if (sub == 1) return;
    add_acc(da, reinterpret_cast<const AccLds*>(slot), lane);
    __builtin_amdgcn_wave_barrier();
  }
  if constexpr (WIN) {
    if (k0 < win.sinks && win.block_end(row0, 32 * KG, S) < S) {
      const int rows = (win.sinks + 31) / 32 * 32;
      float* part = win.partial + ((size_t)bh * (win.pieces + 1) + piece) * 2 * rows * D;
      store_rows_t<D>(part, k0, rows, dka, 1.0f, slot, lane);
      store_rows_t<D>(part + rows * D, k0, rows, dva, 1.0f, slot, lane);
    }
    if (piece > 0) return;
  }
  store_rows_t<D>(dk + base, k0, S, dka, 1.0f, slot, lane);
  store_rows_t<D>(dv + base, k0, S, dva, 1.0f, slot, lane);  // after the wave's dK reads
}

// One workgroup's dQ. OWN_DELTA: delta of its rows is computed here and written; otherwise read.
template <int D, bool DROP, int KS, bool OWN_DELTA, bool WIN = false, int KG = kGroups>
__device__ __forceinline__ void dq_f32_workgroup(const F32BwdArgs& a, int bh, int blk,
                                                 F32BwdShared<D, KS, KG>& sm,
                                                 const WindowArg<WIN>& win = {}) {
  // K and V tiles: planes and raw
  using Lds = BwdLds<D, KS>;
  constexpr int TR = Lds::TR, NT = 64 * KG * KS;
  char* smem = sm.tiles;
  bf16 *skp = reinterpret_cast<bf16*>(smem), *svp = skp + Lds::kPlane;
  float* raw = reinterpret_cast<float*>(svp + Lds::kPlane);
  constexpr int kSlot = Lds::slot_floats(D / 32);
  static_assert(KG * kSlot * 4 <= Lds::kBytes, "partials and staging fit");
  const float *q = a.q, *k = a.k, *v = a.v, *dout = a.dout, *lse = a.lse;
  float *dq = a.dq, *delta = a.delta;
  const int S = a.S;
  const float scale = a.scale;
  const DropParams& dr = a.dr;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform: scalar
  const int grp = wave % KG, sub = wave / KG;
  const size_t base = (size_t)bh * S * D;
  const int row0 = blk * 32 * KG;
  const int q0 = row0 + 32 * grp;
  const int qi = q0 + l32;
  const int qc = min(qi, S - 1);
  const int last = min(S, row0 + 32 * KG) - 1;
  const KeyTiles<WIN, TR> keys(row0, last, win);
  const int n_tiles = keys.count();

  X3 qb[D / 16], gb[D / 16];  // the lane's Q and dO rows (score-product B layout), split
  load_split_row<D>(qb, q + base + (size_t)qc * D, h);
  load_split_row<D>(gb, dout + base + (size_t)qc * D, h);
  const float my_lse = lse[(size_t)bh * S + qc];
  float my_delta;
  if constexpr (OWN_DELTA) {
    const float* g = dout + base + (size_t)qc * D + 8 * h;
    const float* o = a.out + base + (size_t)qc * D + 8 * h;
    float part = 0.f;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(g + 16 * ds + e);
        const f32x4 y = *reinterpret_cast<const f32x4*>(o + 16 * ds + e);
        part += x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3];
      }
    my_delta = sum_halves(part);
    if (h == 0 && qi < S && sub == 0) delta[(size_t)bh * S + qi] = my_delta;
  } else {
    my_delta = delta[(size_t)bh * S + qc];
  }
  const float my_dscale = my_delta * scale;
  f32x16 acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) acc[db] = zero16();

  const RawTile<D, TR, NT> tk{k + base, raw, S, wave, lane},
      tv{v + base, raw + TR * D, S, wave, lane};
  tk.issue(keys.row(0));
  tv.issue(keys.row(0));
  for (int t = 0; t < n_tiles; ++t) {
    wait_vm_lds<0>();  // this wave's pieces of the tile
    __syncthreads();   // every wave is done with the previous tile's planes
    store_x3<D, TR>(tk, skp);
    store_x3<D, TR>(tv, svp);
    __syncthreads();
    if (t + 1 < n_tiles) {
      tk.issue(keys.row(t + 1));
      tv.issue(keys.row(t + 1));
    }
    const int key0 = keys.row(t) + 32 * sub;
    if (key0 > q0 + 31) continue;  // wave-uniform: the whole chunk is in the future
    if constexpr (WIN)
      if (!chunk_visible(key0, q0, win)) continue;
    // lane (l32, h), register u: query qi, key key0 + reg_row(u, h)
    f32x16 s = score_tile_p<D, TR>(skp, 32 * sub, qb, lane);   // K Q^T
    f32x16 dp = score_tile_p<D, TR>(svp, 32 * sub, gb, lane);  // V dO^T
    KeepWords16 keep = {};
    if constexpr (DROP) keep = keep_words16(dr, (uint64_t)bh * S + qi, key0, h);
    // only the chunk whose first key is the wave's first query holds keys after a query (or
    // past S): waves are 32-query aligned
    const bool diag = key0 == q0;
#pragma unroll
    for (int u = 0; u < 16; ++u) s[u] = exp_acc(fmaf(s[u], scale, -my_lse));  // P
    if constexpr (WIN) {
      if (!chunk_whole(key0, q0, win)) {
        const HiddenKeys hidden(key0 + 8 * h, qi, win);
#pragma unroll
        for (int u = 0; u < 16; ++u) s[u] = hidden(reg_row(u, 0)) ? 0.f : s[u];
      }
    } else if (diag) {
#pragma unroll
      for (int u = 0; u < 16; ++u)
        if (key0 + reg_row(u, h) > qi) s[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const float p = s[u];
      float g = dp[u];
      if constexpr (DROP) g *= keep_factor(keep, u, dr);
      s[u] = p * fmaf(g, scale, -my_dscale);  // P (dP - delta) scale
    }
    accumulate_t_p<D, TR>(acc, skp, 32 * sub, s, lane);  // dQ^T += K^T dS^T
  }
  __syncthreads();
  float* slot = reinterpret_cast<float*>(smem) + grp * kSlot;
  if constexpr (KS == 2) {
    if (sub == 1) put_acc(acc, reinterpret_cast<AccLds*>(slot), lane);
    __syncthreads();
    if (sub == 1) return;
    add_acc(acc, reinterpret_cast<const AccLds*>(slot), lane);
    __builtin_amdgcn_wave_barrier();
  }
  store_rows_t<D>(dq + base, q0, S, acc, 1.0f, slot, lane);
}

// The backward is one launch: grid (BH, blocks, 2), dK/dV workgroups first (z = 0, the longer
// chains), then the dQ ones, which fill the CUs as those run out. As two launches, each
// with its own start, end and half-idle last round (B4 H12 S1024 / B1 H24 S1024 / B16 H12 S256,
// us): 158 -> 143, 140 -> 86, 68 -> 55; where the CUs are full anyway (B16 H12 S1024) 532 -> 527.
// OWN_DELTA: both kinds compute delta themselves, which saves the small grids a launch (4 x 64:
// 10.0 -> 8.3 us); past kOwnDeltaMaxS rows, where dK/dV would read O and dO once per key block
// more, a pass before does it (96 x 1024: 268 against 263.5 us).
constexpr int kOwnDeltaMaxS = 512;
template <int D, bool DROP, int KS, bool OWN_DELTA>
__global__ __launch_bounds__(64 * kGroups * KS, wgs_per_cu(KS)) void bwd_f32_kernel(
    const F32BwdArgs a) {
  __shared__ F32BwdShared<D, KS> sm;
  __shared__ float own_delta[OWN_DELTA ? kOwnDeltaMaxS : 1];
  if (blockIdx.z == 0)
    dkdv_f32_workgroup<D, DROP, KS, OWN_DELTA>(a, blockIdx.x, blockIdx.y, sm, own_delta);
  else
    dq_f32_workgroup<D, DROP, KS, OWN_DELTA>(a, blockIdx.x, gridDim.y - 1 - blockIdx.y, sm);
}

// A backward in place (dq = q or dout, or any gradient = out) runs as the delta pass, dK/dV and
// dQ, one after the other.
template <int D, bool DROP>
__global__ __launch_bounds__(64 * kGroups, wgs_per_cu(1)) void dkdv_f32_kernel(
    const F32BwdArgs a) {
  __shared__ F32BwdShared<D, 1> sm;
  dkdv_f32_workgroup<D, DROP, 1, false>(a, blockIdx.x, blockIdx.y, sm, nullptr);
}
template <int D, bool DROP>
__global__ __launch_bounds__(64 * kGroups, wgs_per_cu(1)) void dq_f32_kernel(const F32BwdArgs a) {
  __shared__ F32BwdShared<D, 1> sm;
  dq_f32_workgroup<D, DROP, 1, false>(a, blockIdx.x, gridDim.y - 1 - blockIdx.y, sm);
}

// The windowed backward: the pieces of the sink blocks' later queries first (`far` workgroups, piece
// by piece: they are short), then dK/dV (`blocks` key blocks), then dQ, with delta computed where
// it is needed (block windows up to kWindowDeltaRows rows) or by a pass before.
constexpr int kWindowDeltaRows = 1024, kPieceRows = 256;
template <int D, int KS, int KG, bool OWN_DELTA>
__global__ __launch_bounds__(64 * KG * KS, wgs_per_cu(KS, KG, D)) void window_bwd_f32_kernel(
    const F32BwdArgs a, const F32WindowBwdArg<true> win, int blocks, int sink_blocks) {
  __shared__ F32BwdShared<D, KS, KG> sm;
  __shared__ float own_delta[OWN_DELTA ? kWindowDeltaRows : 1];
  const int y = blockIdx.y, far = win.pieces * sink_blocks;
  if (y < far + blocks) {
    const int piece = y < far ? y / sink_blocks + 1 : 0;
    const int blk = y < far ? y - (piece - 1) * sink_blocks : y - far;
    dkdv_f32_workgroup<D, false, KS, OWN_DELTA, true, KG>(a, blockIdx.x, blk, sm, own_delta, win,
                                                          piece);
  } else {
    dq_f32_workgroup<D, false, KS, OWN_DELTA, true, KG>(a, blockIdx.x, y - far - blocks, sm,
                                                        {win});
  }
}

// The sink rows of dK and dV of blocks with pieces, from the partials: kJoinWays threads for four
// columns, each summing every kJoinWays-th partial, and their sums in order (BH 1, S 65536, 256
// pieces: 72 us with one thread for all of them).
constexpr int kJoinWays = 8, kJoinCols = 256 / kJoinWays;
template <int D>
__global__ __launch_bounds__(256) void window_join_f32_kernel(const F32BwdArgs a,
                                                              const F32WindowBwdArgs win) {
  __shared__ f32x4 sums[kJoinWays][kJoinCols];
  const int way = threadIdx.x / kJoinCols, at = threadIdx.x % kJoinCols;
  const int i = blockIdx.y * kJoinCols + at, col = i % (D / 4) * 4, row = i / (D / 4) % win.sinks;
  const int which = i / (D / 4) / win.sinks, bh = blockIdx.x;
  const int rows = (win.sinks + 31) / 32 * 32;
  // without pieces its workgroup has written the final row
  const int far = which > 1 ? 0 : win.far_pieces(row, a.S);
  const float* p = win.partial + ((size_t)bh * (win.pieces + 1) * 2 + which) * rows * D +
                   (size_t)row * D + col;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (far > 0)
    for (int j = way; j <= far; j += kJoinWays)
      sum += *reinterpret_cast<const f32x4*>(p + (size_t)j * 2 * rows * D);
  sums[way][at] = sum;
  __syncthreads();
  if (way != 0 || far == 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWays; ++w) sum += sums[w][at];
  *reinterpret_cast<f32x4*>((which == 0 ? a.dk : a.dv) + ((size_t)bh * a.S + row) * D + col) = sum;
}

// Waves per row group. With one, a workgroup walks its chunks four waves wide, two workgroups
// to a CU; a grid of no more workgroups than that (all of them start at once) lasts as long as
// the longest one's chain, so each group then gets a second wave and the chain is half as long.
// Past one workgroup per CU the gain shrinks with the chain's length. Forward, one -> two (us):
// 128 x 256 (256 workgroups) 21.0 -> 18.4, 48 x 1024 (384) 64.6 -> 49.6, 64 x 1024 (512) 68.8 ->
// 64.7, 96 x 512 (384) 37.8 -> 32.7; 128 x 512 (512) 38.1 -> 39.0, 128 x 300 (384) 24.8 -> 27.3,
// 40 x 2048 (640) 141 -> 147, 192 x 1024 165 -> 186; up to three chunks (S <= 96) there is too
// little to share.
int fwd_waves_per_group(int BH, int S) {
  const long long wgs = (long long)BH * ((S + kRows - 1) / kRows), cus = device_cus();
  const long long most = S >= 768 ? 4 * cus : S >= 512 ? 3 * cus : 2 * cus;  // halves of a CU
  return S > 96 && 2 * wgs <= most ? 2 : 1;
}
// The backward's grid holds two workgroups per 128 rows, so its line is at half as many rows:
// 24 x 1024 (192 of each kind) 120 -> 86, 128 x 128 22.6 -> 19.6, 48 x 1024 (384) 143 -> 150,
// 96 x 512 81 -> 94. Short sequences: 4 x 64 8.4 -> 7.2, 192 x 64 15.5 -> 20.6.
int bwd_waves_per_group(int BH, int S) {
  const long long wgs = (long long)BH * ((S + kRows - 1) / kRows), cus = device_cus();
  return wgs <= (S > 96 ? cus : cus / 4) ? 2 : 1;
}

// With a window a workgroup's chain is as long as its rows and the window together, so 64 rows by
// two waves each (KG = 2, KS = 2) have the shortest, and are taken while all such workgroups start at
// once; then 128 rows by two waves each while those do, one to a CU (at D = 64 only: at 32 a CU holds
// the other two kinds as well); then one wave each. 41 / 42 / 22 for KG and KS, us: forward 24 x 777
// x 32 with a window of 100 and 3 sinks (168 workgroups of 128 rows) 20.9 / 20.5 / 16.3, 24 x 2048 x
// 32 of 256 (384) 31.4 / 30.9 / 26.3, 56 x 1024 x 32 of 128 (448) 24.3 / 26.0 / 28.2, 12 x 1024 x 64 of
// 256 (96) 33.2 / 29.7 / 25.2, 24 x 777 x 64 of 100 27.7 / 25.6 / 34.2, 48 x 1024 x 64 of 64 29.5 /
// 40.1 / 41.8; backward 64 x 256 x 32 of 32 (256 of both kinds) 21.1 / 17.7 / 17.0, 28 x 1024 x 32 of
// 400 (448) 43.3 / 51.9 / 49.1, 8 x 1024 x 64 of 400 (128) 60.8 / 48.5 / 38.8, 16 x 1024 x 64 of 400
// (256) 61.8 / 50.1 / 65.0, 20 x 1024 x 64 of 400 (320) 67.6 / 65.6 / 81.3.
// f(KG, KS) for workgroups of `kinds` kinds for each 128 rows and `more` besides, times BH; `twos` is
// how many workgroups of KG = KS = 2 a CU holds.
template <int D, typename F>
void with_window_f32_shape(int BH, int S, int kinds, int more, int twos, F f) {
  const long long wgs = (long long)BH * (kinds * ((S + kRows - 1) / kRows) + more);
  const int cus = device_cus();
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, kGroups> all;
  if (2 * wgs <= (long long)twos * cus) return f(two, two);
  if constexpr (D == 64)
    if (S > 96 && wgs <= cus) return f(all, two);
  f(all, one);
}

// f(whether to drop, waves per row group) as compile-time constants.
template <typename F>
void with_f32_shape(int waves_per_group, bool drop, F f) {
  const bool two = waves_per_group == 2;
  auto with_drop = [&](auto d) {
    if (two)
      f(d, std::integral_constant<int, 2>{});
    else
      f(d, std::integral_constant<int, 1>{});
  };
  if (drop)
    with_drop(std::true_type{});
  else
    with_drop(std::false_type{});
}

template <int D>
hipError_t fwd_f32_t(float* out, float* lse, const float* q, const float* k, const float* v,
                     int BH, int S, float scale, hipStream_t stream, const Dropout* drop,
                     const Window* window) {
  const dim3 grid(BH, (S + kRows - 1) / kRows);
  const DropParams dr = drop_params(drop);
  if (window != nullptr) {
    with_window_f32_shape<D>(BH, S, 1, 0, D == 64 ? 1 : 3, [&](auto kg, auto ks) {
      const dim3 blocks(BH, (S + 32 * kg() - 1) / (32 * kg()));
      fwd_f32_kernel<D, false, ks(), true, true, kg()>
          <<<blocks, 64 * kg() * ks(), 0, stream>>>(out, lse, q, k, v, S, scale, dr, {*window});
    });
    return hipGetLastError();
  }
  with_f32_shape(fwd_waves_per_group(BH, S), drop != nullptr, [&](auto drop_c, auto ks) {
    auto launch = [&](auto once) {
      fwd_f32_kernel<D, drop_c(), ks(), once()>
          <<<grid, 64 * kGroups * ks(), 0, stream>>>(out, lse, q, k, v, S, scale, dr, {});
    };
    // At d_head 64 with one wave per group, up to two rounds of workgroups (two per CU), the last
    // of which run a wave per SIMD: a lone wave is faster if the conversions need not wait for
    // each other (once -> not: 192 x 400 54.7 -> 48.3 us, 256 x 384 47.1 -> 43.1, 128 x 777 90.8 ->
    // 85.8; 400 x 483 103 -> 107, 192 x 1024 158.4 -> 161.6). With dropout or at d_head 32 once is
    // faster everywhere.
    constexpr bool kEither = D == 64 && !drop_c() && ks() == 1;
    if constexpr (kEither)
      if ((long long)grid.x * grid.y <= 4LL * device_cus()) return launch(std::false_type{});
    launch(std::true_type{});
  });
  return hipGetLastError();
}

template <int D>
hipError_t bwd_f32_t(float* dq, float* dk, float* dv, float* delta, const float* dout,
                     const float* out, const float* lse, const float* q, const float* k,
                     const float* v, int BH, int S, float scale, hipStream_t stream,
                     const Dropout* drop) {
  const F32BwdArgs args{dq, dk, dv, delta, q, k, v, dout, out, lse, S, scale, drop_params(drop)};
  auto span = [&](const float* p) { return Span{p, (size_t)BH * S * D * sizeof(float)}; };
  const bool separate = in_place({span(dq), span(dk), span(dv)},
                                 {span(q), span(k), span(v), span(dout), span(out)});
  const bool own = S <= kOwnDeltaMaxS && !separate;
  hipError_t e = hipSuccess;
  if (!own) {
    const long long rows = (long long)BH * S, blocks = (rows * (D / 4) + 255) / 256;
    delta_f32_kernel<D><<<(unsigned)(blocks < 16384 ? blocks : 16384), 256, 0, stream>>>(
        delta, dout, out, rows);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  const dim3 blocks(BH, (S + kRows - 1) / kRows), grid(blocks.x, blocks.y, 2);
  with_f32_shape(bwd_waves_per_group(BH, S), drop != nullptr, [&](auto drop_c, auto ks) {
    constexpr int threads = 64 * kGroups * ks();
    if (separate) {
      dkdv_f32_kernel<D, drop_c()><<<blocks, 64 * kGroups, 0, stream>>>(args);
      if ((e = hipGetLastError()) != hipSuccess) return;
      dq_f32_kernel<D, drop_c()><<<blocks, 64 * kGroups, 0, stream>>>(args);
    } else if (own) {
      bwd_f32_kernel<D, drop_c(), ks(), true><<<grid, threads, 0, stream>>>(args);
    } else {
      bwd_f32_kernel<D, drop_c(), ks(), false><<<grid, threads, 0, stream>>>(args);
    }
    e = hipGetLastError();
  });
  return e;
}

// How a windowed backward is launched: the pieces of its sink keys' later queries, and the bytes
// of their partials. Small grids last as long as a sink block's chain, and pieces shorten it (24 x
// 512 x 64 with a window of 100 46 -> 32 us, 24 x 777 x 32 of 400 57 -> 46, 12 x 300 x 32 of 64 17 ->
// 15); in larger ones pieces and their join cost more than the chain where the later queries are
// few next to the window or in all (192 x 500 x 64 of 64 113 -> 118, 192 x 1024 x 64 of 400 433 ->
// 443).
struct F32WindowPlan {
  int pieces;
  size_t workspace;
};
F32WindowPlan window_f32_plan(int BH, int S, int D, const Window& w) {
  const long long end = ((long long)kRows + w.window - 2) / 64 * 64 + 64;  // of block 0
  const long long far = S - end;
  F32WindowPlan p{0, 0};
  const bool small = (long long)BH * S <= 1 << 16 && far > 64;
  if (w.sinks > 0 && (small || (far > 384 && (far > end || S > kWindowDeltaRows))))
    p.pieces = (int)((far + kPieceRows - 1) / kPieceRows);
  const size_t rows = (size_t)(w.sinks + 31) / 32 * 32;
  if (p.pieces > 0) p.workspace = sizeof(float) * BH * (size_t)(p.pieces + 1) * 2 * rows * D;
  return p;
}

template <int D>
hipError_t window_bwd_f32_t(const F32BwdArgs& args, int BH, const Window& w, float* partial,
                            size_t workspace_bytes, hipStream_t stream) {
  const int S = args.S;
  const F32WindowPlan plan = window_f32_plan(BH, S, D, w);
  if (plan.workspace > workspace_bytes) return hipErrorInvalidValue;
  F32WindowBwdArg<true> win;
  static_cast<Window&>(win) = w;
  win.piece_rows = kPieceRows;
  win.pieces = plan.pieces;
  win.partial = partial;
  // rows that a dK/dV workgroup may walk: all, or a block's window in whole 64s
  const bool own =
      S <= kWindowDeltaRows ||
      (kRows + w.window + 64 <= kWindowDeltaRows && (w.sinks == 0 || plan.pieces > 0));
  hipError_t e = hipSuccess;
  if (!own) {
    const long long rows = (long long)BH * S, n = (rows * (D / 4) + 255) / 256;
    delta_f32_kernel<D><<<(unsigned)(n < 16384 ? n : 16384), 256, 0, stream>>>(
        args.delta, args.dout, args.out, rows);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  with_window_f32_shape<D>(BH, S, 2, plan.pieces, D == 64 ? 1 : 2, [&](auto kg, auto ks) {
    constexpr int rows = 32 * kg(), threads = 64 * kg() * ks();
    const int blocks = (S + rows - 1) / rows, sink_blocks = (w.sinks + rows - 1) / rows;
    const dim3 grid(BH, plan.pieces * sink_blocks + 2 * blocks);
    if (own)
      window_bwd_f32_kernel<D, ks(), kg(), true>
          <<<grid, threads, 0, stream>>>(args, win, blocks, sink_blocks);
    else
      window_bwd_f32_kernel<D, ks(), kg(), false>
          <<<grid, threads, 0, stream>>>(args, win, blocks, sink_blocks);
    e = hipGetLastError();
  });
  if (e != hipSuccess || plan.pieces == 0) return e;
  window_join_f32_kernel<D>
      <<<dim3(BH, (w.sinks * (D / 4) * 2 + kJoinCols - 1) / kJoinCols), 256, 0, stream>>>(args, win);
  return hipGetLastError();
}

}  // namespace

size_t window_f32_workspace_bytes(int BH, int S, int D, const Window& w) {
  return w.window >= S ? 0 : window_f32_plan(BH, S, D, {w.window, w.sinks < S ? w.sinks : S}).workspace;
}

hipError_t launch_window_bwd_f32(float* dq, float* dk, float* dv, float* delta,
                                 const float* dout, const float* out, const float* lse,
                                 const float* q, const float* k, const float* v, int BH, int S,
                                 int D, float scale, const Window& window, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  if (window.window >= S)
    return launch_bwd_f32(dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, D, scale, stream);
  const F32BwdArgs args{dq, dk, dv, delta, q, k, v, dout, out, lse, S, scale, drop_params(nullptr)};
  const Window w{window.window, window.sinks < S ? window.sinks : S};
  float* partial = static_cast<float*>(workspace);
  if (D == 64) return window_bwd_f32_t<64>(args, BH, w, partial, workspace_bytes, stream);
  if (D == 32) return window_bwd_f32_t<32>(args, BH, w, partial, workspace_bytes, stream);
  return hipErrorInvalidValue;
}

hipError_t launch_fwd_f32(float* out, float* lse, const float* q, const float* k,
                          const float* v, int BH, int S, int D, float scale,
                          hipStream_t stream, const Dropout* drop, const Window* window) {
  if (window != nullptr && window->window >= S) window = nullptr;  // every earlier key is seen
  if (D == 64) return fwd_f32_t<64>(out, lse, q, k, v, BH, S, scale, stream, drop, window);
  if (D == 32) return fwd_f32_t<32>(out, lse, q, k, v, BH, S, scale, stream, drop, window);
  return hipErrorInvalidValue;
}

hipError_t launch_bwd_f32(float* dq, float* dk, float* dv, float* delta, const float* dout,
                          const float* out, const float* lse, const float* q, const float* k,
                          const float* v, int BH, int S, int D, float scale,
                          hipStream_t stream, const Dropout* drop) {
  if (D == 64)
    return bwd_f32_t<64>(dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, scale, stream,
                         drop);
  if (D == 32)
    return bwd_f32_t<32>(dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, scale, stream,
                         drop);
  return hipErrorInvalidValue;
}

}  // namespace dadgpt
