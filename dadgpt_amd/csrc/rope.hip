// Rotary positions of a training step for gfx950: q and k rotated by their positions, and their
// gradients back. y = magnitude R(position * f) x pair by pair, so the transposed map, the backward, is
// the rotation by the negative angle with the same magnitude, and one kernel does both.
//
// Bound by HBM: every element is read and written once (4 operations an element). The angles cost
// more than the rotation (a double product and a sincospi for each pair of a token), so a thread
// computes those of its pairs once and takes up to eight heads of the token.
#include "common.hpp"
#include "rope.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct RopeArgs {
  T *q_out, *k_out;
  const T *q, *k;
  const int* positions;
  RopeShape s;
  Rope r;
  int groups;          // of heads: a thread takes heads g, g + groups, ..
  bool tokens_first;   // consecutive threads along the tokens of a head, not along the heads
  uint32_t n;
};

// Consecutive threads run along a head's chunks and then along what lies next in memory: the heads of a
// token, or the tokens of a head.
template <typename T, int VEC, bool INTER, int HPT>
__global__ __launch_bounds__(kThreads) void rope_kernel(const RopeArgs<T> a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= a.n) return;
  const int D = a.s.D, S = a.s.S, chunks = D / (2 * VEC);
  const uint32_t c = id % chunks, j = id / chunks, tokens = (uint32_t)a.s.B * S;
  const uint32_t token = a.tokens_first ? j % tokens : j / a.groups;
  const uint32_t g = a.tokens_first ? j / tokens : j % a.groups;
  const uint32_t b = token / S, row = token - b * S;
  const rotary::Chunk ch = rotary::chunk_of<VEC, INTER>(c, a.r.rot_dim);

  const T* src[HPT];
  T* dst[HPT];
  rotary::Piece<T, VEC> x[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int head = i * a.groups + g;
    const bool is_k = head >= a.s.H;
    const int h = is_k ? head - a.s.H : head;
    const Strides64 from = a.s.t[is_k ? 1 : 0], to = a.s.t[is_k ? 3 : 2];
    src[i] = (is_k ? a.k : a.q) + (b * from.batch + h * from.head + row * from.row);
    dst[i] = (is_k ? a.k_out : a.q_out) + (b * to.batch + h * to.head + row * to.row);
    if (head >= a.s.H + a.s.Hkv) dst[i] = nullptr;
    if (dst[i] == nullptr) continue;
    x[i][0].load(src[i] + ch.at[0]);
    x[i][1].load(src[i] + ch.at[1]);
  }
  if (ch.rotated) {
    const int pos = a.positions == nullptr ? (int)row : a.positions[token];
    const auto turn = rotary::turn_of<VEC>(a.r.freqs + c * VEC, pos, a.r.magnitude, a.r.inverse);
#pragma unroll
    for (int i = 0; i < HPT; ++i) rotary::turn_pieces<T, VEC, INTER>(x[i][0], x[i][1], turn);
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    if (dst[i] == nullptr) continue;
    x[i][0].store(dst[i] + ch.at[0]);
    x[i][1].store(dst[i] + ch.at[1]);
  }
}

template <typename T>
hipError_t launch_rope_t(T* q_out, T* k_out, const T* q, const T* k, const RopeShape& s,
                         const Rope& r, const int* positions, hipStream_t stream) {
  RopeArgs<T> a{q_out, k_out, q, k, positions, s, r, 0, false, 0};
  const int heads = s.H + s.Hkv;
  const Strides64& t = s.H > 0 ? s.t[0] : s.t[1];
  a.tokens_first = t.row < t.head;
  auto run = [&](auto vec, auto inter) {
    const long long per_head = (long long)s.B * s.S * (s.D / (2 * vec()));
    const int hpt = rotary::heads_per_thread(per_head, heads);
    a.groups = (heads + hpt - 1) / hpt;
    a.n = (uint32_t)(per_head * a.groups);
    const unsigned grid = (a.n + kThreads - 1) / kThreads;
    switch (hpt) {
      case 1: rope_kernel<T, vec(), inter(), 1><<<grid, kThreads, 0, stream>>>(a); break;
      case 2: rope_kernel<T, vec(), inter(), 2><<<grid, kThreads, 0, stream>>>(a); break;
      case 4: rope_kernel<T, vec(), inter(), 4><<<grid, kThreads, 0, stream>>>(a); break;
      default: rope_kernel<T, vec(), inter(), 8><<<grid, kThreads, 0, stream>>>(a); break;
    }
    return hipGetLastError();
  };
  auto with = [&](auto vec) {
    return r.interleaved ? run(vec, std::true_type{}) : run(vec, std::false_type{});
  };
  if constexpr (sizeof(T) == 2)
    if (rotary::wide<T>(r.rot_dim, s.D)) return with(std::integral_constant<int, 8>{});
  return with(std::integral_constant<int, 4>{});
}

}  // namespace

long long rope_threads(const RopeShape& s) {
  return (long long)s.B * s.S * (s.D / 8) * (s.H + s.Hkv);
}

hipError_t launch_rope_bf16(bf16* q_out, bf16* k_out, const bf16* q, const bf16* k,
                            const RopeShape& shape, const Rope& rope, const int* positions,
                            hipStream_t stream) {
  return launch_rope_t<bf16>(q_out, k_out, q, k, shape, rope, positions, stream);
}
hipError_t launch_rope_f32(float* q_out, float* k_out, const float* q, const float* k,
                           const RopeShape& shape, const Rope& rope, const int* positions,
                           hipStream_t stream) {
  return launch_rope_t<float>(q_out, k_out, q, k, shape, rope, positions, stream);
}

}  // namespace dadgpt
