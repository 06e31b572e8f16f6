// Rotary positions of a training step for gfx950: q and k rotated by their positions, and their
// gradients back. y = magnitude R(position * f) x pair by pair, so the transposed map, the backward, is
// the rotation by the negative angle with the same magnitude, and one kernel does both.
//
// Bound by HBM: every element is read and written once (4 operations an element). A thread turns one
// chunk of one head, so that the waves are many and short and loads, angles and stores of different ones
// overlap: B16 T1024, q and k of 12 heads of 64 in bf16, one way, takes 24 us (4.2 TB/s; a copy 19.5 us),
// B1 T32768, 10 heads of 64 in fp32, 34 us (5.0 TB/s). (Several heads a thread share its angles, but
// with 2, 4 and 8 of them these took 25, 27 and 27 us, and 36, 40 and 45.)
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
  bool tokens_first;   // consecutive threads along the tokens of a head, not along the heads
  uint32_t n;
};

// Consecutive threads run along a head's chunks and then along what lies next in memory: the heads of a
// token, or the tokens of a head.
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(const RopeArgs<T> a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= a.n) return;
  const uint32_t chunks = a.s.D / (2 * VEC), heads = a.s.H + a.s.Hkv, tokens = (uint32_t)a.s.B * a.s.S;
  const uint32_t c = id % chunks, j = id / chunks;
  const uint32_t token = a.tokens_first ? j % tokens : j / heads;
  const uint32_t head = a.tokens_first ? j / tokens : j % heads;
  const uint32_t b = token / a.s.S, row = token - b * a.s.S;
  const rotary::Chunk ch = rotary::chunk_of<VEC, INTER>(c, a.r.rot_dim);

  const bool is_k = head >= (uint32_t)a.s.H;
  const uint32_t h = is_k ? head - a.s.H : head;
  const Strides64 from = a.s.t[is_k ? 1 : 0], to = a.s.t[is_k ? 3 : 2];
  const T* src = (is_k ? a.k : a.q) + (b * from.batch + h * from.head + row * from.row);
  T* dst = (is_k ? a.k_out : a.q_out) + (b * to.batch + h * to.head + row * to.row);
  rotary::Piece<T, VEC> x, y;
  x.load(src + ch.at[0]);
  y.load(src + ch.at[1]);
  if (ch.rotated) {
    const int pos = a.positions == nullptr ? (int)row : a.positions[token];
    rotary::turn_pieces<T, VEC, INTER>(
        x, y, rotary::turn_of<VEC, sizeof(T) == 2>(a.r.freqs + c * VEC, pos, a.r.magnitude, a.r.inverse));
  }
  x.store(dst + ch.at[0]);
  y.store(dst + ch.at[1]);
}

template <typename T>
hipError_t launch_rope_t(T* q_out, T* k_out, const T* q, const T* k, const RopeShape& s,
                         const Rope& r, const int* positions, hipStream_t stream) {
  RopeArgs<T> a{q_out, k_out, q, k, positions, s, r, false, 0};
  const int heads = s.H + s.Hkv;
  const Strides64& t = s.t[0];
  a.tokens_first = t.row < t.head;
  auto run = [&](auto vec, auto inter) {
    a.n = (uint32_t)((long long)s.B * s.S * heads * (s.D / (2 * vec())));
    rope_kernel<T, vec(), inter()><<<(a.n + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
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
