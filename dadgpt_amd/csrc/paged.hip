// Appending to paged caches for gfx950: the new rows of ragged sequences out of a fused projection's
// output into the pages that the block table names, q and k rotated on the way (one launch for what
// would be three: rotation, and a scatter each of k and v), one chunk of one head a thread (as
// rope.hip). Bound by HBM, and for a token a sequence by the launch and the chain row_start, lens -> page
// -> store: 8192 tokens of 16 prompts, 12 heads of 64 in bf16, 15.7 us (4.8 TB/s; a copy 14.6 us); one
// token of 32 sequences 3.4 us of 13, the rest is the call's.
#include "common.hpp"
#include "paged.hpp"
#include "rope.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct AppendArgs {
  T *k_pages, *v_pages, *q_out;
  const T *q, *k, *v;
  long long ld_out, ld_q, ld_kv;
  PagedStep p;
  Rope r;
  int heads_q;  // query heads to move (0 without q)
};

// Grid (rows of a sequence, sequences). Consecutive threads run along a head's chunks, then the heads
// of a row, which lie side by side in the projection's output.
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(const AppendArgs<T> a) {
  const auto seq = paged::NewRows::of<true>(a.p, blockIdx.y);
  const int D = a.p.D, chunks = D / (2 * VEC), heads = a.heads_q + 2 * a.p.Hkv;
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t c = id % chunks, j = id / chunks;
  const int t = j / heads, head = j % heads;
  const int token = seq.token + t;
  if (t >= seq.count || token < 0) return;
  const int kh = head - a.heads_q, vh = kh - a.p.Hkv;
  const long long row = seq.first + t;
  const T* src;
  T* dst;
  if (kh < 0) {
    src = a.q + row * a.ld_q + head * D;
    dst = a.q_out + row * a.ld_out + head * D;
  } else {
    const int page = a.p.table[(size_t)blockIdx.y * a.p.max_pages + token / a.p.page];
    if (!paged::is_page(a.p, page)) return;
    const int h = vh >= 0 ? vh : kh;
    src = (vh >= 0 ? a.v : a.k) + row * a.ld_kv + h * D;
    dst = (vh >= 0 ? a.v_pages : a.k_pages) + paged::page_row(a.p, page, h, token % a.p.page);
  }
  const rotary::Chunk ch =
      vh >= 0 ? rotary::Chunk{{2 * (int)c * VEC, 2 * (int)c * VEC + VEC}, false}
              : rotary::chunk_of<VEC, INTER>(c, a.r.rot_dim);
  rotary::Piece<T, VEC> x, y;
  x.load(src + ch.at[0]);
  y.load(src + ch.at[1]);
  if (ch.rotated)
    rotary::turn_pieces<T, VEC, INTER>(
        x, y, rotary::turn_of<VEC, sizeof(T) == 2>(a.r.freqs + c * VEC, token, a.r.magnitude, false));
  x.store(dst + ch.at[0]);
  y.store(dst + ch.at[1]);
}

template <typename T>
hipError_t launch_append_t(T* k_pages, T* v_pages, T* q_out, long long ld_out, const T* q,
                           long long ld_q, const T* k, const T* v, long long ld_kv,
                           const PagedStep& p, const Rope& r, hipStream_t stream) {
  AppendArgs<T> a{k_pages, v_pages, q_out, q, k, v, ld_out, ld_q, ld_kv, p, r, q ? p.H : 0};
  const int heads = a.heads_q + 2 * p.Hkv;
  auto run = [&](auto vec, auto inter) {
    const long long chunks = p.D / (2 * vec());
    const dim3 grid((unsigned)((p.max_rows * chunks * heads + kThreads - 1) / kThreads), p.n_seq);
    paged_append_kernel<T, vec(), inter()><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  };
  auto with = [&](auto vec) {
    return r.interleaved ? run(vec, std::true_type{}) : run(vec, std::false_type{});
  };
  if constexpr (sizeof(T) == 2)
    if (rotary::wide<T>(r.rot_dim, p.D)) return with(std::integral_constant<int, 8>{});
  return with(std::integral_constant<int, 4>{});
}

}  // namespace

hipError_t launch_paged_append_bf16(bf16* k_pages, bf16* v_pages, bf16* q_out, long long ld_out,
                                    const bf16* q, long long ld_q, const bf16* k, const bf16* v,
                                    long long ld_kv, const PagedStep& step, const Rope& rope,
                                    hipStream_t stream) {
  return launch_append_t<bf16>(k_pages, v_pages, q_out, ld_out, q, ld_q, k, v, ld_kv, step, rope, stream);
}
hipError_t launch_paged_append_f32(float* k_pages, float* v_pages, float* q_out, long long ld_out,
                                   const float* q, long long ld_q, const float* k, const float* v,
                                   long long ld_kv, const PagedStep& step, const Rope& rope,
                                    hipStream_t stream) {
  return launch_append_t<float>(k_pages, v_pages, q_out, ld_out, q, ld_q, k, v, ld_kv, step, rope, stream);
}

}  // namespace dadgpt
