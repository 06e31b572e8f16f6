// extern "C" entry points of the bounded KV caches (declared in include/dadgpt/kv_cache.h), with the
// checks and errors of capi.cpp.
#include <hip/hip_runtime.h>

#include <cmath>

#include "capi_util.hpp"
#include "dadgpt/kv_cache.h"
#include "kernels.hpp"

namespace {

using namespace dadgpt::capi;
using dadgpt::bf16;
using dadgpt::Span;

const bf16* B(const uint16_t* p) { return reinterpret_cast<const bf16*>(p); }
bf16* B(uint16_t* p) { return reinterpret_cast<bf16*>(p); }

// fp32 and int32 side arrays (scales, weights, lengths, indices): non-null and 4-byte aligned.
struct Named {
  const void* p;
  const char* name;
};
int check_words(const char* fn, std::initializer_list<Named> arrays) {
  for (const Named& a : arrays) {
    if (a.p == nullptr) return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s is null", fn, a.name);
    if (reinterpret_cast<uintptr_t>(a.p) % 4 != 0)
      return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s is not 4-byte aligned", fn, a.name);
  }
  return DADGPT_OK;
}

int check_block(const char* fn, int block) {
  if (block != 16 && block != 32 && block != 64 && block != 128)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: block=%d must be 16, 32, 64 or 128", fn, block);
  return DADGPT_OK;
}

// Outputs against each other and against inputs; `inputs` may hold spans that one output replaces
// on purpose (the caller leaves those out).
struct NamedSpan {
  Span span;
  const char* name;
};
int check_apart(const char* fn, std::initializer_list<NamedSpan> outputs,
                std::initializer_list<NamedSpan> inputs) {
  for (const NamedSpan* a = outputs.begin(); a != outputs.end(); ++a) {
    for (const NamedSpan* b = a + 1; b != outputs.end(); ++b)
      if (dadgpt::overlap(a->span, b->span))
        return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s overlaps %s", fn, a->name, b->name);
    for (const NamedSpan& b : inputs)
      if (b.span.p != nullptr && dadgpt::overlap(a->span, b.span))
        return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s overlaps %s", fn, a->name, b.name);
  }
  return DADGPT_OK;
}

int check_new_rows(const char* fn, const char* name, const dadgpt_head_strides* st,
                   dadgpt::HeadStrides64* to) {
  if (st == nullptr)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: strides of %s are null", fn, name);
  constexpr int64_t kMost = int64_t(1) << 40;
  if (st->batch < 0 || st->head < 0 || st->row < 0 || st->batch % 8 || st->head % 8 ||
      st->row % 8 || st->batch > kMost || st->head > kMost || st->row > kMost)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: strides of %s {batch %lld, head %lld, row %lld}: each must be a non-negative "
                "multiple of 8, at most 2^40",
                fn, name, (long long)st->batch, (long long)st->head, (long long)st->row);
  *to = dadgpt::HeadStrides64{st->batch, st->head, st->row};
  return DADGPT_OK;
}

template <typename T, typename F>
int append(const char* fn, uint8_t* k8, uint8_t* v8, float* k_scale, float* v_scale, const T* k,
           const T* v, const dadgpt_head_strides* k_strides, const dadgpt_head_strides* v_strides,
           const int32_t* lens, const int32_t* counts, int n_seq, int H, int rows, int max_len,
           int d_head, int block, F launch) {
  if (int st = check_decode_shape(fn, n_seq, H, max_len, d_head, 1.0f, {k8, v8, k, v})) return st;
  if (int st = check_words(fn, {{k_scale, "k_scale"}, {v_scale, "v_scale"}, {lens, "lens"}}))
    return st;
  if (counts != nullptr)
    if (int st = check_words(fn, {{counts, "counts"}})) return st;
  if (int st = check_block(fn, block)) return st;
  dadgpt::HeadStrides64 ks, vs;
  if (int st = check_new_rows(fn, "k", k_strides, &ks)) return st;
  if (int st = check_new_rows(fn, "v", v_strides, &vs)) return st;
  if (rows < 1)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: rows=%d must be positive", fn, rows);
  // grid (heads, touched blocks, sequences)
  if (n_seq > 65535 || dadgpt::kv8_touched_blocks(rows, block) > 65535)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: n_seq=%d x n_heads=%d x rows=%d exceeds the launch limits", fn, n_seq, H,
                rows);
  const size_t caches = (size_t)n_seq * H;
  const size_t codes = caches * max_len * d_head;
  const size_t scales = caches * ((max_len + block - 1) / block) * sizeof(float);
  const NamedSpan K{{k8, codes}, "k_cache"}, V{{v8, codes}, "v_cache"};
  const NamedSpan KS{{k_scale, scales}, "k_scale"}, VS{{v_scale, scales}, "v_scale"};
  auto extent = [&](const dadgpt::HeadStrides64& t) {
    return sizeof(T) * ((size_t)(n_seq - 1) * t.batch + (size_t)(H - 1) * t.head +
                        (size_t)(rows - 1) * t.row + d_head);
  };
  if (int st = check_apart(fn, {K, V, KS, VS},
                           {{{k, extent(ks)}, "k"},
                            {{v, extent(vs)}, "v"},
                            {{lens, 4 * (size_t)n_seq}, "lens"},
                            {{counts, 4 * (size_t)n_seq}, "counts"}}))
    return st;
  return from_hip(launch(ks, vs), fn);
}

// The workspace, and that what the call uses of it (`used` bytes) lies apart from its other buffers.
int check_workspace(const char* fn, const void* ws, size_t ws_bytes, size_t need, size_t used,
                    std::initializer_list<NamedSpan> others) {
  if (need == 0) return DADGPT_OK;
  if (ws == nullptr || ws_bytes < need)
    return fail(DADGPT_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", fn,
                ws == nullptr ? 0 : ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: workspace is not 16-byte aligned", fn);
  return check_apart(fn, {{{ws, used}, "the workspace"}}, others);
}

// An output row replaces the query that only its own workgroups have read, or lies apart from it.
NamedSpan query(const void* q, const void* out, size_t bytes) {
  return {{q == out ? nullptr : q, bytes}, "q"};
}

// Shared checks of the 8-bit decode (`elem_bytes` of q and out); window 0: none.
int check_kv8_decode(const char* fn, const void* out, const void* q, const uint8_t* k8,
                     const uint8_t* v8, const float* k_scale, const float* v_scale,
                     const int32_t* lens, int n_seq, int H, int max_len, int d_head, int block,
                     int elem_bytes, float scale, int window, int sinks, const void* ws,
                     size_t ws_bytes) {
  if (int st = check_decode_shape(fn, n_seq, H, max_len, d_head, scale, {out, q, k8, v8}))
    return st;
  if (int st = check_words(fn, {{k_scale, "k_scale"}, {v_scale, "v_scale"}, {lens, "lens"}}))
    return st;
  if (int st = check_block(fn, block)) return st;
  int most = max_len;
  if (window == 0) {
    if (sinks != 0)
      return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: sinks=%d without a window", fn, sinks);
  } else {
    if (int st = check_window(fn, 0, window, sinks)) return st;
    most = dadgpt::visible_keys(max_len, {window, sinks});
  }
  const size_t caches = (size_t)n_seq * H, row = caches * d_head * elem_bytes;
  const size_t codes = caches * max_len * d_head;
  const size_t scales = caches * ((max_len + block - 1) / block) * sizeof(float);
  const NamedSpan O{{out, row}, "out"}, K{{k8, codes}, "k_cache"}, V{{v8, codes}, "v_cache"};
  const NamedSpan KS{{k_scale, scales}, "k_scale"}, VS{{v_scale, scales}, "v_scale"};
  const NamedSpan len{{lens, 4 * (size_t)n_seq}, "lens"};
  if (int st = check_apart(fn, {O}, {query(q, out, row), K, V, KS, VS, len})) return st;
  // (counters at its start, partials against its end)
  return check_workspace(fn, ws, ws_bytes,
                         dadgpt::kv8_decode_workspace_bytes(n_seq, H, most, d_head), ws_bytes,
                         {O, {{q, row}, "q"}, K, V, KS, VS, len});
}

int check_weights_decode(const char* fn, const void* out, const float* wout, const void* q,
                         const void* kc, const void* vc, const float* weights,
                         const int32_t* lens, int n_seq, int H, int max_len, int d_head,
                         int elem_bytes, float scale, const void* ws, size_t ws_bytes) {
  if (int st = check_decode_shape(fn, n_seq, H, max_len, d_head, scale, {out, q, kc, vc}))
    return st;
  if (int st = check_words(
          fn, {{wout, "weights_out"}, {weights, "weights"}, {lens, "lens"}}))
    return st;
  const size_t caches = (size_t)n_seq * H, row = caches * d_head * elem_bytes;
  const size_t w = sizeof(float) * caches * max_len, cache = row * max_len;
  const NamedSpan O{{out, row}, "out"}, W{{wout, w}, "weights_out"};
  const NamedSpan K{{kc, cache}, "k_cache"}, V{{vc, cache}, "v_cache"};
  const NamedSpan win{{wout == weights ? nullptr : weights, w}, "weights"};
  const NamedSpan len{{lens, 4 * (size_t)n_seq}, "lens"};
  if (int st = check_apart(fn, {O}, {W, query(q, out, row), K, V, {{weights, w}, "weights"}, len}))
    return st;
  if (int st = check_apart(fn, {W}, {{{q, row}, "q"}, K, V, win, len})) return st;
  const size_t need = dadgpt::weights_decode_workspace_bytes(n_seq, H, max_len, d_head);
  return check_workspace(fn, ws, ws_bytes, need, need, {O, W, {{q, row}, "q"}, K, V, win, len});
}

int evict(const char* fn, void* k_out, void* v_out, float* wout, int32_t* kept,
          int32_t* lens_out, const void* k, const void* v, const float* weights,
          const int32_t* lens, int n_seq, int H, int max_len, int max_out, int d_head,
          int elem_bytes, int budget, int sinks, int recent, void* stream) {
  if (int st = check_decode_shape(fn, n_seq, H, max_len, d_head, 1.0f, {k_out, v_out, k, v}))
    return st;
  if (int st = check_words(fn, {{wout, "weights_out"}, {kept, "kept"}, {lens_out, "lens_out"},
                                {weights, "weights"}, {lens, "lens"}}))
    return st;
  if (budget < 1 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: budget=%d must be positive and hold sinks=%d and recent=%d", fn, budget, sinks,
                recent);
  // 1024 lanes a (sequence, head) in place, counted in 32 bits; grid.y of the gather: 64 rows a
  // workgroup at least
  if ((long long)n_seq * H >= (1LL << 22))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: n_seq=%d x n_heads=%d exceeds the launch limits",
                fn, n_seq, H);
  const int most = budget < max_len ? budget : max_len;
  if (max_out < most || max_out > 65535L * 256 || most > 65535L * 64 || budget > 65535L * 256)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: max_out=%d cannot hold budget=%d of max_len=%d rows, or one exceeds the launch "
                "limits",
                fn, max_out, budget, max_len);
  const bool in_place = k_out == k || v_out == v;
  if (in_place && (k_out != k || v_out != v || max_out != max_len))
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: in place, k_out = k, v_out = v and max_out=%d = max_len=%d together", fn,
                max_out, max_len);
  if (wout == weights && max_out != max_len)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: weights_out = weights needs max_out = max_len",
                fn);
  const size_t caches = (size_t)n_seq * H, row = (size_t)d_head * elem_bytes;
  const size_t in = caches * max_len, out = caches * max_out;
  auto input = [](const void* p, size_t n, const char* name, bool replaced) {
    return NamedSpan{{replaced ? nullptr : p, n}, name};
  };
  if (int st = check_apart(
          fn,
          {{{k_out, out * row}, "k_out"},
           {{v_out, out * row}, "v_out"},
           {{wout, out * 4}, "weights_out"},
           {{kept, caches * budget * 4}, "kept"},
           {{lens_out, 4 * (size_t)n_seq}, "lens_out"}},
          {input(k, in * row, "k", in_place), input(v, in * row, "v", in_place),
           input(weights, in * 4, "weights", wout == weights),
           input(lens, 4 * (size_t)n_seq, "lens", lens_out == lens)}))
    return st;
  // an input left out above must still be apart from the other outputs: it is its replacement's
  // own extent, which they are apart from
  return from_hip(dadgpt::launch_kv_evict(k_out, v_out, wout, kept, lens_out, k, v, weights, lens,
                                          n_seq, H, max_len, max_out, (int)row, budget, sinks,
                                          recent, as_stream(stream)),
                  fn);
}

}  // namespace

extern "C" {

int dadgpt_kv8_blocks(int max_len, int block) {
  if (max_len < 1 || (block != 16 && block != 32 && block != 64 && block != 128)) return 0;
  return (int)(((long long)max_len + block - 1) / block);
}

int dadgpt_kv8_append_bf16(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale,
                           const uint16_t* k, const uint16_t* v,
                           const dadgpt_head_strides* k_strides,
                           const dadgpt_head_strides* v_strides, const int32_t* lens,
                           const int32_t* counts, int n_seq, int n_heads, int rows, int max_len,
                           int d_head, int block, void* stream) {
  return append("dadgpt_kv8_append_bf16", k_cache, v_cache, k_scale, v_scale, k, v, k_strides,
                v_strides, lens, counts, n_seq, n_heads, rows, max_len, d_head, block,
                [&](const dadgpt::HeadStrides64& ks, const dadgpt::HeadStrides64& vs) {
                  return dadgpt::launch_kv8_append_bf16(k_cache, v_cache, k_scale, v_scale, B(k),
                                                        B(v), ks, vs, lens, counts, n_seq, n_heads,
                                                        rows, max_len, d_head, block,
                                                        as_stream(stream));
                });
}

int dadgpt_kv8_append_f32(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale,
                          const float* k, const float* v, const dadgpt_head_strides* k_strides,
                          const dadgpt_head_strides* v_strides, const int32_t* lens,
                          const int32_t* counts, int n_seq, int n_heads, int rows, int max_len,
                          int d_head, int block, void* stream) {
  return append("dadgpt_kv8_append_f32", k_cache, v_cache, k_scale, v_scale, k, v, k_strides,
                v_strides, lens, counts, n_seq, n_heads, rows, max_len, d_head, block,
                [&](const dadgpt::HeadStrides64& ks, const dadgpt::HeadStrides64& vs) {
                  return dadgpt::launch_kv8_append_f32(k_cache, v_cache, k_scale, v_scale, k, v,
                                                       ks, vs, lens, counts, n_seq, n_heads, rows,
                                                       max_len, d_head, block, as_stream(stream));
                });
}

size_t dadgpt_decode_kv8_workspace_bytes(int n_seq, int n_heads, int max_len, int d_head) {
  if (n_seq < 1 || n_heads < 1 || max_len < 1 || !supported(d_head)) return 0;
  return dadgpt::kv8_decode_workspace_bytes(n_seq, n_heads, max_len, d_head);
}

int dadgpt_decode_attention_kv8_bf16(uint16_t* out, const uint16_t* q, const uint8_t* k_cache,
                                     const uint8_t* v_cache, const float* k_scale,
                                     const float* v_scale, const int32_t* lens, int n_seq,
                                     int n_heads, int max_len, int d_head, int block, float scale,
                                     int window, int sinks, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* fn = "dadgpt_decode_attention_kv8_bf16";
  if (int st = check_kv8_decode(fn, out, q, k_cache, v_cache, k_scale, v_scale, lens, n_seq,
                                n_heads, max_len, d_head, block, sizeof(*out), scale, window, sinks,
                                workspace, workspace_bytes))
    return st;
  const dadgpt::Window w{window, sinks};
  return from_hip(dadgpt::launch_kv8_decode_bf16(
                      B(out), B(q), k_cache, v_cache, k_scale, v_scale, lens, n_seq, n_heads,
                      max_len, d_head, block, scale, window ? &w : nullptr, workspace,
                      workspace_bytes, as_stream(stream)),
                  fn);
}

int dadgpt_decode_attention_kv8_f32(float* out, const float* q, const uint8_t* k_cache,
                                    const uint8_t* v_cache, const float* k_scale,
                                    const float* v_scale, const int32_t* lens, int n_seq,
                                    int n_heads, int max_len, int d_head, int block, float scale,
                                    int window, int sinks, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* fn = "dadgpt_decode_attention_kv8_f32";
  if (int st = check_kv8_decode(fn, out, q, k_cache, v_cache, k_scale, v_scale, lens, n_seq,
                                n_heads, max_len, d_head, block, sizeof(*out), scale, window, sinks,
                                workspace, workspace_bytes))
    return st;
  const dadgpt::Window w{window, sinks};
  return from_hip(dadgpt::launch_kv8_decode_f32(out, q, k_cache, v_cache, k_scale, v_scale, lens,
                                                n_seq, n_heads, max_len, d_head, block, scale,
                                                window ? &w : nullptr, workspace, workspace_bytes,
                                                as_stream(stream)),
                  fn);
}

size_t dadgpt_decode_weights_workspace_bytes(int n_seq, int n_heads, int max_len, int d_head) {
  if (n_seq < 1 || n_heads < 1 || max_len < 1 || !supported(d_head)) return 0;
  return dadgpt::weights_decode_workspace_bytes(n_seq, n_heads, max_len, d_head);
}

int dadgpt_decode_attention_weights_bf16(uint16_t* out, float* weights_out, const uint16_t* q,
                                         const uint16_t* k_cache, const uint16_t* v_cache,
                                         const float* weights, const int32_t* lens, int n_seq,
                                         int n_heads, int max_len, int d_head, float scale,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "dadgpt_decode_attention_weights_bf16";
  if (int st = check_weights_decode(fn, out, weights_out, q, k_cache, v_cache, weights, lens, n_seq,
                                    n_heads, max_len, d_head, sizeof(*out), scale, workspace,
                                    workspace_bytes))
    return st;
  return from_hip(dadgpt::launch_weights_decode_bf16(
                      B(out), weights_out, B(q), B(k_cache), B(v_cache), weights, lens, n_seq,
                      n_heads, max_len, d_head, scale, workspace, as_stream(stream)),
                  fn);
}

int dadgpt_decode_attention_weights_f32(float* out, float* weights_out, const float* q,
                                        const float* k_cache, const float* v_cache,
                                        const float* weights, const int32_t* lens, int n_seq,
                                        int n_heads, int max_len, int d_head, float scale,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "dadgpt_decode_attention_weights_f32";
  if (int st = check_weights_decode(fn, out, weights_out, q, k_cache, v_cache, weights, lens, n_seq,
                                    n_heads, max_len, d_head, sizeof(*out), scale, workspace,
                                    workspace_bytes))
    return st;
  return from_hip(dadgpt::launch_weights_decode_f32(out, weights_out, q, k_cache, v_cache, weights,
                                                    lens, n_seq, n_heads, max_len, d_head, scale,
                                                    workspace, as_stream(stream)),
                  fn);
}

int dadgpt_kv_evict_bf16(uint16_t* k_out, uint16_t* v_out, float* weights_out, int32_t* kept,
                         int32_t* lens_out, const uint16_t* k, const uint16_t* v,
                         const float* weights, const int32_t* lens, int n_seq, int n_heads,
                         int max_len, int max_out, int d_head, int budget, int sinks, int recent,
                         void* stream) {
  return evict("dadgpt_kv_evict_bf16", k_out, v_out, weights_out, kept, lens_out, k, v, weights,
               lens, n_seq, n_heads, max_len, max_out, d_head, 2, budget, sinks, recent, stream);
}

int dadgpt_kv_evict_f32(float* k_out, float* v_out, float* weights_out, int32_t* kept,
                        int32_t* lens_out, const float* k, const float* v, const float* weights,
                        const int32_t* lens, int n_seq, int n_heads, int max_len, int max_out,
                        int d_head, int budget, int sinks, int recent, void* stream) {
  return evict("dadgpt_kv_evict_f32", k_out, v_out, weights_out, kept, lens_out, k, v, weights,
               lens, n_seq, n_heads, max_len, max_out, d_head, 4, budget, sinks, recent, stream);
}

}  // extern "C"
