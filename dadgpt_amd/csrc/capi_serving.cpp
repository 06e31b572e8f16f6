// extern "C" entry points of the rotary positions, the paged caches and the sampling (declared in
// include/dadgpt/rope.h, paged_cache.h and sampling.h), with the checks and errors of capi.cpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "capi_util.hpp"
#include "dadgpt/paged_cache.h"
#include "dadgpt/rope.h"
#include "dadgpt/sampling.h"
#include "kernels.hpp"
#include "serving.hpp"

namespace {

using namespace dadgpt::capi;
using dadgpt::bf16;
using dadgpt::PagedStep;
using dadgpt::Rope;
using dadgpt::Span;
using dadgpt::Strides64;

constexpr int64_t kMostPitch = 1 << 24;

int check_aligned(const char* fn, const char* name, const void* p, uintptr_t bytes) {
  if (p == nullptr) return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s is null", fn, name);
  if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s is not %d-byte aligned", fn, name, (int)bytes);
  return DADGPT_OK;
}

int check_head(const char* fn, int d_head) {
  if (!supported(d_head))
    return fail(DADGPT_ERR_UNSUPPORTED, "%s: unsupported d_head %d", fn, d_head);
  return DADGPT_OK;
}

// ------------------------------------------------------------------------ overlap

// A tensor of rows of `width` elements at batch, head and row strides (elements): B, H and S of them.
struct View {
  const void* p;
  const char* name;
  Strides64 t;
  long long n[3], width;
  int elem;
  Span span() const {
    return {p, (size_t)elem * ((n[0] - 1) * t.batch + (n[1] - 1) * t.head + (n[2] - 1) * t.row + width)};
  }
};

struct Dim {
  long long stride, lo, hi;  // the difference of two indices lies in [lo, hi]
};

// Whether `off` = sum of i_x stride_x, lo_x <= i_x <= hi_x, but for a difference d with -wb < d < wa:
// whether some row of one tensor (width wa) meets one of another (wb) that begins `off` elements behind.
// Searched from the largest stride down; rows that a short search does not tell apart meet.
bool rows_meet(long long off, const Dim* dim, const Dim* end, long long wa, long long wb, int* steps) {
  if (++*steps > 4096) return true;
  if (dim == end) return off < wa && -off < wb;
  long long most = wa - 1, least = 1 - wb;  // what the dimensions after this one reach
  for (const Dim* x = dim + 1; x != end; ++x) most += x->stride * x->hi, least += x->stride * x->lo;
  if (dim->stride == 0) return rows_meet(off, dim + 1, end, wa, wb, steps);
  auto floor_div = [](long long a, long long b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
  const long long first = std::max(dim->lo, -floor_div(-(off - most), dim->stride));
  const long long last = std::min(dim->hi, floor_div(off - least, dim->stride));
  for (long long i = first; i <= last; ++i)
    if (rows_meet(off - i * dim->stride, dim + 1, end, wa, wb, steps)) return true;
  return false;
}

// Whether two tensors have an element in common: by their rows where the strides of the dimensions that
// both have more than one of agree, otherwise by their whole extents.
bool meet(const View& a, const View& b) {
  if (a.p == nullptr || b.p == nullptr || !dadgpt::overlap(a.span(), b.span())) return false;
  const long long d = reinterpret_cast<intptr_t>(b.p) - reinterpret_cast<intptr_t>(a.p);
  if (d % a.elem != 0) return true;
  const long long sa[3] = {a.t.batch, a.t.head, a.t.row}, sb[3] = {b.t.batch, b.t.head, b.t.row};
  Dim dims[3];
  for (int i = 0; i < 3; ++i) {
    if (a.n[i] > 1 && b.n[i] > 1 && sa[i] != sb[i]) return true;
    dims[i] = Dim{a.n[i] > 1 ? sa[i] : sb[i], 1 - b.n[i], a.n[i] - 1};
  }
  std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  int steps = 0;
  return rows_meet(d / a.elem, dims, dims + 3, a.width, b.width, &steps);
}

// Whether two of a tensor's own rows have an element in common.
bool own_rows_meet(const View& a) {
  Dim dims[3] = {{a.t.batch, 1 - a.n[0], a.n[0] - 1},
                 {a.t.head, 1 - a.n[1], a.n[1] - 1},
                 {a.t.row, 1 - a.n[2], a.n[2] - 1}};
  std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  int steps = 0;
  for (int x = 0; x < 3; ++x) {  // the first dimension in which the two rows differ
    if (dims[x].hi == 0) continue;
    const Dim differ{dims[x].stride, 1, dims[x].hi};
    Dim rest[3] = {differ};
    for (int y = x + 1; y < 3; ++y) rest[y - x] = dims[y];
    if (rows_meet(0, rest, rest + 3 - x, a.width, a.width, &steps)) return true;
  }
  return false;
}

int overlaps(const char* fn, const char* a, const char* b) {
  return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: %s overlaps %s", fn, a, b);
}

// A flat array as a View of one row of bytes.
View flat(const void* p, size_t bytes, const char* name) {
  return View{p, name, {0, 0, 0}, {1, 1, 1}, (long long)bytes, 1};
}
bool flat_meets(const View& f, const View& v) {
  return f.p != nullptr && v.p != nullptr && dadgpt::overlap(f.span(), v.span());
}

// ------------------------------------------------------------------------ rotary positions

int check_rope(const char* fn, int d_head, const double* freqs, int rot_dim, float magnitude) {
  if (int st = check_aligned(fn, "freqs", freqs, 8)) return st;
  if (rot_dim < 8 || rot_dim > d_head || rot_dim % 8 != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: rot_dim=%d must be a multiple of 8 in [8, d_head = %d]", fn, rot_dim, d_head);
  if (!std::isfinite(magnitude))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: magnitude must be finite", fn);
  return DADGPT_OK;
}

template <typename T, typename U, typename F>
int rope(const char* fn, T* q_out, T* k_out, const T* q, const T* k,
         const dadgpt_head_strides* strides, int batch, int H, int Hkv, int S, int d_head,
         const double* freqs, int rot_dim, int interleaved, float magnitude, bool inverse,
         const int32_t* positions, void* stream, F launch) {
  const bool backward = inverse;
  const char* names[4] = {backward ? "dq_out" : "q", backward ? "dk_out" : "k",
                          backward ? "dq" : "q_out", backward ? "dk" : "k_out"};
  const bool has_k = Hkv != 0 || k != nullptr || k_out != nullptr;
  if (int st = check_ptrs(fn, {q_out, q})) return st;
  if (has_k)
    if (int st = check_ptrs(fn, {k_out, k})) return st;
  if (strides == nullptr) return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: strides is null", fn);
  if (int st = check_head(fn, d_head)) return st;
  if (batch < 1 || H < 1 || S < 1 || Hkv < (has_k ? 1 : 0))
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: B=%d, n_heads=%d, n_kv_heads=%d and S=%d must be positive", fn, batch, H, Hkv, S);
  if (int st = check_rope(fn, d_head, freqs, rot_dim, magnitude)) return st;
  if (positions != nullptr)
    if (int st = check_aligned(fn, "positions", positions, 4)) return st;
  dadgpt::RopeShape shape{batch, H, Hkv, S, d_head, {}};
  constexpr int64_t kMost = int64_t(1) << 40;
  for (int i = 0; i < 4; ++i) {
    if (!has_k && i % 2 == 1) continue;
    const dadgpt_head_strides& t = strides[i];
    for (int64_t x : {t.batch, t.head, t.row})
      if (x < 0 || x % 8 != 0 || x > kMost)
        return fail(DADGPT_ERR_INVALID_ARGUMENT,
                    "%s: strides of %s {batch %lld, head %lld, row %lld}: each must be a non-negative "
                    "multiple of 8, at most 2^40",
                    fn, names[i], (long long)t.batch, (long long)t.head, (long long)t.row);
    shape.t[i] = Strides64{t.batch, t.head, t.row};
  }
  // threads: 8 for a head of a row at most, numbered in 32 bits
  if ((long long)batch * S > (1LL << 31) / 8 ||
      (long long)batch * S * (H + (long long)Hkv) > (1LL << 31) / 8)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: B=%d x S=%d x %d heads exceeds the launch limits", fn, batch, S, H + Hkv);
  const void* tensor[4] = {q, k, q_out, k_out};
  View v[4];
  for (int i = 0; i < 4; ++i)
    v[i] = View{has_k || i % 2 == 0 ? tensor[i] : nullptr, names[i], shape.t[i],
                {batch, i % 2 == 0 ? H : Hkv, S}, d_head, (int)sizeof(T)};
  auto replaces = [&](int out, int in) {
    return v[out].p == v[in].p && shape.t[out].batch == shape.t[in].batch &&
           shape.t[out].head == shape.t[in].head && shape.t[out].row == shape.t[in].row;
  };
  const View f = flat(freqs, sizeof(double) * rot_dim / 2, "freqs");
  const View pos = flat(positions, 4 * (size_t)batch * S, "positions");
  for (int out = 2; out < 4; ++out) {
    if (v[out].p == nullptr) continue;
    if (own_rows_meet(v[out]))
      return fail(DADGPT_ERR_INVALID_ARGUMENT,
                  "%s: rows of %s overlap each other (strides {batch %lld, head %lld, row %lld})", fn,
                  names[out], shape.t[out].batch, shape.t[out].head, shape.t[out].row);
    for (int in = 0; in < 2; ++in)
      if (!(out - 2 == in && replaces(out, in)) && meet(v[out], v[in]))
        return overlaps(fn, names[out], names[in]);
    if (flat_meets(f, v[out])) return overlaps(fn, names[out], "freqs");
    if (flat_meets(pos, v[out])) return overlaps(fn, names[out], "positions");
  }
  if (meet(v[2], v[3])) return overlaps(fn, names[2], names[3]);
  const Rope r{freqs, rot_dim, interleaved != 0, inverse, magnitude};
  return from_hip(launch((U*)q_out, (U*)k_out, (const U*)q, (const U*)k, shape, r, positions,
                         as_stream(stream)),
                  fn);
}

// ------------------------------------------------------------------------ paged caches

int check_step(const char* fn, const PagedStep& s) {
  if (int st = check_aligned(fn, "block_table", s.table, 4)) return st;
  if (int st = check_aligned(fn, "row_start", s.row_start, 4)) return st;
  if (int st = check_aligned(fn, "lens", s.lens, 4)) return st;
  if (s.n_seq < 1 || s.H < 1 || s.Hkv < 1 || s.rows < 1 || s.max_rows < 1 || s.n_pages < 1 ||
      s.max_pages < 1)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: n_seq=%d, n_heads=%d, n_kv_heads=%d, rows=%d, max_rows=%d, n_pages=%d and "
                "max_pages=%d must be positive",
                fn, s.n_seq, s.H, s.Hkv, s.rows, s.max_rows, s.n_pages, s.max_pages);
  if (s.H % s.Hkv != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: n_heads=%d is no multiple of n_kv_heads=%d", fn,
                s.H, s.Hkv);
  if (s.page != 16 && s.page != 32 && s.page != 64 && s.page != 128)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: page=%d must be 16, 32, 64 or 128", fn, s.page);
  if (int st = check_head(fn, s.D)) return st;
  if ((long long)s.max_pages * s.page > DADGPT_PAGED_MAX_LEN)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: max_pages=%d x page=%d exceeds %d tokens", fn,
                s.max_pages, s.page, DADGPT_PAGED_MAX_LEN);
  if (s.n_seq > 65535 || s.H > 65535 || s.rows > (1 << 24))
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: n_seq=%d, n_heads=%d or rows=%d exceeds the launch limits", fn, s.n_seq, s.H,
                s.rows);
  return DADGPT_OK;
}

int check_pitch(const char* fn, const char* name, int64_t ld, long long width) {
  if (ld < width || ld > kMostPitch || ld % 8 != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: %s=%lld must be a multiple of 8 in [%lld, 2^24]", fn, name, (long long)ld, width);
  return DADGPT_OK;
}

View token_rows(const void* p, const char* name, int rows, int64_t ld, long long width, int elem) {
  return View{p, name, {0, 0, ld}, {1, 1, rows}, width, elem};
}

// The step's device arrays and pages against an output.
int check_step_apart(const char* fn, const PagedStep& s, const View& out) {
  const View arrays[3] = {flat(s.table, 4 * (size_t)s.n_seq * s.max_pages, "block_table"),
                          flat(s.row_start, 4 * ((size_t)s.n_seq + 1), "row_start"),
                          flat(s.lens, 4 * (size_t)s.n_seq, "lens")};
  for (const View& a : arrays)
    if (flat_meets(a, out)) return overlaps(fn, out.name, a.name);
  return DADGPT_OK;
}

size_t cache_bytes(const PagedStep& s, size_t elem) {
  return elem * s.n_pages * s.Hkv * s.page * s.D;
}

template <typename T, typename U, typename F>
int append(const char* fn, T* k_pages, T* v_pages, T* q_out, int64_t ld_out, const T* q,
           int64_t ld_q, const T* k, const T* v, int64_t ld_kv, const PagedStep& s, const double* freqs, int rot_dim,
           int interleaved, float magnitude, void* stream, F launch) {
  if (int st = check_ptrs(fn, {k_pages, v_pages, k, v})) return st;
  if ((q == nullptr) != (q_out == nullptr))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: q and q_out are null together", fn);
  if (q != nullptr)
    if (int st = check_ptrs(fn, {q_out, q})) return st;
  if (int st = check_step(fn, s)) return st;
  const long long wq = (long long)s.H * s.D, wkv = (long long)s.Hkv * s.D;
  if (int st = check_pitch(fn, "ld_kv", ld_kv, wkv)) return st;
  if (q != nullptr) {
    if (int st = check_pitch(fn, "ld_q", ld_q, wq)) return st;
    if (int st = check_pitch(fn, "ld_out", ld_out, wq)) return st;
  }
  if (freqs == nullptr) {
    if (rot_dim != 0)
      return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: rot_dim=%d without freqs", fn, rot_dim);
  } else if (int st = check_rope(fn, s.D, freqs, rot_dim, magnitude)) {
    return st;
  }
  const int elem = sizeof(T);
  // threads: 8 for a head of a row at most; workgroups of one sequence along grid.x
  if ((long long)s.max_rows * (s.H + 2LL * s.Hkv) > (1LL << 31) / 8)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: max_rows=%d x n_heads=%d exceeds the launch limits",
                fn, s.max_rows, s.H);
  const View K = flat(k_pages, cache_bytes(s, elem), "k_pages");
  const View V = flat(v_pages, cache_bytes(s, elem), "v_pages");
  const View QO = token_rows(q_out, "q_out", s.rows, ld_out, wq, elem);
  const View in[3] = {token_rows(q, "q", s.rows, ld_q, wq, elem),
                      token_rows(k, "k", s.rows, ld_kv, wkv, elem),
                      token_rows(v, "v", s.rows, ld_kv, wkv, elem)};
  const View f = flat(freqs, sizeof(double) * rot_dim / 2, "freqs");
  if (flat_meets(K, V)) return overlaps(fn, "k_pages", "v_pages");
  for (const View& c : {K, V}) {
    if (flat_meets(c, QO)) return overlaps(fn, c.name, "q_out");
    for (const View& x : in)
      if (flat_meets(c, x)) return overlaps(fn, c.name, x.name);
    if (flat_meets(f, c)) return overlaps(fn, c.name, "freqs");
    if (int st = check_step_apart(fn, s, c)) return st;
  }
  if (q_out != nullptr) {
    const bool in_place = q_out == q && ld_out == ld_q;
    for (const View& x : in)
      if (!(in_place && &x == &in[0]) && meet(QO, x)) return overlaps(fn, "q_out", x.name);
    if (flat_meets(f, QO)) return overlaps(fn, "q_out", "freqs");
    if (int st = check_step_apart(fn, s, QO)) return st;
  }
  const Rope r{freqs, freqs == nullptr ? 0 : rot_dim, interleaved != 0, false, magnitude};
  return from_hip(launch((U*)k_pages, (U*)v_pages, (U*)q_out, ld_out, (const U*)q, ld_q, (const U*)k,
                         (const U*)v, ld_kv, s, r, as_stream(stream)),
                  fn);
}

template <typename T, typename U, typename F>
int attend(const char* fn, T* out, int64_t ld_out, const T* q, int64_t ld_q, const T* k_pages,
           const T* v_pages, const PagedStep& s, float scale, void* ws, size_t ws_bytes,
           void* stream, F launch) {
  if (int st = check_ptrs(fn, {out, q, k_pages, v_pages})) return st;
  if (int st = check_step(fn, s)) return st;
  const long long wq = (long long)s.H * s.D;
  if (int st = check_pitch(fn, "ld_out", ld_out, wq)) return st;
  if (int st = check_pitch(fn, "ld_q", ld_q, wq)) return st;
  if (!std::isfinite(scale))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: scale must be finite", fn);
  const int elem = sizeof(T);
  if (!dadgpt::paged_fits(s, elem))
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: n_seq=%d and rows=%d x %d query heads to a KV head exceed the launch limits", fn,
                s.n_seq, s.rows, s.H / s.Hkv);
  const View O = token_rows(out, "out", s.rows, ld_out, wq, elem);
  const View Q = token_rows(q, "q", s.rows, ld_q, wq, elem);
  const View K = flat(k_pages, cache_bytes(s, elem), "k_pages");
  const View V = flat(v_pages, cache_bytes(s, elem), "v_pages");
  if (!(out == q && ld_out == ld_q) && meet(O, Q)) return overlaps(fn, "out", "q");
  if (flat_meets(K, O)) return overlaps(fn, "out", "k_pages");
  if (flat_meets(V, O)) return overlaps(fn, "out", "v_pages");
  if (int st = check_step_apart(fn, s, O)) return st;
  const size_t need = dadgpt::paged_workspace_needed(s, elem);
  if (need > 0) {
    if (ws == nullptr || ws_bytes < need)
      return fail(DADGPT_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", fn,
                  ws == nullptr ? 0 : ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
      return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: workspace is not 16-byte aligned", fn);
    const View W = flat(ws, ws_bytes, "the workspace");
    for (const View& x : {O, Q, K, V})
      if (flat_meets(W, x)) return overlaps(fn, "the workspace", x.name);
    if (int st = check_step_apart(fn, s, W)) return st;
  }
  return from_hip(launch((U*)out, ld_out, (const U*)q, ld_q, (const U*)k_pages, (const U*)v_pages, s,
                         scale, ws, ws_bytes, as_stream(stream)),
                  fn);
}

// ------------------------------------------------------------------------ sampling

template <typename T, typename U, typename F>
int sample(const char* fn, int32_t* tokens, float* probs, const T* logits, int64_t ld, int rows,
           int vocab, const dadgpt::SampleSettings& set, void* stream, F launch) {
  if (int st = check_aligned(fn, "tokens", tokens, 4)) return st;
  if (int st = check_aligned(fn, "logits", logits, sizeof(T))) return st;
  if (int st = check_aligned(fn, "uniforms", set.uniforms, 4)) return st;
  const void* optional[5] = {probs, set.temperature, set.top_k, set.top_p, set.min_p};
  const char* names[5] = {"probs", "temperature", "top_k", "top_p", "min_p"};
  for (int i = 0; i < 5; ++i)
    if (optional[i] != nullptr)
      if (int st = check_aligned(fn, names[i], optional[i], 4)) return st;
  if (rows < 1 || vocab < 1)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: rows=%d and vocab=%d must be positive", fn, rows,
                vocab);
  if (vocab > DADGPT_SAMPLE_MAX_VOCAB || rows >= (1 << 21))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: rows=%d or vocab=%d exceeds the limits", fn, rows,
                vocab);
  if (ld < vocab || ld > (int64_t(1) << 40))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: ld=%lld must be in [vocab = %d, 2^40]", fn,
                (long long)ld, vocab);
  const size_t n = 4 * (size_t)rows;
  const View L = flat(logits, sizeof(T) * ((rows - 1) * ld + vocab), "logits");
  const View tok = flat(tokens, n, "tokens"), pr = flat(probs, n, "probs");
  if (flat_meets(tok, pr)) return overlaps(fn, "tokens", "probs");
  for (const View& o : {tok, pr}) {
    if (flat_meets(o, L)) return overlaps(fn, o.name, "logits");
    if (flat_meets(o, flat(set.uniforms, n, "uniforms"))) return overlaps(fn, o.name, "uniforms");
    for (int i = 1; i < 5; ++i)
      if (flat_meets(o, flat(optional[i], n, names[i]))) return overlaps(fn, o.name, names[i]);
  }
  return from_hip(launch(tokens, probs, (const U*)logits, ld, rows, vocab, set, as_stream(stream)),
                  fn);
}

PagedStep step_of(const int32_t* table, const int32_t* row_start, const int32_t* lens, int n_seq,
                  int H, int Hkv, int rows, int max_rows, int n_pages, int page, int max_pages,
                  int D) {
  return PagedStep{table,  row_start, lens, n_seq, H, Hkv, rows, std::min(max_rows, rows),
                   n_pages, page, max_pages, D};
}

}  // namespace

extern "C" {

int dadgpt_rope_frequencies(double* freqs, int rot_dim, double base, int scaling, double factor,
                            int original_len, double slow, double fast) {
  const char* fn = "dadgpt_rope_frequencies";
  if (freqs == nullptr) return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: freqs is null", fn);
  if (rot_dim < 2 || rot_dim % 2 != 0)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: rot_dim=%d must be even and positive", fn, rot_dim);
  if (!(base > 0.0) || !std::isfinite(base) || !(factor > 0.0) || !std::isfinite(factor))
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: base=%g and factor=%g must be positive and finite",
                fn, base, factor);
  if (scaling < DADGPT_ROPE_UNSCALED || scaling > DADGPT_ROPE_PARTS)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: no scaling %d", fn, scaling);
  if (scaling == DADGPT_ROPE_BASE && rot_dim < 4)
    return fail(DADGPT_ERR_INVALID_ARGUMENT, "%s: scaling by the base wants rot_dim >= 4", fn);
  if (scaling == DADGPT_ROPE_PARTS &&
      (original_len < 1 || !(slow < fast) || !std::isfinite(slow) || !std::isfinite(fast)))
    return fail(DADGPT_ERR_INVALID_ARGUMENT,
                "%s: original_len=%d must be positive, slow=%g below fast=%g", fn, original_len, slow,
                fast);
  if (scaling == DADGPT_ROPE_BASE) base *= std::pow(factor, rot_dim / (rot_dim - 2.0));
  for (int i = 0; i < rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot_dim);
    if (scaling == DADGPT_ROPE_LINEAR) f /= factor;
    if (scaling == DADGPT_ROPE_PARTS) {
      const double turns = original_len * f / (2.0 * M_PI);
      const double g = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
      f *= g + (1.0 - g) / factor;
    }
    freqs[i] = f;
  }
  return ok();
}

int dadgpt_rope_bf16(uint16_t* q_out, uint16_t* k_out, const uint16_t* q, const uint16_t* k,
                     const dadgpt_head_strides* strides, int batch, int H, int Hkv, int S, int d_head,
                     const double* freqs, int rot_dim, int interleaved, float magnitude,
                     const int32_t* positions, void* stream) {
  return rope<uint16_t, bf16>("dadgpt_rope_bf16", q_out, k_out, q, k, strides, batch, H, Hkv, S,
                              d_head, freqs, rot_dim, interleaved, magnitude, false, positions, stream,
                              dadgpt::launch_rope_bf16);
}
int dadgpt_rope_f32(float* q_out, float* k_out, const float* q, const float* k,
                    const dadgpt_head_strides* strides, int batch, int H, int Hkv, int S, int d_head,
                    const double* freqs, int rot_dim, int interleaved, float magnitude,
                    const int32_t* positions, void* stream) {
  return rope<float, float>("dadgpt_rope_f32", q_out, k_out, q, k, strides, batch, H, Hkv, S, d_head,
                            freqs, rot_dim, interleaved, magnitude, false, positions, stream,
                            dadgpt::launch_rope_f32);
}
int dadgpt_rope_backward_bf16(uint16_t* dq, uint16_t* dk, const uint16_t* dq_out,
                              const uint16_t* dk_out, const dadgpt_head_strides* strides, int batch,
                              int H, int Hkv, int S, int d_head, const double* freqs, int rot_dim,
                              int interleaved, float magnitude, const int32_t* positions,
                              void* stream) {
  return rope<uint16_t, bf16>("dadgpt_rope_backward_bf16", dq, dk, dq_out, dk_out, strides, batch, H,
                              Hkv, S, d_head, freqs, rot_dim, interleaved, magnitude, true, positions,
                              stream, dadgpt::launch_rope_bf16);
}
int dadgpt_rope_backward_f32(float* dq, float* dk, const float* dq_out, const float* dk_out,
                             const dadgpt_head_strides* strides, int batch, int H, int Hkv, int S,
                             int d_head, const double* freqs, int rot_dim, int interleaved,
                             float magnitude, const int32_t* positions, void* stream) {
  return rope<float, float>("dadgpt_rope_backward_f32", dq, dk, dq_out, dk_out, strides, batch, H, Hkv,
                            S, d_head, freqs, rot_dim, interleaved, magnitude, true, positions, stream,
                            dadgpt::launch_rope_f32);
}

int dadgpt_paged_append_bf16(uint16_t* k_pages, uint16_t* v_pages, uint16_t* q_out, int64_t ld_out,
                             const uint16_t* q, int64_t ld_q, const uint16_t* k,
                             const uint16_t* v, int64_t ld_kv, const int32_t* block_table, const int32_t* row_start,
                             const int32_t* lens, int n_seq, int n_heads, int n_kv_heads, int rows,
                             int max_rows, int n_pages, int page, int max_pages, int d_head,
                             const double* freqs, int rot_dim, int interleaved, float magnitude,
                             void* stream) {
  return append<uint16_t, bf16>(
      "dadgpt_paged_append_bf16", k_pages, v_pages, q_out, ld_out, q, ld_q, k, v, ld_kv,
      step_of(block_table, row_start, lens, n_seq, n_heads, n_kv_heads, rows, max_rows, n_pages, page,
              max_pages, d_head),
      freqs, rot_dim, interleaved, magnitude, stream, dadgpt::launch_paged_append_bf16);
}
int dadgpt_paged_append_f32(float* k_pages, float* v_pages, float* q_out, int64_t ld_out,
                            const float* q, int64_t ld_q, const float* k, const float* v,
                            int64_t ld_kv, const int32_t* block_table, const int32_t* row_start,
                            const int32_t* lens, int n_seq, int n_heads, int n_kv_heads, int rows,
                            int max_rows, int n_pages, int page, int max_pages, int d_head,
                            const double* freqs, int rot_dim, int interleaved, float magnitude,
                            void* stream) {
  return append<float, float>(
      "dadgpt_paged_append_f32", k_pages, v_pages, q_out, ld_out, q, ld_q, k, v, ld_kv,
      step_of(block_table, row_start, lens, n_seq, n_heads, n_kv_heads, rows, max_rows, n_pages, page,
              max_pages, d_head),
      freqs, rot_dim, interleaved, magnitude, stream, dadgpt::launch_paged_append_f32);
}

size_t dadgpt_paged_workspace_bytes(int n_seq, int n_heads, int n_kv_heads, int rows, int max_rows,
                                    int page, int max_pages, int d_head) {
  static const int32_t none[1] = {0};  // (the arrays are not looked at)
  const PagedStep s = step_of(none, none, none, n_seq, n_heads, n_kv_heads, rows, max_rows, 1, page,
                              max_pages, d_head);
  return check_step("dadgpt_paged_workspace_bytes", s) ? 0 : dadgpt::paged_workspace_bytes(s);
}

int dadgpt_paged_attention_bf16(uint16_t* out, int64_t ld_out, const uint16_t* q, int64_t ld_q,
                                const uint16_t* k_pages, const uint16_t* v_pages,
                                const int32_t* block_table, const int32_t* row_start,
                                const int32_t* lens, int n_seq, int n_heads, int n_kv_heads,
                                int rows, int max_rows, int n_pages, int page, int max_pages,
                                int d_head, float scale, void* workspace, size_t workspace_bytes,
                                void* stream) {
  return attend<uint16_t, bf16>(
      "dadgpt_paged_attention_bf16", out, ld_out, q, ld_q, k_pages, v_pages,
      step_of(block_table, row_start, lens, n_seq, n_heads, n_kv_heads, rows, max_rows, n_pages, page,
              max_pages, d_head),
      scale, workspace, workspace_bytes, stream, dadgpt::launch_paged_attention_bf16);
}
int dadgpt_paged_attention_f32(float* out, int64_t ld_out, const float* q, int64_t ld_q,
                               const float* k_pages, const float* v_pages,
                               const int32_t* block_table, const int32_t* row_start,
                               const int32_t* lens, int n_seq, int n_heads, int n_kv_heads,
                               int rows, int max_rows, int n_pages, int page, int max_pages,
                               int d_head, float scale, void* workspace, size_t workspace_bytes,
                               void* stream) {
  return attend<float, float>(
      "dadgpt_paged_attention_f32", out, ld_out, q, ld_q, k_pages, v_pages,
      step_of(block_table, row_start, lens, n_seq, n_heads, n_kv_heads, rows, max_rows, n_pages, page,
              max_pages, d_head),
      scale, workspace, workspace_bytes, stream, dadgpt::launch_paged_attention_f32);
}

int dadgpt_sample_bf16(int32_t* tokens, float* probs, const uint16_t* logits, int64_t ld, int rows,
                       int vocab, const float* uniforms, const float* temperature,
                       const int32_t* top_k, const float* top_p, const float* min_p, void* stream) {
  return sample<uint16_t, bf16>("dadgpt_sample_bf16", tokens, probs, logits, ld, rows, vocab,
                                {uniforms, temperature, top_p, min_p, top_k}, stream,
                                dadgpt::launch_sample_bf16);
}
int dadgpt_sample_f32(int32_t* tokens, float* probs, const float* logits, int64_t ld, int rows,
                      int vocab, const float* uniforms, const float* temperature,
                      const int32_t* top_k, const float* top_p, const float* min_p, void* stream) {
  return sample<float, float>("dadgpt_sample_f32", tokens, probs, logits, ld, rows, vocab,
                              {uniforms, temperature, top_p, min_p, top_k}, stream,
                              dadgpt::launch_sample_f32);
}

}  // extern "C"
