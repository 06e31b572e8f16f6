"""Python mirror of include/dadgpt/paged_cache.h: KV caches in pages over libdadgpt_attn.so.

- ``paged_append`` writes the new tokens of ragged sequences into the pages that a block table names,
  rotating q and k on the way (``rope``);
- ``paged_attention`` attends from each sequence's new tokens, one or thousands, over its pages.

The reference has one cache for one sequence (``src/model.hpp:140-152``). As in ``attention``, the
buffers are torch tensors, work runs on torch's current stream, every call raises on failure and
there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import attention as _attn
from .attention import _check, _ptrs, _same_device, _stream_ptr, _workspace

# Symbols declared in include/dadgpt/paged_cache.h.
PAGED_SYMBOLS = (
    "dadgpt_paged_append_bf16",
    "dadgpt_paged_append_f32",
    "dadgpt_paged_workspace_bytes",
    "dadgpt_paged_attention_bf16",
    "dadgpt_paged_attention_f32",
)

# Tokens that a page can have (of one KV head), and those that a sequence can (the header's
# DADGPT_PAGED_MAX_LEN).
PAGES, MAX_LEN = (16, 32, 64, 128), 65535 * 256

_lib = None


def lib():
    """The loaded library with this header's signatures."""
    global _lib
    if _lib is not None:
        return _lib
    L = _attn.lib()
    vp, i, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    i64 = ctypes.c_int64
    L.dadgpt_paged_workspace_bytes.argtypes = [i] * 8
    for name in ("bf16", "f32"):
        getattr(L, "dadgpt_paged_append_" + name).argtypes = (
            [vp, vp, vp, i64, vp, i64, vp, vp, i64, vp, vp, vp] + [i] * 9 + [vp, i, i, f, vp])
        getattr(L, "dadgpt_paged_attention_" + name).argtypes = (
            [vp, i64, vp, i64] + [vp] * 5 + [i] * 9 + [f, vp, sz, vp])
    for name in PAGED_SYMBOLS:
        getattr(L, name).restype = sz if name.endswith("workspace_bytes") else i
    _lib = L
    return L


_entries = {}  # (name, element type) -> entry point


def _by_dtype(name, dtype):
    fn = _entries.get((name, dtype))
    if fn is None:
        suffix = {torch.bfloat16: "_bf16", torch.float32: "_f32"}.get(dtype)
        if suffix is None:
            raise TypeError(f"{name}: tensors must be bfloat16 or float32, got {dtype}")
        fn = _entries[name, dtype] = getattr(lib(), name + suffix)
    return fn


def paged_cache(n_pages: int, n_kv_heads: int, page: int, d_head: int, dtype=torch.bfloat16,
                device="cuda"):
    """An empty pool of pages: (k_pages, v_pages)."""
    if page not in PAGES:
        raise ValueError(f"page={page} must be one of {PAGES}")
    shape = (n_pages, n_kv_heads, page, d_head)
    return tuple(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))


def _rows(t, name, shape, dtype):
    """Address and pitch of a [rows, heads, d_head] view whose rows hold their heads side by side."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not dtype:
        raise TypeError(f"{name} must be a device tensor of {dtype}")
    s, (rows, heads, D) = t.stride(), shape
    if t.shape != shape or s[2] != 1 or (heads > 1 and s[1] != D):
        raise ValueError(f"{name} must be a {tuple(shape)} view with the heads of a row side by side, "
                         f"got {tuple(t.shape)} with strides {s}")
    return t.data_ptr(), s[0] if rows > 1 else heads * D


def _step(k_pages, v_pages, block_table, row_start, lens, dtype):
    """Addresses and sizes of what every call takes."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must be [n_pages, n_kv_heads, page, d_head]")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_seq, max_pages]")
    n = k_pages.numel()
    pk, pv = _ptrs(dtype, n, (k_pages, v_pages), ("k_pages", "v_pages"))
    n_seq, max_pages = block_table.shape
    pt, = _ptrs(torch.int32, n_seq * max_pages, (block_table,), ("block_table",))
    pr, = _ptrs(torch.int32, n_seq + 1, (row_start,), ("row_start",))
    pl, = _ptrs(torch.int32, n_seq, (lens,), ("lens",))
    return pk, pv, pt, pr, pl, n_seq, max_pages


def paged_append(k_pages, v_pages, q_out, q, k, v, block_table, row_start, lens, max_rows: int,
                 freqs=None, interleaved: bool = False, magnitude: float = 1.0,
                 stream=None) -> None:
    """Writes the rows of k and v [rows, n_kv_heads, d_head] into the pages, and q [rows, n_heads,
    d_head] into q_out (may be q; both None: k and v alone), views whose rows hold their heads side by
    side, as slices of a fused projection's output do; those of k and v lie equally far apart. Sequence s owns rows row_start[s] ..
    row_start[s + 1] - 1, max_rows at most; lens counts its tokens with them, so they are its last;
    token j goes to slot j % page of page block_table[s, j // page]. freqs (rope.rope_frequencies):
    rotate q and k by their token numbers as rope.rope does."""
    dtype = k_pages.dtype
    fn = _by_dtype("dadgpt_paged_append", dtype)
    pk, pv, pt, pr, pl, n_seq, max_pages = _step(k_pages, v_pages, block_table, row_start, lens, dtype)
    n_pages, Hkv, page, D = k_pages.shape
    rows = k.shape[0]
    xk, ld_kv = _rows(k, "k", (rows, Hkv, D), dtype)
    xv, ld_v = _rows(v, "v", (rows, Hkv, D), dtype)
    if ld_v != ld_kv:
        raise ValueError("the rows of k and v must lie equally far apart")
    H, xq, xo, ld_q, ld_out = Hkv, None, None, 0, 0
    if q is not None or q_out is not None:
        if q is None or q_out is None or q.dim() != 3:
            raise ValueError("q and q_out must be [rows, n_heads, d_head] views together, or both None")
        H = q.shape[1]
        xq, ld_q = _rows(q, "q", (rows, H, D), dtype)
        xo, ld_out = _rows(q_out, "q_out", (rows, H, D), dtype)
    pf, rot = None, 0
    if freqs is not None:
        pf, = _ptrs(torch.float64, 1, (freqs,), ("freqs",))
        rot = 2 * freqs.numel()
    _same_device((k_pages, v_pages, q_out, q, k, v, block_table, row_start, lens, freqs))
    _check(fn(pk, pv, xo, ld_out, xq, ld_q, xk, xv, ld_kv, pt, pr, pl, n_seq, H, Hkv, rows, max_rows,
              n_pages, page, max_pages, D, pf, rot, interleaved, magnitude, _stream_ptr(stream)))


def paged_workspace_bytes(n_seq: int, n_heads: int, n_kv_heads: int, rows: int, max_rows: int,
                          page: int, max_pages: int, d_head: int) -> int:
    return int(lib().dadgpt_paged_workspace_bytes(n_seq, n_heads, n_kv_heads, rows, max_rows, page,
                                                  max_pages, d_head))


def paged_workspace(q, k_pages, block_table, max_rows: int):
    """The zero-filled workspace that paged_attention needs for tensors of these shapes (and for fewer
    sequences, rows or pages to a sequence), or None when it needs none. Calls that overlap in time
    need one each."""
    rows, H, D = q.shape
    n_seq, max_pages = block_table.shape
    nbytes = paged_workspace_bytes(n_seq, H, k_pages.shape[1], rows, max_rows, k_pages.shape[2],
                                   max_pages, D)
    return torch.zeros(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None


def paged_attention(out, q, k_pages, v_pages, block_table, row_start, lens, max_rows: int,
                    scale: float, workspace, stream=None) -> None:
    """out = softmax(scale q k^T) v for the new tokens q [rows, n_heads, d_head] (rows as in
    paged_append, out may be q), each over its sequence's tokens up to itself. Query head h reads KV head
    h // (n_heads // n_kv_heads). Rows behind the last sequence are left as they were. Equal steps give
    equal bits; in a step with other sequences a sequence's may differ by roundings."""
    dtype = q.dtype
    fn = _by_dtype("dadgpt_paged_attention", dtype)
    pk, pv, pt, pr, pl, n_seq, max_pages = _step(k_pages, v_pages, block_table, row_start, lens, dtype)
    n_pages, Hkv, page, D = k_pages.shape
    if q.dim() != 3:
        raise ValueError("q must be a [rows, n_heads, d_head] view")
    rows, H = q.shape[:2]
    xq, ld_q = _rows(q, "q", (rows, H, D), dtype)
    xo, ld_out = _rows(out, "out", (rows, H, D), dtype)
    _same_device((out, q, k_pages, v_pages, block_table, row_start, lens, workspace))
    _check(fn(xo, ld_out, xq, ld_q, pk, pv, pt, pr, pl, n_seq, H, Hkv, rows, max_rows, n_pages, page,
              max_pages, D, scale, *_workspace(workspace), _stream_ptr(stream)))
