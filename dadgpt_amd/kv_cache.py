"""Python mirror of include/dadgpt/kv_cache.h: bounded KV caches over libdadgpt_attn.so.

- a cache held in 8 bits (e4m3 codes with a power-of-two scale for each block of tokens and head):
  ``kv8_append`` quantises new rows into it, ``decode_attention_kv8`` attends over it;
- eviction by accumulated attention weight: ``decode_attention_weights`` adds each key's
  probability to its weight, ``kv_evict`` cuts a cache back to its sinks, its last rows and the
  heaviest rows between.

The reference has one cache, fp32 and of full length (``src/model.hpp:140-152``). As in
``attention``, the buffers are torch tensors, work runs on torch's current stream, every call raises
on failure and there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import attention as _attn
from .attention import _check, _ptrs, _same_device, _stream_ptr, _workspace

# Symbols declared in include/dadgpt/kv_cache.h.
CACHE_SYMBOLS = (
    "dadgpt_kv8_blocks",
    "dadgpt_kv8_append_bf16",
    "dadgpt_kv8_append_f32",
    "dadgpt_decode_kv8_workspace_bytes",
    "dadgpt_decode_attention_kv8_bf16",
    "dadgpt_decode_attention_kv8_f32",
    "dadgpt_decode_weights_workspace_bytes",
    "dadgpt_decode_attention_weights_bf16",
    "dadgpt_decode_attention_weights_f32",
    "dadgpt_kv_evict_bf16",
    "dadgpt_kv_evict_f32",
)

# Tokens a block of an 8-bit cache can have, and the codes' type.
KV8_BLOCKS = (16, 32, 64, 128)
KV8_DTYPE = torch.float8_e4m3fn

_lib = None


def lib():
    """The loaded library with this header's signatures."""
    global _lib
    if _lib is not None:
        return _lib
    L = _attn.lib()
    vp, i, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    L.dadgpt_kv8_blocks.argtypes = [i, i]
    L.dadgpt_decode_kv8_workspace_bytes.argtypes = [i] * 4
    L.dadgpt_decode_weights_workspace_bytes.argtypes = [i] * 4
    for name in ("bf16", "f32"):
        getattr(L, "dadgpt_kv8_append_" + name).argtypes = ([vp] * 10 + [i] * 6 + [vp])
        getattr(L, "dadgpt_decode_attention_kv8_" + name).argtypes = (
            [vp] * 7 + [i] * 5 + [f, i, i, vp, sz, vp])
        getattr(L, "dadgpt_decode_attention_weights_" + name).argtypes = (
            [vp] * 7 + [i] * 4 + [f, vp, sz, vp])
        getattr(L, "dadgpt_kv_evict_" + name).argtypes = [vp] * 9 + [i] * 8 + [vp]
    for name in CACHE_SYMBOLS:
        getattr(L, name).restype = sz if name.endswith("workspace_bytes") else i
    _lib = L
    return L


_entries = {}  # (name, element type) -> entry point


def _by_dtype(name, dtype):
    """The entry point of `name` for bf16 or fp32 tensors."""
    fn = _entries.get((name, dtype))
    if fn is None:
        suffix = {torch.bfloat16: "_bf16", torch.float32: "_f32"}.get(dtype)
        if suffix is None:
            raise TypeError(f"{name}: tensors must be bfloat16 or float32, got {dtype}")
        fn = _entries[name, dtype] = getattr(lib(), name + suffix)
    return fn


# ------------------------------------------------------------------------ 8-bit cache

def kv8_blocks(max_len: int, block: int) -> int:
    """Blocks of `block` tokens in a cache of max_len rows: the scales' last dimension."""
    if max_len < 1 or block not in KV8_BLOCKS:
        raise ValueError(f"max_len={max_len} must be positive, block={block} one of {KV8_BLOCKS}")
    return (max_len + block - 1) // block


def kv8_cache(n_seq: int, n_heads: int, max_len: int, d_head: int, block: int, device="cuda"):
    """An empty 8-bit cache: (k_cache, v_cache, k_scale, v_scale)."""
    codes = (n_seq, n_heads, max_len, d_head)
    scales = (n_seq, n_heads, kv8_blocks(max_len, block))
    return (*(torch.zeros(codes, dtype=torch.uint8, device=device).view(KV8_DTYPE)
              for _ in range(2)),
            *(torch.zeros(scales, dtype=torch.float32, device=device) for _ in range(2)))


_Int64x6 = ctypes.c_int64 * 6


def _new_rows(t, name, shape, dtype):
    """Address and (batch, head, row) strides of a view of new rows; a dimension of one has no
    stride."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not dtype:
        raise TypeError(f"{name} must be a device tensor of {dtype}")
    strides = t.stride()
    if t.shape != shape or strides[3] != 1:
        raise ValueError(f"{name} must be a [n_seq, n_heads, rows, d_head] view with contiguous "
                         f"rows, got {tuple(t.shape)} with strides {strides}")
    return t.data_ptr(), [st if size > 1 else 0 for st, size in zip(strides, shape[:3])]


def kv8_append(k_cache, v_cache, k_scale, v_scale, k, v, lens, counts, n_seq: int, n_heads: int,
               rows: int, max_len: int, d_head: int, block: int, stream=None) -> None:
    """Appends k and v, [n_seq, n_heads, rows, d_head] views with contiguous rows (bf16 or fp32;
    the heads of a token-major projection will do), at cache rows lens[s] + t for t < counts[s]
    (counts None: all). lens, counts: device int32; the caller advances lens."""
    fn = _by_dtype("dadgpt_kv8_append", k.dtype)
    shape = (n_seq, n_heads, rows, d_head)
    pk, ks = _new_rows(k, "k", shape, k.dtype)
    pv, vs = _new_rows(v, "v", shape, k.dtype)
    c8, d8 = _ptrs(KV8_DTYPE, n_seq * n_heads * max_len * d_head, (k_cache, v_cache),
                   ("k_cache", "v_cache"))
    sc, sd = _ptrs(torch.float32, n_seq * n_heads * kv8_blocks(max_len, block),
                   (k_scale, v_scale), ("k_scale", "v_scale"))
    pl, pc = _ptrs(torch.int32, n_seq, (lens, counts), ("lens", "counts"))
    _same_device((k_cache, v_cache, k_scale, v_scale, k, v, lens, counts))
    strides = _Int64x6(*ks, *vs)  # two dadgpt_head_strides
    _check(fn(c8, d8, sc, sd, pk, pv, ctypes.byref(strides), ctypes.byref(strides, 24), pl, pc,
              n_seq, n_heads, rows, max_len, d_head, block, _stream_ptr(stream)))


def decode_kv8_workspace_bytes(n_seq: int, n_heads: int, max_len: int, d_head: int) -> int:
    return int(lib().dadgpt_decode_kv8_workspace_bytes(n_seq, n_heads, max_len, d_head))


def decode_kv8_workspace(n_seq, n_heads, max_len, d_head, device="cuda"):
    """The zero-filled workspace that decode_attention_kv8 needs, or None when it needs none."""
    nbytes = decode_kv8_workspace_bytes(n_seq, n_heads, max_len, d_head)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def decode_attention_kv8(out, q, k_cache, v_cache, k_scale, v_scale, lens, n_seq: int,
                         n_heads: int, max_len: int, d_head: int, block: int, scale: float,
                         window: int, sinks: int, workspace, stream=None) -> None:
    """attention.decode_attention over an 8-bit cache (q and out bf16 or fp32). window 0 sees the
    whole cache, window >= 1 rows [0, sinks) and [len - window, len)."""
    fn = _by_dtype("dadgpt_decode_attention_kv8", q.dtype)
    po, pq = _ptrs(q.dtype, n_seq * n_heads * d_head, (out, q), ("out", "q"))
    pk, pv = _ptrs(KV8_DTYPE, n_seq * n_heads * max_len * d_head, (k_cache, v_cache),
                   ("k_cache", "v_cache"))
    ps, pt = _ptrs(torch.float32, n_seq * n_heads * kv8_blocks(max_len, block),
                   (k_scale, v_scale), ("k_scale", "v_scale"))
    pl, = _ptrs(torch.int32, n_seq, (lens,), ("lens",))
    _same_device((out, q, k_cache, v_cache, k_scale, v_scale, lens, workspace))
    _check(fn(po, pq, pk, pv, ps, pt, pl, n_seq, n_heads, max_len, d_head, block, scale, window,
              sinks, *_workspace(workspace), _stream_ptr(stream)))


# ------------------------------------------------------------------------ eviction

def decode_weights_workspace_bytes(n_seq: int, n_heads: int, max_len: int, d_head: int) -> int:
    return int(lib().dadgpt_decode_weights_workspace_bytes(n_seq, n_heads, max_len, d_head))


def decode_weights_workspace(n_seq, n_heads, max_len, d_head, device="cuda"):
    """The workspace that decode_attention_weights needs, or None when it needs none. It holds
    nothing between calls; calls that overlap in time need one each."""
    nbytes = decode_weights_workspace_bytes(n_seq, n_heads, max_len, d_head)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def decode_attention_weights(out, weights_out, q, k_cache, v_cache, weights, lens, n_seq: int,
                             n_heads: int, max_len: int, d_head: int, scale: float, workspace,
                             stream=None) -> None:
    """attention.decode_attention that accumulates: weights_out = weights + each key's
    probability, fp32 [n_seq, n_heads, max_len] (weights_out may be weights)."""
    fn = _by_dtype("dadgpt_decode_attention_weights", q.dtype)
    rows = n_seq * n_heads
    po, pq = _ptrs(q.dtype, rows * d_head, (out, q), ("out", "q"))
    pk, pv = _ptrs(q.dtype, rows * max_len * d_head, (k_cache, v_cache), ("k_cache", "v_cache"))
    pw, px = _ptrs(torch.float32, rows * max_len, (weights_out, weights),
                   ("weights_out", "weights"))
    pl, = _ptrs(torch.int32, n_seq, (lens,), ("lens",))
    _same_device((out, weights_out, q, k_cache, v_cache, weights, lens, workspace))
    _check(fn(po, pw, pq, pk, pv, px, pl, n_seq, n_heads, max_len, d_head, scale,
              *_workspace(workspace), _stream_ptr(stream)))


def kv_evict(k_out, v_out, weights_out, kept, lens_out, k, v, weights, lens, n_seq: int,
             n_heads: int, max_len: int, max_out: int, d_head: int, budget: int, sinks: int,
             recent: int, stream=None) -> None:
    """Cuts every (sequence, head) of a bf16 or fp32 cache [n_seq, n_heads, max_len, d_head] back to
    `budget` rows: its first `sinks`, its last `recent`, and between them those of the largest
    weights, in order, into a cache of max_out rows or (k_out is k, v_out is v) in place. kept
    [n_seq, n_heads, budget] int32 receives the rows' former indices (-1 past the end), lens_out
    min(lens, budget) (lens_out may be lens). weights_out from lens_out on is left as it was: set a
    row's weight to 0 when a row is appended there."""
    fn = _by_dtype("dadgpt_kv_evict", k.dtype)
    rows = n_seq * n_heads
    po, pp = _ptrs(k.dtype, rows * max_out * d_head, (k_out, v_out), ("k_out", "v_out"))
    pk, pv = _ptrs(k.dtype, rows * max_len * d_head, (k, v), ("k", "v"))
    pw, = _ptrs(torch.float32, rows * max_out, (weights_out,), ("weights_out",))
    px, = _ptrs(torch.float32, rows * max_len, (weights,), ("weights",))
    pn, = _ptrs(torch.int32, rows * budget, (kept,), ("kept",))
    pm, pl = _ptrs(torch.int32, n_seq, (lens_out, lens), ("lens_out", "lens"))
    _same_device((k_out, v_out, weights_out, kept, lens_out, k, v, weights, lens))
    _check(fn(po, pp, pw, pn, pm, pk, pv, px, pl, n_seq, n_heads, max_len, max_out, d_head, budget,
              sinks, recent, _stream_ptr(stream)))
