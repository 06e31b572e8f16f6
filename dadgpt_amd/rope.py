"""Python mirror of include/dadgpt/rope.h: rotary positions over libdadgpt_attn.so, forward and
backward, for q and k wherever the projections keep them.

The reference's positions are learned embeddings (``src/model.cpp:17-56``). As in ``attention``, the
buffers are torch tensors, work runs on torch's current stream, every call raises on failure and
there is no fallback.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import attention as _attn
from .attention import _check, _ptrs, _same_device, _stream_ptr

# Symbols declared in include/dadgpt/rope.h.
ROPE_SYMBOLS = (
    "dadgpt_rope_frequencies",
    "dadgpt_rope_bf16",
    "dadgpt_rope_f32",
    "dadgpt_rope_backward_bf16",
    "dadgpt_rope_backward_f32",
)

SCALINGS = {None: 0, "linear": 1, "base": 2, "parts": 3}

_lib = None


def lib():
    """The loaded library with this header's signatures."""
    global _lib
    if _lib is not None:
        return _lib
    L = _attn.lib()
    vp, i, f, d = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_double
    L.dadgpt_rope_frequencies.argtypes = [vp, i, d, i, d, i, d, d]
    for name in ROPE_SYMBOLS[1:]:
        getattr(L, name).argtypes = [vp] * 5 + [i] * 5 + [vp, i, i, f, vp, vp]
    for name in ROPE_SYMBOLS:
        getattr(L, name).restype = i
    _lib = L
    return L


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling: str | None = None,
                     factor: float = 1.0, original_len: int = 0, slow: float = 1.0,
                     fast: float = 32.0, device="cuda") -> torch.Tensor:
    """The frequencies (radians a position, float64) of the rot_dim / 2 pairs, base^(-2i / rot_dim), for
    contexts `factor` times as long as the trained ones by `scaling`: None, 'linear' (all divided by
    factor), 'base' (a larger base: the slowest pair divided, the fastest kept) or 'parts' (pairs that
    turn `fast` times over original_len tokens kept, those that turn `slow` times divided, a ramp
    between)."""
    host = torch.empty(max(rot_dim // 2, 0), dtype=torch.float64)
    _check(lib().dadgpt_rope_frequencies(host.data_ptr() or None, rot_dim, base, SCALINGS[scaling],
                                         factor, original_len, slow, fast))
    return host.to(device)


def rope_magnitude(factor: float) -> float:
    """The magnitude that goes with 'parts' scaling by `factor`: 1 + ln(factor) / 10."""
    return 1.0 + 0.1 * math.log(factor) if factor > 1.0 else 1.0


_Int64x12 = ctypes.c_int64 * 12
_NONE = (0, 0, 0)


def _heads(t, name, shape, dtype):
    """Address and (batch, head, row) strides of a [B, heads, S, d_head] view with contiguous rows; a
    dimension of one has no stride."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not dtype:
        raise TypeError(f"{name} must be a device tensor of {dtype}")
    s = t.stride()
    if t.shape != shape or s[3] != 1:
        raise ValueError(f"{name} must be a {tuple(shape)} view with contiguous rows, got "
                         f"{tuple(t.shape)} with strides {s}")
    n = shape[0], shape[1], shape[2]
    return t.data_ptr(), (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


_entries = {}


def _call(name, names, q_out, k_out, q, k, freqs, positions, interleaved, magnitude, stream):
    dtype = q.dtype
    fn = _entries.get((name, dtype))
    if fn is None:
        suffix = {torch.bfloat16: "_bf16", torch.float32: "_f32"}.get(dtype)
        if suffix is None:
            raise TypeError(f"{name}: tensors must be bfloat16 or float32, got {dtype}")
        fn = _entries[name, dtype] = getattr(lib(), name + suffix)
    if q.dim() != 4:
        raise ValueError(f"{names[0]} must be a [B, n_heads, S, d_head] view")
    B, H, S, D = shape = q.shape
    pq, sq = _heads(q, names[0], shape, dtype)
    po, so = _heads(q_out, names[2], shape, dtype)
    pk = pko = None
    sk = sko = _NONE
    Hkv = 0
    if k is not None or k_out is not None:
        if k is None or k_out is None or k.dim() != 4:
            raise ValueError(f"{names[1]} and {names[3]} must be [B, n_kv_heads, S, d_head] views "
                             f"together, or both None")
        Hkv = k.shape[1]
        kv = torch.Size((B, Hkv, S, D))
        pk, sk = _heads(k, names[1], kv, dtype)
        pko, sko = _heads(k_out, names[3], kv, dtype)
    pf, = _ptrs(torch.float64, 1, (freqs,), ("freqs",))
    pp, = _ptrs(torch.int32, B * S, (positions,), ("positions",))
    _same_device((q_out, k_out, q, k, freqs, positions))
    strides = _Int64x12(*sq, *sk, *so, *sko)  # four dadgpt_head_strides
    _check(fn(po, pko, pq, pk, strides, B, H, Hkv, S, D, pf, 2 * freqs.numel(), interleaved,
              magnitude, pp, _stream_ptr(stream)))


def rope(q_out, k_out, q, k, freqs, positions=None, interleaved: bool = False,
         magnitude: float = 1.0, stream=None) -> None:
    """Rotates the first 2 * freqs.numel() elements of every head of q [B, n_heads, S, d_head] and k [B,
    n_kv_heads, S, d_head], views with contiguous rows (the heads of a fused projection will do),
    bf16 or fp32, into q_out and k_out; the other elements are copied. Pair i, the elements (i, i +
    freqs.numel()) or (2i, 2i + 1) where interleaved, turns by position * freqs[i] and is multiplied by
    magnitude. positions: int32 [B, S], or None: row s is at position s. In place: q_out is q (k_out is
    k). k and k_out may be None."""
    _call("dadgpt_rope", ("q", "k", "q_out", "k_out"), q_out, k_out, q, k, freqs, positions,
          interleaved, magnitude, stream)


def rope_backward(dq, dk, dq_out, dk_out, freqs, positions=None, interleaved: bool = False,
                  magnitude: float = 1.0, stream=None) -> None:
    """Its gradient: dq and dk of the gradients of q_out and k_out (in place: dq is dq_out)."""
    _call("dadgpt_rope_backward", ("dq_out", "dk_out", "dq", "dk"), dq, dk, dq_out, dk_out, freqs,
          positions, interleaved, magnitude, stream)
