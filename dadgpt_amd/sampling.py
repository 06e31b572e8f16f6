"""Python mirror of include/dadgpt/sampling.h: picking tokens from logits by given random numbers over
libdadgpt_attn.so, every row with its own temperature, top-k, top-p and min-p.

The reference picks on the host, a row at a time (``src/generate.cpp:16-92``). As in ``attention``, the
buffers are torch tensors, work runs on torch's current stream, every call raises on failure and
there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import attention as _attn
from .attention import _check, _ptrs, _same_device, _stream_ptr

# Symbols declared in include/dadgpt/sampling.h.
SAMPLING_SYMBOLS = ("dadgpt_sample_bf16", "dadgpt_sample_f32")

# The largest vocabulary (the header's DADGPT_SAMPLE_MAX_VOCAB).
MAX_VOCAB = 1 << 19

_lib = None


def lib():
    """The loaded library with this header's signatures."""
    global _lib
    if _lib is not None:
        return _lib
    L = _attn.lib()
    vp, i, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    for name in SAMPLING_SYMBOLS:
        getattr(L, name).argtypes = [vp, vp, vp, i64, i, i] + [vp] * 6
        getattr(L, name).restype = i
    _lib = L
    return L


def sample(tokens, probs, logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None,
           stream=None) -> None:
    """A token for each row of logits [rows, vocab] (bf16 or fp32, a view with contiguous rows) into
    tokens (int32 [rows]), and into probs (float32 [rows], or None) the probability that it was drawn
    with. Per row: weights exp((logit - largest) / temperature) (0: the first largest logit);
    of the descending order the first top_k (0: all), of these the fewest with top_p of their
    weight (1: all), of these the ones of at least min_p times the largest weight; and the first token
    of the vocabulary at which the sum of what stayed exceeds uniforms (in [0, 1)) times the whole.
    Settings are device arrays [rows] (float32, top_k int32), None: 1, 0, 1, 0."""
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, vocab]")
    if not logits.is_cuda:
        raise ValueError("logits must be a device tensor")
    rows, vocab = logits.shape
    ld, one = logits.stride()
    if (one != 1 and vocab > 1) or (rows > 1 and ld < vocab):
        raise ValueError(f"logits must have contiguous rows, got strides {logits.stride()}")
    if rows == 1:
        ld = vocab
    if logits.dtype is torch.float32:
        fn = lib().dadgpt_sample_f32
    elif logits.dtype is torch.bfloat16:
        fn = lib().dadgpt_sample_bf16
    else:
        raise TypeError(f"sample: logits must be bfloat16 or float32, got {logits.dtype}")
    pt, pk = _ptrs(torch.int32, rows, (tokens, top_k), ("tokens", "top_k"))
    pp, pu, pm, pq, pn = _ptrs(torch.float32, rows, (probs, uniforms, temperature, top_p, min_p),
                               ("probs", "uniforms", "temperature", "top_p", "min_p"))
    _same_device((tokens, probs, logits, uniforms, temperature, top_k, top_p, min_p))
    _check(fn(pt, pp, logits.data_ptr(), ld, rows, vocab, pu, pm, pk, pq, pn, _stream_ptr(stream)))
