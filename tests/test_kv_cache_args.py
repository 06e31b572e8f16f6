"""CPU tests of the bounded caches' C ABI: header and binding agree, every check answers on the host
before any HIP call."""
import ctypes
import os
import re

import pytest

from dadgpt_amd import attention as A
from dadgpt_amd import kv_cache as C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE, STEP = 0x1000000, 0x10000000  # non-null addresses, far apart; no call below gets past its checks


def _ptrs(n):
    return [FAKE + i * STEP for i in range(n)]


def test_header_and_binding_agree():
    text = open(os.path.join(ROOT, "include", "dadgpt", "kv_cache.h")).read()
    declared = set(re.findall(r"^(?:int|size_t) (dadgpt_\w+)\s*\(", text, re.M))
    assert declared == set(C.CACHE_SYMBOLS)
    assert all(hasattr(C.lib(), s) for s in C.CACHE_SYMBOLS)


def test_blocks():
    for block in C.KV8_BLOCKS:
        for L in (1, 15, 16, 17, 127, 128, 129, 1024):
            assert C.kv8_blocks(L, block) == C.lib().dadgpt_kv8_blocks(L, block)
    assert [C.kv8_blocks(L, 32) for L in (1, 32, 33, 1024)] == [1, 1, 2, 32]
    for L, block in ((0, 32), (10, 0), (10, 8), (10, 48), (10, 256)):
        with pytest.raises(ValueError):
            C.kv8_blocks(L, block)
        assert C.lib().dadgpt_kv8_blocks(L, block) == 0


def _st(batch=1 << 16, head=64, row=768):
    return A.HeadStrides(batch, head, row)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_append_validation(name):
    f = getattr(C.lib(), "dadgpt_kv8_append_" + name)

    def call(ptrs=None, ks=None, vs=None, lens=FAKE + 6 * STEP, counts=None, n=4, h=2, rows=3, L=100,
             d=64, block=32):
        return f(*(ptrs or _ptrs(6)), ctypes.byref(ks or _st()), ctypes.byref(vs or _st()), lens, counts, n, h, rows, L, d, block,
                 None)

    for i in range(6):
        bad = _ptrs(6)
        bad[i] = None
        assert call(bad) == 1 and "null" in A.last_error()
        bad[i] = FAKE + i * STEP + 2
        assert call(bad) == 1 and "aligned" in A.last_error()
    assert call(lens=None) == 1 and call(lens=FAKE + 2) == 1 and call(counts=FAKE + 2) == 1
    assert call(d=48) == 2
    for kw in ({"n": 0}, {"h": 0}, {"rows": 0}, {"rows": -1}, {"L": 0}, {"block": 8}, {"block": 48},
               {"block": 0}):
        assert call(**kw) == 1, kw
    for kw in ({"batch": -8}, {"head": 4}, {"row": 12}, {"row": 1 << 41}):
        assert call(ks=_st(**kw)) == 1 and "strides of k" in A.last_error()
        assert call(vs=_st(**kw)) == 1 and "strides of v" in A.last_error()
    assert f(*_ptrs(6), None, ctypes.byref(_st()), FAKE, None, 4, 2, 3, 100, 64, 32, None) == 1
    assert call(n=65536) == 1 and "launch limits" in A.last_error()
    assert call(rows=16 * 65535 + 2, block=16) == 1 and "launch limits" in A.last_error()
    same = _ptrs(6)
    same[1] = same[0]
    assert call(same) == 1 and "k_cache overlaps v_cache" in A.last_error()
    same = _ptrs(6)
    same[3] = same[0] + 4 * 2 * 100 * 64 - 4
    assert call(same) == 1 and "k_cache overlaps v_scale" in A.last_error()
    assert call(lens=FAKE) == 1 and "k_cache overlaps lens" in A.last_error()


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_kv8_decode_validation(name):
    f = getattr(C.lib(), "dadgpt_decode_attention_kv8_" + name)

    def call(ptrs=None, n=4, h=2, L=5000, d=64, block=32, scale=0.125, window=0, sinks=0, ws=None,
             wsb=0):
        return f(*(ptrs or _ptrs(7)), n, h, L, d, block, scale, window, sinks, ws, wsb, None)

    for i in range(7):
        bad = _ptrs(7)
        bad[i] = None
        assert call(bad) == 1 and "null" in A.last_error()
    assert call(d=16) == 2 and call(block=24) == 1 and call(n=0) == 1
    assert call(scale=float("nan")) == 1
    assert call(sinks=3) == 1 and "without a window" in A.last_error()
    assert call(window=-1) == 1 and call(window=5, sinks=-1) == 1 and call(window=5, sinks=1025) == 1
    need = C.decode_kv8_workspace_bytes(4, 2, 5000, 64)
    assert need > 0
    assert call() == 4 and call(ws=FAKE, wsb=need - 1) == 4 and call(ws=FAKE + 8, wsb=need) == 1
    # a window needs what its own keys need
    less = C.decode_kv8_workspace_bytes(4, 2, 1104, 64)
    assert 0 < less < need and call(window=1100, sinks=4, ws=FAKE, wsb=less - 1) == 4
    assert C.decode_kv8_workspace_bytes(4, 2, 64, 64) == 0
    for bad in ((0, 2, 2000, 64), (4, 0, 2000, 64), (4, 2, 0, 64), (4, 2, 2000, 48)):
        assert C.decode_kv8_workspace_bytes(*bad) == 0
        assert C.decode_weights_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_weights_decode_validation(name):
    f = getattr(C.lib(), "dadgpt_decode_attention_weights_" + name)

    def call(ptrs=None, n=4, h=2, L=2000, d=64, scale=0.125, ws=None, wsb=0):
        return f(*(ptrs or _ptrs(7)), n, h, L, d, scale, ws, wsb, None)

    for i in range(7):
        bad = _ptrs(7)
        bad[i] = None
        assert call(bad) == 1 and "null" in A.last_error()
    assert call(d=16) == 2 and call(L=0) == 1 and call(scale=float("inf")) == 1
    part = _ptrs(7)
    part[1] = part[5] + 4  # weights_out a word into weights
    assert call(part) == 1 and "weights_out overlaps weights" in A.last_error()
    need = C.decode_weights_workspace_bytes(4, 2, 2000, 64)
    assert need > 0
    assert call() == 4 and call(ws=FAKE, wsb=need - 1) == 4


@pytest.mark.parametrize("name,size", [("bf16", 2), ("f32", 4)])
def test_evict_validation(name, size):
    f = getattr(C.lib(), "dadgpt_kv_evict_" + name)

    def call(ptrs=None, n=4, h=2, L=200, out=64, d=64, budget=64, sinks=4, recent=16):
        return f(*(ptrs or _ptrs(9)), n, h, L, out, d, budget, sinks, recent, None)

    for i in range(9):
        bad = _ptrs(9)
        bad[i] = None
        assert call(bad) == 1 and "null" in A.last_error()
        bad[i] = FAKE + i * STEP + 2
        assert call(bad) == 1 and "aligned" in A.last_error()
    assert call(d=16) == 2
    for kw in ({"budget": 0}, {"sinks": -1}, {"recent": -1}, {"sinks": 60}, {"out": 63}, {"n": 0},
               {"L": 0}, {"n": 1 << 21, "h": 2}, {"sinks": 2 ** 31 - 1, "recent": 2 ** 31 - 1}):
        assert call(**kw) == 1, kw
    # a budget far past any cache: row numbers are counted in 32 bits in steps of a workgroup
    assert call(budget=2 ** 31 - 1, out=200) == 1 and "launch limits" in A.last_error()
    # in place: both tensors, and caches of one length
    p = _ptrs(9)
    p[0] = p[5]
    assert call(p, out=200) == 1 and "in place" in A.last_error()
    p[1] = p[6]
    assert call(p, out=64) == 1 and "in place" in A.last_error()
    w = _ptrs(9)
    w[2] = w[7]
    assert call(w, out=64) == 1 and "max_out = max_len" in A.last_error()
    # any other overlap
    for a, b, text in ((0, 5, "k_out overlaps k"), (1, 5, "v_out overlaps k"),
                       (0, 1, "k_out overlaps v_out"), (3, 8, "kept overlaps lens"),
                       (2, 6, "weights_out overlaps v"), (4, 7, "lens_out overlaps weights")):
        p = _ptrs(9)
        p[a] = p[b] + 16
        if b == 8:
            p[a] = p[b]
        assert call(p) == 1 and text in A.last_error(), (text, A.last_error())
