"""CPU tests of what the windowed backward, the 8-bit and the weighted decode refuse because two of
a call's buffers share memory or the workspace is not aligned. Every check answers on the host before
any HIP call: a call whose buffers are apart gets as far as a workspace that is missing (status 4)."""
import ctypes

import pytest

from dadgpt_amd import attention as A
from dadgpt_amd import kv_cache as C

FAKE, STEP = 0x1000000, 0x10000000  # non-null addresses, far apart


def _ptrs(n):
    return [FAKE + i * STEP for i in range(n)]


# ------------------------------------------------------------- windowed backward

BWD = ("dq", "dk", "dv", "delta", "dout", "out", "lse", "q", "k", "v")
BH, S, D = 4, 2000, 64


def _bwd(name, ptrs, ws=None, wsb=0):
    return getattr(A.lib(), "dadgpt_flash_attention_window_" + name)(
        *ptrs, BH, S, D, 0.125, 16, 2, ws, wsb, None)


@pytest.mark.parametrize("name,size", [("backward", 4), ("backward_bf16", 2)])
def test_window_backward_refuses_outputs_over_each_other(name, size):
    nbytes = {n: BH * S * D * size for n in BWD}
    nbytes["delta"] = nbytes["lse"] = BH * S * 4
    need = A.window_workspace_bytes(BH, S, D, 16, 2)
    assert _bwd(name, _ptrs(10)) == 4  # apart: the missing workspace
    pairs = [("dq", "dk"), ("dq", "dv"), ("dk", "dv")]
    pairs += [(g, n) for g in ("dq", "dk", "dv") for n in ("delta", "lse")]
    pairs += [("delta", n) for n in ("dout", "out", "lse", "q", "k", "v")]
    for a, b in pairs:
        # from the same address, with the last bytes shared, with the first bytes shared
        for at in (0, nbytes[b] - 16, 16 - nbytes[a]):
            p = _ptrs(10)
            p[BWD.index(a)] = p[BWD.index(b)] + at
            assert _bwd(name, p) == 1, (a, b, at)
            assert f"{a} overlaps {b}" in A.last_error(), (a, b, at, A.last_error())
        for at in (nbytes[b], -nbytes[a]):  # side by side
            p = _ptrs(10)
            p[BWD.index(a)] = p[BWD.index(b)] + at
            assert _bwd(name, p) == 4, (a, b, at, A.last_error())
    for n in BWD:
        p = _ptrs(10)
        assert _bwd(name, p, p[BWD.index(n)] + nbytes[n] - 16, need) == 1
        assert f"{n} overlaps the workspace" in A.last_error()


def _strides(*rows):
    return (A.HeadStrides * len(rows))(*[A.HeadStrides(*r) for r in rows])


def test_window_backward_in_rows_of_one_buffer():
    """Gradients side by side in one projection's rows are apart, a column or a head into each other
    they are not."""
    B, H = 2, 12
    d = H * D
    tok = A.lib().dadgpt_flash_attention_window_backward_bf16_tokens
    strided = A.lib().dadgpt_flash_attention_window_backward_bf16_strided

    def both(dq, dk, dv, ld):
        p = _ptrs(10)
        p[:3] = dq, dk, dv
        a = tok(p[0], p[1], p[2], ld, p[3], p[4], p[5], d, p[6], p[7], p[8], p[9], 3 * d, B, H, S, D,
                0.125, 16, 2, None, 0, None)
        text = A.last_error()
        g, x, o = (ld * S, D, ld), (3 * d * S, D, 3 * d), (d * S, D, d)
        b = strided(*p, B, H, S, D, 0.125, 16, 2, _strides(x, x, x, o, o, g, g, g), None, 0, None)
        assert a == b and text.split(": ")[1:] == A.last_error().split(": ")[1:]
        return a, text

    base = FAKE
    assert both(base, base + 2 * d, base + 4 * d, 3 * d)[0] == 4
    assert both(base + 4 * d, base, base + 2 * d, 3 * d)[0] == 4
    assert both(base, base + 2 * d, base + 4 * d, 3 * d + 64)[0] == 4
    for dq, dk, dv, text in (
            (base, base, base + 2 * d, "dq overlaps dk"),
            (base, base + 2 * d, base + 2 * d, "dk overlaps dv"),
            (base, base + 2 * d - 16, base + 4 * d, "dq overlaps dk"),
            (base, base + 2 * d, base + 4 * d + 16, "dq overlaps dv"),  # into the next row
            (base + 6 * d * 100, base + 2 * d, base + 6 * d * 1500 + 128, "dq overlaps dv"),
            (base, base + 2 * d, base + 4 * d - 2 * D, "dk overlaps dv")):
        status, got = both(dq, dk, dv, 3 * d)
        assert status == 1 and text in got, (text, got)
    # one gradient in the gaps of another, a row further down
    assert both(base, base + 6 * d + 2 * d, base + 4 * d, 3 * d)[0] == 4
    # head-major buffers: whole slices, side by side and one row into each other
    h = (H * S * D, S * D, D)
    n = B * H * S * D * 2
    p = _ptrs(10)
    p[1], p[2] = p[0] + n, p[0] - n
    st = _strides(h, h, h, h, h, h, h, h)
    assert strided(*p, B, H, S, D, 0.125, 16, 2, st, None, 0, None) == 4
    p[1] = p[0] + n - 2 * D
    assert strided(*p, B, H, S, D, 0.125, 16, 2, st, None, 0, None) == 1
    assert "dq overlaps dk" in A.last_error()


# ------------------------------------------------------------- caches

@pytest.mark.parametrize("name,size", [("bf16", 2), ("f32", 4)])
def test_weights_decode_refuses_outputs_over_other_buffers(name, size):
    f = getattr(C.lib(), "dadgpt_decode_attention_weights_" + name)
    n, h, L, d = 4, 2, 2000, 64
    names = ("out", "weights_out", "q", "k_cache", "v_cache", "weights", "lens")
    rows, cache, w = n * h * d * size, n * h * L * d * size, n * h * L * 4
    nbytes = dict(zip(names, (rows, w, rows, cache, cache, w, 4 * n)))
    need = C.decode_weights_workspace_bytes(n, h, L, d)

    def call(p, ws=None, wsb=0):
        return f(*p, n, h, L, d, 0.125, ws, wsb, None)

    assert call(_ptrs(7)) == 4
    for a, others in (("out", names[1:]), ("weights_out", names[2:])):
        for b in others:
            for at in (16, nbytes[b] - 16, 16 - nbytes[a]):
                if at >= nbytes[b]:
                    continue
                p = _ptrs(7)
                p[names.index(a)] = p[names.index(b)] + at
                assert call(p) == 1, (a, b, at)
                assert f"{a} overlaps {b}" in A.last_error(), (a, b, at, A.last_error())
            for at in ((nbytes[b] + 15) // 16 * 16, -nbytes[a]):
                p = _ptrs(7)
                p[names.index(a)] = p[names.index(b)] + at
                assert call(p) == 4, (a, b, at, A.last_error())
    for b in ("k_cache", "weights", "lens", "weights_out"):
        p = _ptrs(7)
        p[0] = p[names.index(b)]
        assert call(p) == 1 and f"out overlaps {b}" in A.last_error()
    p = _ptrs(7)
    p[1] = p[5]  # in place
    assert call(p) == 4
    for b in names:
        p = _ptrs(7)
        assert call(p, p[names.index(b)] - need + 16, need) == 1
        assert f"the workspace overlaps {b}" in A.last_error()


@pytest.mark.parametrize("name,size", [("bf16", 2), ("f32", 4)])
def test_kv8_decode_refuses_its_output_and_workspace_over_inputs(name, size):
    f = getattr(C.lib(), "dadgpt_decode_attention_kv8_" + name)
    n, h, L, d, block = 4, 2, 5000, 64, 32
    names = ("out", "q", "k_cache", "v_cache", "k_scale", "v_scale", "lens")
    rows, cache, scales = n * h * d * size, n * h * L * d, n * h * 157 * 4
    nbytes = dict(zip(names, (rows, rows, cache, cache, scales, scales, 4 * n)))
    need = C.decode_kv8_workspace_bytes(n, h, L, d)

    def call(p, ws=None, wsb=0, window=0):
        return f(*p, n, h, L, d, block, 0.125, window, 0, ws, wsb, None)

    assert call(_ptrs(7)) == 4
    for b in names[1:]:
        for at in (16, nbytes[b] - 16, 16 - rows):
            if at >= nbytes[b]:
                continue
            p = _ptrs(7)
            p[0] = p[names.index(b)] + at
            assert call(p) == 1 and f"out overlaps {b}" in A.last_error(), (b, at, A.last_error())
        p = _ptrs(7)
        p[0] = p[names.index(b)] + (nbytes[b] + 15) // 16 * 16
        assert call(p) == 4
    for b in names:
        p = _ptrs(7)
        assert call(p, p[names.index(b)] - need + 16, need) == 1
        assert f"the workspace overlaps {b}" in A.last_error()


@pytest.mark.parametrize("name,size", [("bf16", 2), ("f32", 4)])
def test_append_refuses_new_rows_that_lie_in_the_cache(name, size):
    f = getattr(C.lib(), "dadgpt_kv8_append_" + name)
    n, h, rows, L, d, block = 4, 2, 3, 100, 64, 32
    st = A.HeadStrides(1 << 12, 64, 768)
    extent = ((n - 1) * (1 << 12) + (h - 1) * 64 + (rows - 1) * 768 + d) * size
    cache, scales = n * h * L * d, n * h * 4 * 4
    names = ("k_cache", "v_cache", "k_scale", "v_scale", "k", "v")
    nbytes = dict(zip(names, (cache, cache, scales, scales, extent, extent)))
    for x in ("k", "v"):
        for c in names[:4]:
            for at in (0, nbytes[c] - 16, 16 - extent):
                p = _ptrs(6)
                p[names.index(x)] = p[names.index(c)] + at
                got = f(*p, ctypes.byref(st), ctypes.byref(st), FAKE + 6 * STEP, None, n, h, rows, L, d,
                        block, None)
                assert got == 1 and f"{c} overlaps {x}" in A.last_error(), (x, c, at)


def test_window_strided_refuses_outputs_whose_own_rows_overlap():
    """An output of a broadcast view (expand: stride 0) or of rows laid into each other would be
    written by several workgroups; inputs may be broadcast. A call with nothing else wrong gets as far
    as its workspace's alignment."""
    B, H = 2, 12
    need = A.window_workspace_bytes(B * H, S, D, 16, 2)
    fwd = A.lib().dadgpt_flash_attention_window_forward_bf16_strided
    bwd = A.lib().dadgpt_flash_attention_window_backward_bf16_strided
    ok = (H * S * D, S * D, D)
    names = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")

    def call(**other):
        st = _strides(*(other.get(n, ok) for n in names))
        assert bwd(*_ptrs(10), B, H, S, D, 0.125, 16, 2, st, FAKE + 20 * STEP + 8, need, None) == 1
        return A.last_error()

    assert "not 16-byte aligned" in call()
    shared = ((H * S * D, 0, D), (0, S * D, D), (S * D, S * D, D), (8, S * D, D),
              (H * S * D, D - 8, H * D), (S * H * D, D, H * D - 8), (S * D // 2, S * D, D))
    for name in ("dq", "dk", "dv"):
        for bad in shared:
            assert f"rows of {name} overlap" in call(**{name: bad}), (name, bad)
        # head-major, token-major, tokens before batches, heads outermost, gaps
        for good in ((S * H * D, D, H * D), (H * D, D, B * H * D), (S * D, B * S * D, D),
                     (H * S * 128, S * 128, 128), (3 * S * H * D + 64, D, 3 * H * D)):
            assert "not 16-byte aligned" in call(**{name: good}), (name, good, A.last_error())
    for name in ("q", "k", "v", "out", "dout"):
        assert "not 16-byte aligned" in call(**{name: (H * S * D, 0, D)}), name
    for bad in shared:
        st = _strides(ok, ok, ok, bad)
        assert fwd(*_ptrs(5), B, H, S, D, 0.125, 16, 2, st, None) == 1
        assert "rows of out overlap" in A.last_error()
