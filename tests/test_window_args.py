"""CPU tests of the windowed calls' refusals: every check answers on the host before any HIP call."""
import pytest

from dadgpt_amd import attention as A

FAKE = 0x1000000  # a non-null address; every call below fails validation before using it
STEP = 0x10000000  # far enough apart that no two tensors overlap


def _ptrs(n):
    return [FAKE + i * STEP for i in range(n)]


def _fwd(name, ptrs=None, BH=4, S=64, D=64, scale=0.125, window=16, sinks=2):
    return getattr(A.lib(), "dadgpt_flash_attention_window_" + name)(
        *(ptrs or _ptrs(5)), BH, S, D, scale, window, sinks, None)


def _bwd(name, ptrs=None, BH=4, S=64, D=64, scale=0.125, window=16, sinks=2, ws=None, wsb=0):
    return getattr(A.lib(), "dadgpt_flash_attention_window_" + name)(
        *(ptrs or _ptrs(10)), BH, S, D, scale, window, sinks, ws, wsb, None)


@pytest.mark.parametrize("call,name,n", [(_fwd, "forward", 5), (_fwd, "forward_bf16", 5),
                                         (_bwd, "backward", 10), (_bwd, "backward_bf16", 10)])
def test_window_validation(call, name, n):
    for i in range(n):
        bad = _ptrs(n)
        bad[i] = None
        assert call(name, bad) == 1
        assert f"pointer argument {i} is null" in A.last_error()
        bad[i] = FAKE + 4
        assert call(name, bad) == 1
        assert "aligned" in A.last_error()
    assert call(name, D=48) == 2
    assert call(name, BH=0) == 1 and call(name, S=0) == 1
    assert call(name, scale=float("nan")) == 1
    for window in (0, -1, -(2 ** 31)):
        assert call(name, window=window) == 1
        assert f"window={window}" in A.last_error()
    for sinks in (-1, A.WINDOW_MAX_SINKS + 1):
        assert call(name, sinks=sinks) == 1
        assert f"sinks={sinks}" in A.last_error()
    assert call(name, BH=1, S=A.WINDOW_MAX_SEQ + 1) == 1
    assert "exceeds" in A.last_error()


@pytest.mark.parametrize("name,size", [("backward", 4), ("backward_bf16", 2)])
def test_window_backward_refuses_gradients_over_inputs(name, size):
    """dq, dk, dv, delta, dout, out, lse, q, k, v: the plain backward takes some of these, the
    windowed one none, also where only the last byte is shared."""
    nbytes = 4 * 64 * 64 * size
    for g, gname in ((0, "dq"), (1, "dk"), (2, "dv")):
        for t, tname in ((4, "dout"), (5, "out"), (7, "q"), (8, "k"), (9, "v")):
            for at in (0, nbytes - 16, 16 - nbytes):
                ptrs = _ptrs(10)
                ptrs[g] = ptrs[t] + at
                assert _bwd(name, ptrs) == 1
                assert f"{gname} overlaps {tname}" in A.last_error()
    need = A.window_workspace_bytes(4, 2000, 64, 16, 2)
    ptrs = _ptrs(10)
    assert _bwd(name, ptrs, S=2000, ws=ptrs[1], wsb=need) == 1
    assert "dk overlaps the workspace" in A.last_error()


@pytest.mark.parametrize("name", ["backward", "backward_bf16"])
def test_window_backward_workspace(name):
    need = A.window_workspace_bytes(4, 2000, 64, 16, 2)
    assert need > 0
    assert _bwd(name, S=2000) == 4
    assert _bwd(name, S=2000, ws=FAKE + 20 * STEP, wsb=need - 1) == 4
    assert "needed" in A.last_error()
    assert _bwd(name, S=2000, ws=FAKE + 20 * STEP + 8, wsb=need) == 1
    # none where every sum is whole: no sinks, or no query past a sink block's window
    assert A.window_workspace_bytes(4, 2000, 64, 16, 0) == 0
    assert A.window_workspace_bytes(4, 128, 64, 16, 2) == 0
    assert A.window_workspace_bytes(4, 2000, 64, 2000, 2) == 0
    # and for what the calls refuse
    for bad in ((0, 2000, 64, 16, 2), (4, 0, 64, 16, 2), (4, 2000, 48, 16, 2), (4, 2000, 64, 0, 2),
                (4, 2000, 64, 16, -1), (4, 2000, 64, 16, 1025), (4, (1 << 19) + 1, 64, 16, 2)):
        assert A.window_workspace_bytes(*bad) == 0


def test_window_workspace_covers_both_types_plans():
    """fp32 partials [BH][piece][2][sink rows in whole 32s][D]. The fp32 backward has pieces of 256
    rows past a 128-key block's window and one for the block itself, or none where the later queries are
    few; the bf16 one pieces of up to 12 64-row tiles."""
    for S in (513, 530, 1024, 5000, 1 << 19):
        for window in (1, 40, 100, 500, 4000):
            for sinks in (1, 32, 33, 700, 1024):
                if window >= S:
                    continue
                end = (128 + window - 2) // 64 * 64 + 64
                far = S - end
                split = far > 384 and (far > end or S > 1024)
                pieces = (far + 255) // 256 if split else 0
                rows = (min(sinks, S) + 31) // 32 * 32
                want = 4 * 3 * (pieces + 1) * 2 * rows * 32 if pieces else 0
                assert A.window_workspace_bytes(3, S, 32, window, sinks) >= want
                # the bf16 plan without a GPU (no compute units known): separate launches, 128 keys
                tiles = max(0, (S + 63) // 64 - ((128 + window - 2) // 64 + 1))
                assert A.window_workspace_bytes(3, S, 32, window, sinks) >= (
                    4 * 3 * ((tiles + 11) // 12) * 2 * rows * 32)


def test_window_strided_validation():
    L = A.lib()
    fwd = L.dadgpt_flash_attention_window_forward_bf16_strided
    bwd = L.dadgpt_flash_attention_window_backward_bf16_strided

    def st(n, **kw):
        return (A.HeadStrides * n)(*[A.HeadStrides(kw.get("batch", 1 << 16), kw.get("head", 64),
                                                   kw.get("row", 768)) for _ in range(n)])

    ok4, ok8 = st(4), st(8)
    p5, p10 = _ptrs(5), _ptrs(10)
    assert fwd(*p5, 2, 12, 64, 64, 0.125, 16, 2, None, None) == 1
    assert fwd(*p5, 2, 12, 64, 48, 0.125, 16, 2, ok4, None) == 2
    assert fwd(*p5, 2, 12, 64, 64, 0.125, 0, 2, ok4, None) == 1
    assert fwd(*p5, 2, 12, 64, 64, 0.125, 16, 2, st(4, row=60), None) == 1
    assert bwd(*p10, 2, 12, 64, 64, 0.125, 16, -2, ok8, None, 0, None) == 1
    assert bwd(*p10, 2, 12, 2000, 64, 0.125, 16, 2, ok8, None, 0, None) == 4
    same = list(p10)
    same[2] = same[9]
    assert bwd(*same, 2, 12, 64, 64, 0.125, 16, 2, ok8, None, 0, None) == 1
    assert "dv overlaps v" in A.last_error()
    tok = L.dadgpt_flash_attention_window_forward_bf16_tokens
    assert tok(p5[0], 760, p5[1], p5[2], p5[3], p5[4], 768, 2, 12, 64, 64, 0.125, 16, 2, None) == 1
    assert "leading dimension 760" in A.last_error()
    tokb = L.dadgpt_flash_attention_window_backward_bf16_tokens
    assert tokb(p10[0], p10[1], p10[2], 700, p10[3], p10[4], p10[5], 768, p10[6], p10[7], p10[8],
                p10[9], 768, 2, 12, 64, 64, 0.125, 16, 2, None, 0, None) == 1


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_window_decode_validation(name):
    f = getattr(A.lib(), "dadgpt_decode_attention_window_" + name)

    def call(ptrs=None, n=4, h=2, L=2000, d=64, scale=0.125, window=1500, sinks=4, ws=None, wsb=0):
        return f(*(ptrs or _ptrs(5)), n, h, L, d, scale, window, sinks, ws, wsb, None)

    assert call(d=48) == 2
    assert call(n=0) == 1 and call(L=0) == 1 and call(scale=float("inf")) == 1
    assert call(window=0) == 1 and call(sinks=-1) == 1 and call(sinks=1025) == 1
    for i in range(5):
        bad = _ptrs(5)
        bad[i] = None
        assert call(bad) == 1
    need = A.decode_workspace_bytes(4, 2, 1504, 64)  # window + sinks keys at most
    assert 0 < need < A.decode_workspace_bytes(4, 2, 2000, 64)
    assert call() == 4
    assert call(ws=FAKE, wsb=need - 1) == 4
    assert A.decode_workspace_bytes(4, 2, 104, 64) == 0


def test_tensors_off_the_current_device_are_refused(monkeypatch):
    """With more than one device, a tensor that is not on the current one would be read on its
    stream: ValueError. None passes; with one device there is nothing to look at."""
    class Fake:
        def __init__(self, device):
            self.device = f"cuda:{device}"
            self._d = device

        def get_device(self):
            return self._d

    monkeypatch.setattr(A, "_devices", 2)
    monkeypatch.setattr(A.torch.cuda, "current_device", lambda: 0)
    A._same_device((Fake(0), None, Fake(0)))
    with pytest.raises(ValueError, match="cuda:1, but the current device is cuda:0"):
        A._same_device((Fake(0), Fake(1)))
    monkeypatch.setattr(A, "_devices", 1)
    A._same_device((Fake(0),))
