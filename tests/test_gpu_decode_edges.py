"""GPU tests of the one-token calls at scores of -inf and at NaN: the windowed decode, the plain one
and the 8-bit one, against float64 over the keys that weigh something."""
import pytest
import torch

from dadgpt_amd import attention as A
from dadgpt_amd import kv_cache as C
from tests import kv_ref as R

BF, F32 = torch.bfloat16, torch.float32


def _randn(shape, seed, dtype=F32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _half(dtype):
    return 2.0 ** -8 if dtype == BF else 2.0 ** -24


def _without(k, v, keep):
    """The rows of k and v that `keep` marks, in float64."""
    return k[:, :, keep].double(), v[:, :, keep].double()


# (rows, window, sinks, first and last key at -inf): whole waves (64 bf16 keys, 32 fp32 ones) and
# whole chunks of eight waves, among the sinks, at the window's start, in the middle and at the end;
# caches of one chunk and of several, the first batch of four chunks whole; windows below, just
# below and at the cache's length
MINUS_INF = [
    (500, 300, 0, 200, 330), (500, 300, 130, 0, 130), (500, 499, 1, 64, 300), (500, 500, 0, 100, 400),
    (500, 2 ** 31 - 1, 3, 0, 200), (3000, 2000, 600, 0, 600), (3000, 2600, 4, 400, 2999),
    (3000, 2999, 0, 1, 1500), (3000, 3000, 0, 0, 2200), (3000, 2000, 0, 1500, 2900),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L,window,sinks,lo,hi", MINUS_INF)
def test_window_decode_of_scores_of_minus_infinity(gpu, dtype, L, window, sinks, lo, hi):
    """Keys whose score is -inf weigh 0, also where a wave, a chunk or a batch of chunks holds
    nothing else: the answer is that of the other visible keys alone."""
    n, H, D, scale = 2, 2, 64, 0.125
    q, k, v = (_randn(s, i, dtype) for i, s in enumerate(((n, H, D), (n, H, L, D), (n, H, L, D))))
    q[..., 0] = 1
    j = torch.arange(L, device="cuda")
    seen = (j >= L - window) | (j < sinks)
    keep = seen & ((j < lo) | (j >= hi))
    m = int(keep.sum())
    assert 0 < m < int(seen.sum())
    ref, bound, _, _ = R.decode(q, *_without(k, v, keep), [m] * n, scale, out_half=_half(dtype))
    k[:, :, lo:hi, 0] = -float("inf")
    out = torch.full_like(q, float("nan"))
    ws = A.decode_workspace(n, H, min(L, window + sinks), D)
    for _ in range(2):  # the second call finds the workspace as the first left it
        A.decode_attention_window(out, q, k, v, _int([L] * n), n, H, L, D, scale, window, sinks, ws)
        assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L,lo,hi", [(500, 0, 200), (250, 60, 249), (3000, 0, 2200), (3000, 700, 2900)])
def test_decode_of_scores_of_minus_infinity(gpu, dtype, L, lo, hi):
    """The same of the decode without a window."""
    n, H, D, scale = 2, 2, 64, 0.125
    q, k, v = (_randn(s, 5 + i, dtype) for i, s in enumerate(((n, H, D), (n, H, L, D), (n, H, L, D))))
    q[..., 0] = 1
    j = torch.arange(L, device="cuda")
    keep = (j < lo) | (j >= hi)
    ref, bound, _, _ = R.decode(q, *_without(k, v, keep), [int(keep.sum())] * n, scale,
                                out_half=_half(dtype))
    k[:, :, lo:hi, 0] = -float("inf")
    out = torch.full_like(q, float("nan"))
    A.decode_attention(out, q, k, v, _int([L] * n), n, H, L, D, scale, A.decode_workspace(n, H, L, D))
    assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L,window,sinks,lo,hi", [
    (500, 0, 0, 0, 256), (500, 400, 4, 160, 448), (6000, 0, 0, 0, 5888), (6000, 0, 0, 1088, 5888),
    (6000, 5000, 128, 0, 4864)])
def test_kv8_decode_of_scores_past_fp32(gpu, dtype, L, window, sinks, lo, hi):
    """Keys whose score lies below fp32's range weigh 0, also where a wave (128 keys), a chunk (1024)
    or a batch of chunks holds nothing else: the answer is that of the other keys alone."""
    n, H, D, block, scale = 2, 2, 64, 32, 0.125
    cache = C.kv8_cache(n, H, L, D, block)
    for i, (codes, scales) in enumerate(((cache[0], cache[2]), (cache[1], cache[3]))):
        codes.copy_((_randn((n, H, L, D), 60 + i) * 16).to(C.KV8_DTYPE))
        scales.fill_(2.0 ** -4)
    cache[0].view(torch.uint8)[..., 0] = 0
    q = _randn((n, H, D), 62, dtype)
    q[..., 0] = 2.0 ** 100
    j = torch.arange(L, device="cuda")
    keep = (j < lo) | (j >= hi)
    if window:
        keep &= (j >= L - window) | (j < sinks)
    row = j // block
    k, v = (R.values(c.view(torch.uint8)) * s.double()[:, :, row, None]
            for c, s in ((cache[0], cache[2]), (cache[1], cache[3])))
    ref, bound, _, _ = R.decode(q, *_without(k, v, keep), [int(keep.sum())] * n, scale,
                                out_half=_half(dtype))
    # codes of -256 in the column of 2^100, blocks of scale 2^40 there: scores of -2^145
    cache[0].view(torch.uint8)[:, :, lo:hi, 0] = 0xF8
    cache[2][:, :, lo // block:hi // block] = 2.0 ** 40
    out = torch.full_like(q, float("nan"))
    ws = C.decode_kv8_workspace(n, H, L, D)
    for _ in range(2):
        C.decode_attention_kv8(out, q, *cache, _int([L] * n), n, H, L, D, block, scale, window, sinks,
                               ws)
        assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L", [200, 2500])
def test_window_decode_of_a_nan_row_does_not_depend_on_the_window(gpu, dtype, L):
    """A visible key of NaN makes its (sequence, head) NaN and no other, for windows below, at and
    past the cache's length."""
    n, H, D = 2, 2, 64
    q, k, v = (_randn(s, 70 + i, dtype) for i, s in enumerate(((n, H, D), (n, H, L, D), (n, H, L, D))))
    k[1, 0, L - 3, 5] = float("nan")
    ws = A.decode_workspace(n, H, L, D)
    for window, sinks in ((64, 0), (L - 1, 0), (L - 2, 2), (L, 0), (L, 7), (2 ** 31 - 1, 1)):
        out = torch.zeros_like(q)
        A.decode_attention_window(out, q, k, v, _int([L, L]), n, H, L, D, 0.125, window, sinks, ws)
        bad = torch.isnan(out)
        assert bad.all(-1).tolist() == bad.any(-1).tolist() == [[False, False], [True, False]], window


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D", [(5, 3, 1, 64), (6, 3, 250, 32), (6, 2, 1024, 64), (5, 2, 5000, 64)])
def test_window_decode_of_the_whole_cache_is_the_plain_decode(gpu, dtype, n, H, L, D):
    q, k, v = (_randn(s, 80 + i, dtype) for i, s in enumerate(((n, H, D), (n, H, L, D), (n, H, L, D))))
    lens = _int([L, 0, 1, L // 2, L + 5, max(L - 1, 0)][:n])
    ws = A.decode_workspace(n, H, L, D)
    want, out = torch.empty_like(q), torch.empty_like(q)
    A.decode_attention(want, q, k, v, lens, n, H, L, D, 0.125, ws)
    for window, sinks in ((L, 0), (max(1, L - 3), 4), (2 ** 31 - 1, 1024)):
        A.decode_attention_window(out, q, k, v, lens, n, H, L, D, 0.125, window, sinks, ws)
        assert torch.equal(out, want), (window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L", [300, 700, 5000])
def test_decode_into_the_query(gpu, dtype, L):
    """The 8-bit decode and the decode with weights may write out over q: the bits of a call that
    does not."""
    n, H, D, block = 5, 3, 64, 32
    q, k, v = (_randn(s, 90 + i, dtype) for i, s in enumerate(((n, H, D), (n, H, L, D), (n, H, L, D))))
    cache = C.kv8_cache(n, H, L, D, block)
    lens = _int([L, 0, 1, L - 1, L // 2])
    C.kv8_append(*cache, k, v, _int([0] * n), None, n, H, L, L, D, block)
    ws8, wsw = C.decode_kv8_workspace(n, H, L, D), C.decode_weights_workspace(n, H, L, D)
    w = torch.zeros((n, H, L), device="cuda")
    for window, sinks in ((0, 0), (L // 2, 3)):
        want, out = torch.empty_like(q), q.clone()
        C.decode_attention_kv8(want, q, *cache, lens, n, H, L, D, block, 0.125, window, sinks, ws8)
        C.decode_attention_kv8(out, out, *cache, lens, n, H, L, D, block, 0.125, window, sinks, ws8)
        assert torch.equal(out, want)
    want, out, w1, w2 = torch.empty_like(q), q.clone(), w.clone(), w.clone()
    C.decode_attention_weights(want, w1, q, k, v, w, lens, n, H, L, D, 0.125, wsw)
    C.decode_attention_weights(out, w2, out, k, v, w, lens, n, H, L, D, 0.125, wsw)
    assert torch.equal(out, want) and torch.equal(w1, w2)
