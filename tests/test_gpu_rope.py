"""GPU tests of the rotary positions against the definition in 64 bits (serving_ref), with bounds counted
from their roundings, and of the gradient against differences."""
import math

import pytest
import torch

from dadgpt_amd import rope as R
from tests import serving_ref as S

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _randn(shape, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(dtype)


def _views(x, B, Sq, H, Hkv, D, layout):
    """q and k as [B, heads, S, D] views of a buffer."""
    if layout == "tokens":
        x = x.view(B, Sq, -1, D).transpose(1, 2)
    else:
        x = x.view(B, -1, Sq, D)
    return x[:, :H], x[:, H:H + Hkv]


CASES = [  # B, S, H, Hkv, D, rot, interleaved, layout, magnitude
    (1, 1, 1, 1, 32, 8, False, "tokens", 1.0),
    (2, 37, 4, 2, 64, 64, False, "tokens", 1.0),
    (2, 37, 4, 2, 64, 64, True, "heads", 1.25),
    (3, 130, 3, 1, 64, 32, False, "heads", 0.5),
    (1, 1000, 12, 12, 64, 48, True, "tokens", 1.0),
    (1, 333, 8, 8, 32, 24, False, "tokens", 1.0),   # pairs in fours
    (2, 65, 5, 5, 32, 32, True, "heads", 1.0),
    (1, 4097, 12, 4, 64, 40, False, "tokens", 1.1),  # several heads a thread
    (4, 2048, 24, 8, 64, 64, False, "heads", 1.0),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(gpu, case, dtype):
    B, Sq, H, Hkv, D, rot, inter, layout, mag = case
    freqs = R.rope_frequencies(rot, device="cpu")
    total = H + 2 * Hkv if layout == "tokens" else H + Hkv
    x, pos = _randn(B * Sq * total * D, 1, dtype), torch.arange(Sq)
    gx = x.cuda()
    out = torch.full((B * Sq * (H + Hkv) * D,), 7.0, dtype=dtype, device="cuda")
    for back in (False, True):
        q, k = _views(gx, B, Sq, H, Hkv, D, layout)
        qo, ko = _views(out, B, Sq, H, Hkv, D, layout)
        (R.rope_backward if back else R.rope)(qo, ko, q, k, freqs.cuda(), None, inter, mag)
        assert torch.equal(gx.cpu(), x)
        for got, src in zip((qo, ko), _views(x, B, Sq, H, Hkv, D, layout)):
            want = S.rotate(src, pos, freqs, inter, mag, back)
            bound = S.rotate_bound(src, pos, freqs, dtype, inter, mag, back)
            assert ((got.cpu().double() - want).abs() <= bound).all()
            assert torch.equal(got[..., rot:].cpu(), src[..., rot:])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_in_place_and_one_tensor(gpu, dtype):
    B, Sq, H, Hkv, D, rot = 2, 77, 4, 2, 64, 32
    freqs = R.rope_frequencies(rot)
    x = _randn(B * Sq * (H + 2 * Hkv) * D, 3, dtype).cuda()
    q, k = _views(x.clone(), B, Sq, H, Hkv, D, "tokens")
    qo, ko = torch.empty_like(q.contiguous()), torch.empty_like(k.contiguous())
    R.rope(qo, ko, q, k, freqs)
    y = x.clone()
    q2, k2 = _views(y, B, Sq, H, Hkv, D, "tokens")
    R.rope(q2, k2, q2, k2, freqs)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    assert torch.equal(y.view(B, Sq, -1, D)[:, :, H + Hkv:], x.view(B, Sq, -1, D)[:, :, H + Hkv:])
    y = x.clone()
    q3, k3 = _views(y, B, Sq, H, Hkv, D, "tokens")
    R.rope(q3, None, q3, None, freqs)
    assert torch.equal(q3, qo) and torch.equal(k3, k)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_positions(gpu, dtype):
    """Any positions: negative, repeated, and as far as int32 reaches."""
    B, Sq, H, D, rot = 2, 9, 3, 64, 64
    pos = torch.tensor([[0, 5, 5, -3, 1 << 20, 123456789, 2 ** 31 - 1, -2 ** 31, 7],
                        [9, 8, 7, 6, 5, 4, 3, 2, 1]], dtype=torch.int32)
    freqs = R.rope_frequencies(rot, 500000.0, "parts", 8.0, 4096, device="cpu")
    x = _randn((B, H, Sq, D), 5, dtype)
    got = torch.empty_like(x.cuda())
    R.rope(got, None, x.cuda(), None, freqs.cuda(), pos.cuda())
    at = pos.long()[:, None, :]
    want, bound = S.rotate(x, at, freqs), S.rotate_bound(x, at, freqs, dtype)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_by_differences(gpu, interleaved):
    """<g, rope(x + h e) - rope(x - h e)> / 2h is the gradient's element: the map is linear, so the
    difference is exact but for roundings (fp32, h = 1: a few 2^-22 of sums of 16 terms)."""
    D, rot = 32, 16
    freqs = R.rope_frequencies(rot)
    x, g = _randn((1, 1, 3, D), 1, F32).cuda(), _randn((1, 1, 3, D), 2, F32).cuda()
    dx = torch.empty_like(x)
    R.rope_backward(dx, None, g, None, freqs, None, interleaved, 1.3)

    def value(x):
        y = torch.empty_like(x)
        R.rope(y, None, x, None, freqs, None, interleaved, 1.3)
        return (y.double() * g.double()).sum()
    for i in range(0, 3 * D, 5):
        e = torch.zeros_like(x).view(-1)
        e[i] = 1.0
        e = e.view_as(x)
        d = (value(x + e) - value(x - e)) / 2
        assert abs(d - dx.view(-1)[i].double()) <= 3 * D * 2.0 ** -20


def test_special_values_stay_in_their_pair(gpu):
    x = torch.zeros((1, 1, 2, 32))
    x[0, 0, 1, 3], x[0, 0, 1, 20], x[0, 0, 0, 5] = math.nan, math.inf, -math.inf
    y = torch.empty_like(x.cuda())
    R.rope(y, None, x.cuda(), None, R.rope_frequencies(16))
    bad = ~torch.isfinite(y[0, 0].cpu())
    assert bad[1].nonzero().flatten().tolist() == [3, 11, 20]
    assert bad[0].nonzero().flatten().tolist() in ([5, 13], [5])  # (-inf * sin 0 is NaN)


def test_other_stream_and_graph(gpu):
    freqs, x = R.rope_frequencies(64), _randn((2, 4, 50, 64), 1, BF).cuda()
    want, got = torch.empty_like(x), torch.zeros_like(x)
    R.rope(want, None, x, None, freqs)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        R.rope(got, None, x, None, freqs)
    for i in range(3):
        x.copy_(_randn((2, 4, 50, 64), 10 + i, BF))
        R.rope(want, None, x, None, freqs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
