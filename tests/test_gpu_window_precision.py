"""How exact the fp32 windowed kernels are, as a norm: the element bounds of window_ref add every
rounding up with one sign, which on long sequences would pass a kernel that dropped the third bf16
plane of its operands.

u = 2^-24. Inputs N(0, 1), scale D^-1/2: scaled scores have size 1. A product over n is 6 n / 16
matrix steps (six bf16 products for an fp32 one), a rounding each, taken all of one sign: 6 D / 16 u
= 24 u at D = 64 for a score (in units of the exponent) and for dP. With the exponent's own rounding
(an argument of size 8: 8 u) and the exponential's (4 u) a probability is off by 36 u. A relative
error that is independent from key to key passes through a sum over keys as it is, and with the sum's
own 6 n / 16 u, n <= 64 visible keys:
  out            36 u + 24 u                      <= 64 u = 2^-18
  dv             the same                         <= 64 u
  dq, dk         36 u (P) + 24 u (dP) + 4 u (delta and the difference) + 24 u <= 96 u
A sink key's sums run over pieces of up to 1024 rows in one chain, which add: + 6 * 1024 / 16 u = 384 u
(and one addition for each piece, of which there are fewer than 64).
With two planes an operand is off by up to 2^-17 of itself, 2^-17 / 3^1/2 = 2^-17.8 = 74 u in the
mean: a score by 2^1/2 of that, and out by (2 + 1)^1/2 74 u = 128 u, dq and dk by more. The CPU test
shows that by computing with such operands in float64."""
import pytest
import torch

from dadgpt_amd import attention as A
from tests import window_ref as R

U = 2.0 ** -24
LIMIT = {"out": 64 * U, "dv": 64 * U, "dq": 96 * U, "dk": 96 * U}
SINK_MORE = (384 + 64) * U


def _planes(x, n):
    """x as the sum of n bf16 values, each the rounding of what the ones before leave."""
    x = x.double()
    y, rest = torch.zeros_like(x), x
    for _ in range(n):
        part = rest.float().bfloat16().double()
        y, rest = y + part, rest - part
    return y


def _exact(q, k, v, g, scale, window, sinks, cut=lambda x: x.double()):
    """float64, with every operand of a product (P and dS too) cut down by `cut`."""
    see = R.visible(q.shape[1], window, sinks, q.device)
    qc, kc, vc, gc = (cut(x) for x in (q, k, v, g))

    def t(x):
        return x.transpose(-1, -2).contiguous()

    s = (torch.bmm(qc, t(kc)) * scale).masked_fill(~see, float("-inf"))
    p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
    out = torch.bmm(cut(p), vc)
    delta = (g.double() * out).sum(-1, keepdim=True)
    ds = p * (torch.bmm(gc, t(vc)) - delta)
    return {"out": out, "dq": torch.bmm(cut(ds), kc) * scale, "dk": torch.bmm(t(cut(ds)), qc) * scale,
            "dv": torch.bmm(t(cut(p)), gc)}


def _rel(x, y):
    return ((x - y).norm() / y.norm()).item()


def _check(got, want, sinks, what):
    """Rows of sink keys apart from the others."""
    for name, y in want.items():
        x = got[name].double()
        cut = sinks if name in ("dk", "dv") else 0
        assert _rel(x[:, cut:], y[:, cut:]) <= LIMIT[name], (what, name, _rel(x[:, cut:], y[:, cut:]) / U)
        if cut:
            r = _rel(x[:, :cut], y[:, :cut])
            assert r <= LIMIT[name] + SINK_MORE, (what, name, "sinks", r / U)


@pytest.mark.parametrize("S,D,window,sinks", [(500, 64, 60, 4), (300, 32, 40, 0)])
def test_two_planes_are_outside_the_limits(S, D, window, sinks):
    gen = torch.Generator().manual_seed(S)
    x = [torch.randn((2, S, D), generator=gen) for _ in range(4)]
    want = _exact(*x, D ** -0.5, window, sinks)
    three = _exact(*x, D ** -0.5, window, sinks, lambda t: _planes(t, 3))
    two = _exact(*x, D ** -0.5, window, sinks, lambda t: _planes(t, 2))
    _check(three, want, sinks, "three planes")
    for name, y in want.items():
        cut = sinks if name in ("dk", "dv") else 0
        assert _rel(two[name][:, cut:], y[:, cut:]) > LIMIT[name], name


@pytest.mark.gpu
@pytest.mark.parametrize("BH,S,D,window,sinks", [
    (3, 500, 64, 60, 4), (60, 500, 64, 60, 4), (200, 500, 64, 60, 0), (3, 500, 32, 40, 4),
    (200, 700, 32, 40, 4), (3, 3000, 64, 60, 4), (24, 3000, 32, 60, 40), (2, 6500, 64, 60, 4),
])
def test_window_f32_keeps_three_planes(gpu, BH, S, D, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(S + BH)
    q, k, v, g = (torch.randn((BH, S, D), generator=gen, device="cuda") for _ in range(4))
    scale = D ** -0.5
    out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse, delta = (torch.empty((BH, S), device="cuda") for _ in range(2))
    ws = A.window_workspace(BH, S, D, window, sinks)
    A.flash_attention_window_forward(out, lse, q, k, v, BH, S, D, scale, window, sinks)
    A.flash_attention_window_backward(dq, dk, dv, delta, g, out, lse, q, k, v, BH, S, D, scale, window,
                                      sinks, ws)
    pick = slice(0, 2)
    want = _exact(q[pick], k[pick], v[pick], g[pick], scale, window, sinks)
    got = {"out": out[pick], "dq": dq[pick], "dk": dk[pick], "dv": dv[pick]}
    _check(got, want, sinks, (BH, S, D, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("BH,S,D,window,sinks,bad", [
    (2, 300, 64, 70, 4, (1, 40, 41, 200, 299)), (2, 129, 32, 20, 0, (0, 128)),
    (200, 500, 64, 100, 3, tuple(range(64, 128))), (3, 600, 32, 33, 1, (31, 32, 63, 599)),
])
def test_window_forward_rows_do_not_depend_on_nan_rows(gpu, dtype, BH, S, D, window, sinks, bad):
    """Query rows of NaN (padding that holds anything) are NaN themselves and change no bit of any
    other row; nor do keys and values of NaN from a row on change the rows of the 128-row blocks
    before it."""
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k, v = (torch.randn((BH, S, D), generator=gen, device="cuda").to(dtype) for _ in range(3))
    f = (A.flash_attention_window_forward_bf16 if dtype == torch.bfloat16
         else A.flash_attention_window_forward)

    def run(q, k, v):
        out, lse = torch.empty_like(q), torch.empty((BH, S), device="cuda")
        f(out, lse, q, k, v, BH, S, D, 0.125, window, sinks)
        return out, lse

    out, lse = run(q, k, v)
    q2 = q.clone()
    q2[BH - 1, list(bad)] = float("nan")
    out2, lse2 = run(q2, k, v)
    hit = torch.zeros((BH, S), dtype=torch.bool, device="cuda")
    hit[BH - 1, list(bad)] = True
    assert out2[hit].isnan().all()
    assert torch.equal(out2[~hit], out[~hit]) and torch.equal(lse2[~hit], lse[~hit])
    end = S // 2 // 128 * 128
    k2, v2 = k.clone(), v.clone()
    k2[:, end:], v2[:, end:] = float("nan"), float("nan")
    out2, lse2 = run(q, k2, v2)
    assert torch.equal(out2[:, :end], out[:, :end]) and torch.equal(lse2[:, :end], lse[:, :end])
