"""float64 reference of sliding-window attention with sinks, with first-order error bounds of the
kernels' arithmetic: what each output may be off by, element by element.

Query i sees key j iff j <= i and (j > i - window or j < sinks). The bounds add up, per product,
the rounding of its operands (half a step: bf16 2^-8, and 0 for the fp32 kernels, whose operands
are split exactly to 2^-24 and below, which `acc` covers) and of its fp32 sum (2^-24 of the
absolute terms for each 16-deep step, six steps for one in the fp32 kernels), and, where a
probability or a delta is used, that value's own error.
"""
import torch

BF16_HALF = 2.0 ** -8
F32_HALF = 2.0 ** -24


def visible(S, window, sinks, device):
    i = torch.arange(S, device=device)[:, None]
    j = torch.arange(S, device=device)[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks))


def _t(x):
    return x.transpose(-1, -2).contiguous()


def attention(q, k, v, dout, scale, window, sinks, dtype):
    """{name: (value, bound)} of out, lse, dq, dk, dv for [BH, S, D] inputs."""
    S, D = q.shape[1:]
    q, k, v, g = (x.double() for x in (q, k, v, dout))
    aq, ak, av, ag = q.abs(), k.abs(), v.abs(), g.abs()
    bf16 = dtype == torch.bfloat16
    u = BF16_HALF if bf16 else F32_HALF            # an operand computed in the kernel, and outputs
    steps = (1 if bf16 else 6) * (max(S, D) / 16 + 2) + 2
    acc = steps * F32_HALF                         # a product's fp32 sum
    see = visible(S, window, sinks, q.device)
    c = abs(scale)
    s = (torch.bmm(q, _t(k)) * scale).masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - lse)
    # the exponents: a score's sum, and the roundings of s * scale - m (or - lse) and of exp
    e_s = torch.bmm(aq, _t(ak)) * c * acc + (s.masked_fill(~see, 0).abs() + lse.abs() + 8) * 2.0 ** -22
    e_row = (e_s * see).amax(-1, keepdim=True)
    e_lse = e_row + acc + (lse.abs() + 8) * 2.0 ** -22
    e_p = p * (e_s + e_lse)                        # of a probability, before it is rounded
    out = torch.bmm(p, v)
    pv = torch.bmm(p, av)
    e_out = torch.bmm(e_p, av) + (u + acc) * pv + u * out.abs()
    delta = (g * out).sum(-1, keepdim=True)
    e_delta = ((ag * e_out).sum(-1, keepdim=True) +
               (ag * out.abs()).sum(-1, keepdim=True) * D * F32_HALF)
    dp = torch.bmm(g, _t(v))
    e_dp = torch.bmm(ag, _t(av)) * acc
    x = dp - delta
    ds = p * x
    e_ds = e_p * x.abs() + p * (e_dp + e_delta + (dp.abs() + delta.abs()) * 2.0 ** -22)
    # rounded to a bf16 value and the rest to another (a window of the sequence is the causal kernels',
    # with one)
    e_ds = e_ds + (u * u if bf16 and window < S else u) * ds.abs()

    def grad(a, e_a, b):                            # a b, a computed in the kernel with error e_a
        y = torch.bmm(a, b)
        return y, torch.bmm(e_a, b.abs()) + acc * torch.bmm(a.abs(), b.abs())

    dq, e_dq = grad(ds, e_ds, k)
    dk, e_dk = grad(_t(ds), _t(e_ds), q)
    dv, e_dv = grad(_t(p), _t(e_p + u * p), g)
    r = {"out": (out, e_out), "lse": (lse.squeeze(-1), e_lse.squeeze(-1))}
    for name, y, e, f in (("dq", dq, e_dq, c), ("dk", dk, e_dk, c), ("dv", dv, e_dv, 1.0)):
        y = y * (scale if name != "dv" else 1.0)
        r[name] = (y, e * f + 2 * u * y.abs())
    return r


def assert_within(got, ref, what=""):
    for name, x in got.items():
        y, bound = ref[name]
        off = (x.double() - y).abs()
        assert torch.isfinite(x.double()).all(), (what, name)
        worst = (off / (bound + 1e-30)).max().item()
        assert worst <= 1.0, (what, name, worst, off.max().item())
