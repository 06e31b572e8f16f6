"""GPU test of the windowed calls at their limits: the longest sequence with the most sinks."""
import pytest
import torch

from dadgpt_amd import attention as A
from tests import window_ref as R


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [32, 64])
def test_the_longest_sequence_with_the_most_sinks(gpu, dtype, D):
    """524,288 tokens, 1,024 sinks, gradients in the first 1,300 and the last 300 rows only: what those
    rows give is what they give in two short sequences, of the first rows, and of the sinks and the
    last rows. The rows between add exact zeros to the sink keys' gradients."""
    S, window, sinks, first, last, scale = A.WINDOW_MAX_SEQ, 33, A.WINDOW_MAX_SINKS, 1300, 300, D ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, g = (torch.randn((1, S, D), generator=gen, device="cuda").to(dtype) for _ in range(4))
    g[:, first:S - last] = 0
    out, dq, dk, dv = (torch.full_like(q, float("nan")) for _ in range(4))
    lse, delta = (torch.empty((1, S), device="cuda") for _ in range(2))
    ws = A.window_workspace(1, S, D, window, sinks)
    ws.fill_(0xFF)
    f, b = ((A.flash_attention_window_forward_bf16, A.flash_attention_window_backward_bf16)
            if dtype == torch.bfloat16 else
            (A.flash_attention_window_forward, A.flash_attention_window_backward))
    f(out, lse, q, k, v, 1, S, D, scale, window, sinks)
    b(dq, dk, dv, delta, g, out, lse, q, k, v, 1, S, D, scale, window, sinks, ws)
    got = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    m = last + 100                                  # enough rows before the last for their window
    a = R.attention(*(x[:, :first + 100] for x in (q, k, v, g)), scale, window, sinks, dtype)
    tail = [torch.cat((x[:, :sinks], x[:, S - m:]), 1) for x in (q, k, v, g)]
    tail[3][:, :sinks] = 0
    z = R.attention(*tail, scale, window, sinks, dtype)
    for ref, rows, mine in ((a, slice(0, first), slice(0, first)),
                            (z, slice(-last, None), slice(S - last, None))):
        R.assert_within({n: got[n][:, mine] for n in ("out", "lse", "dq")},
                        {n: tuple(t[:, rows] for t in ref[n]) for n in ("out", "lse", "dq")})
    R.assert_within({n: got[n][:, S - last:] for n in ("dk", "dv")},
                    {n: tuple(t[:, -last:] for t in z[n]) for n in ("dk", "dv")})
    R.assert_within({n: got[n][:, sinks:first - window] for n in ("dk", "dv")},
                    {n: tuple(t[:, sinks:first - window] for t in a[n]) for n in ("dk", "dv")})
    for n in ("dk", "dv"):
        y, e = (a[n][i][:, :sinks] + z[n][i][:, :sinks] for i in range(2))
        assert ((got[n][:, :sinks].double() - y).abs() <= e).all(), n
    # keys that none but rows without a gradient see
    assert (dk[:, first + 100:S - m] == 0).all() and (dv[:, first + 100:S - m] == 0).all()
    assert (dq[:, first:S - last] == 0).all() and torch.isfinite(lse).all()
