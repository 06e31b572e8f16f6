"""GPU tests of the windowed strided calls over broadcast inputs: one K/V head shared by all query heads
(a head stride of 0) gives the bits of copies, and an expanded gradient is refused."""
import pytest
import torch

from dadgpt_amd import attention as A

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,S,D,window,sinks", [(2, 3, 300, 64, 70, 3), (16, 12, 700, 64, 90, 4),
                                                  (3, 4, 65, 32, 20, 0)])
def test_a_shared_kv_head(gpu, B, H, S, D, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(S)

    def randn(h):
        return torch.randn((B, h, S, D), generator=gen, device="cuda").to(BF)

    q, g, k1, v1 = randn(H), randn(H), randn(1), randn(1)
    ws = A.window_workspace(B * H, S, D, window, sinks)

    def run(k, v):
        out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
        lse, delta = (torch.empty((B * H, S), device="cuda") for _ in range(2))
        A.flash_attention_window_forward_bf16_strided(out, lse, q, k, v, 0.125, window, sinks)
        A.flash_attention_window_backward_bf16_strided(dq, dk, dv, delta, g, out, lse, q, k, v, 0.125,
                                                       window, sinks, ws)
        return out, lse, dq, dk, dv

    k, v = (x.expand(B, H, S, D) for x in (k1, v1))
    for a, b in zip(run(k, v), run(k.contiguous(), v.contiguous())):
        assert torch.equal(a, b)
    out, lse, dq, dk, dv = run(k, v)
    delta, shared = torch.empty_like(lse), torch.empty_like(k1).expand(B, H, S, D)
    with pytest.raises(A.AttentionError, match="rows of dk overlap"):
        A.flash_attention_window_backward_bf16_strided(dq, shared, dv, delta, g, out, lse, q, k, v,
                                                       0.125, window, sinks, ws)
    with pytest.raises(A.AttentionError, match="rows of out overlap"):
        A.flash_attention_window_forward_bf16_strided(shared, lse, q, k, v, 0.125, window, sinks)
