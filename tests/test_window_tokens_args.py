"""What the Python wrappers of the token-major windowed calls refuse before the library is called:
tensors that are not bf16 device rows, and buffers shorter than the rows that would be read or written."""
import pytest
import torch

from dadgpt_amd import attention as A

BF = torch.bfloat16
B, H, S, D = 2, 3, 40, 64
d = H * D


def _call(backward, device, **other):
    """A valid call's tensors, some replaced."""
    def new(shape, dtype=BF):
        return torch.zeros(shape, dtype=dtype, device=device)

    t = {"qkv": new((B * S, 3 * d)), "dqkv": new((B * S, 3 * d)), "out": new((B * S, d)),
         "dout": new((B * S, d)), "lse": new((B * H, S), torch.float32),
         "delta": new((B * H, S), torch.float32)}
    for i, x in enumerate("qkv"):
        t[x], t["d" + x] = t["qkv"][:, i * d:], t["dqkv"][:, i * d:]
    t.update(other)
    if not backward:
        return A.flash_attention_window_forward_bf16_tokens(
            t["out"], d, t["lse"], t["q"], t["k"], t["v"], 3 * d, B, H, S, D, 0.125, 16, 2)
    return A.flash_attention_window_backward_bf16_tokens(
        t["dq"], t["dk"], t["dv"], 3 * d, t["delta"], t["dout"], t["out"], d, t["lse"], t["q"], t["k"],
        t["v"], 3 * d, B, H, S, D, 0.125, 16, 2, A.window_workspace(B * H, S, D, 16, 2))


@pytest.mark.parametrize("backward", [False, True])
def test_host_tensors_are_refused(backward):
    with pytest.raises((TypeError, ValueError), match="device tensor"):
        _call(backward, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [False, True])
def test_tensors_that_do_not_fit_are_refused(gpu, backward):
    _call(backward, gpu)
    names = ("q", "k", "v", "out") + (("dout", "dq", "dk", "dv") if backward else ())
    for name in names:
        width = d if name in ("out", "dout") else 3 * d
        short = torch.zeros((B * S - 1) * width + d - 1, dtype=BF, device=gpu)
        with pytest.raises(ValueError, match=f"{name} .*too short"):
            _call(backward, gpu, **{name: short})
        _call(backward, gpu, **{name: torch.zeros((B * S - 1) * width + d, dtype=BF, device=gpu)})
        with pytest.raises(TypeError, match=f"{name} must be"):
            _call(backward, gpu, **{name: torch.zeros((B * S, width), device=gpu)})
    for name in ("lse",) + (("delta",) if backward else ()):
        with pytest.raises(ValueError, match=f"{name} has"):
            _call(backward, gpu, **{name: torch.zeros(B * H * S - 1, device=gpu)})
