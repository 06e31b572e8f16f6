"""GPU tests of the decode with weights and the eviction at the longest caches (16,776,960 rows, the
launch limit), several of them, so that rows lie past 2^32 bytes."""
import pytest
import torch

from dadgpt_amd import kv_cache as C

L = 65535 * 256


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_weights_decode_of_the_longest_caches(gpu, dtype):
    """Keys of zero weigh the same: weights_out is weights + 1/len, the output the mean of the values,
    which are zero but for one in 2^16 rows. The sums add up len equal terms exactly for 2^24 of them
    or fewer; 1/len, a product and the sum's own rounding are three of 2^-24, taken as eight."""
    n, H, D = 3, 1, 64
    k, v = (torch.zeros((n, H, L, D), dtype=dtype, device="cuda") for _ in range(2))
    v[:, :, ::1 << 16] = 1.0
    q = torch.ones((n, H, D), dtype=dtype, device="cuda")
    lens = [0, 1 << 16, L - 5]
    w = torch.zeros((n, H, L), device="cuda")
    w[:, :, 7] = 0.5
    out, got = torch.full_like(q, float("nan")), torch.full_like(w, float("nan"))
    C.decode_attention_weights(out, got, q, k, v, w, _int(lens), n, H, L, D, 0.125,
                               C.decode_weights_workspace(n, H, L, D))
    for i, end in enumerate(lens):
        want = w[i, 0].double()
        if end:
            want[:end] += 1.0 / end
        assert ((got[i, 0].double() - want).abs() <= want * 8 * 2.0 ** -24).all(), i
        mean = ((end + (1 << 16) - 1) >> 16) / end if end else 0.0
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert ((out[i].double() - mean).abs() <= mean * (half + 8 * 2.0 ** -24)).all(), i


@pytest.mark.gpu
def test_evict_of_the_longest_caches(gpu):
    n, H, D, budget, sinks, recent = 5, 1, 32, 3000, 4, 100
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.zeros((n, H, L, D), dtype=torch.bfloat16, device="cuda")  # 1.07 GB a cache
    k[..., 0] = torch.arange(L, device="cuda") % 251
    k[..., 1] = torch.arange(L, device="cuda") // 251 % 251
    v = -k
    w = torch.rand((n, H, L), generator=gen, device="cuda")
    w[1] = torch.floor(w[1] * 50)                      # many equal weights
    lens = _int([L, L - 3, 2500, 0, L])
    out = [torch.zeros((n, H, budget, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    w_out = torch.zeros((n, H, budget), device="cuda")
    kept, lens_out = torch.empty((n, H, budget), dtype=torch.int32, device="cuda"), _int([9] * n)
    C.kv_evict(*out, w_out, kept, lens_out, k, v, w, lens, n, H, L, budget, D, budget, sinks, recent)
    assert lens_out.tolist() == [budget, budget, 2500, 0, budget]
    for i, end in enumerate(lens.tolist()):
        m = min(end, budget)
        if end > budget:
            mid = torch.sort(w[i, 0, sinks:end - recent], descending=True, stable=True)[1]
            mid = mid[:budget - sinks - recent].sort()[0] + sinks
            want = torch.cat((torch.arange(sinks, device="cuda"), mid,
                              torch.arange(end - recent, end, device="cuda")))
        else:
            want = torch.arange(m, device="cuda")
        assert torch.equal(kept[i, 0, :m].long(), want) and (kept[i, 0, m:] == -1).all(), i
        assert torch.equal(out[0][i, 0, :m], k[i, 0, want]) and torch.equal(out[1][i, 0, :m], v[i, 0, want])
        assert torch.equal(w_out[i, 0, :m], w[i, 0, want])
    kept2, want_k = torch.empty_like(kept), [k[i, 0, kept[i, 0, :int(lens_out[i])].long()] for i in range(n)]
    C.kv_evict(k, v, w, kept2, lens, k, v, w, lens, n, H, L, L, D, budget, sinks, recent)
    assert torch.equal(kept2, kept) and torch.equal(lens, lens_out)
    for i in range(n):
        m = int(lens[i])
        assert torch.equal(k[i, 0, :m], want_k[i]) and torch.equal(v[i, 0, :m], -want_k[i])
        assert torch.equal(w[i, 0, :m], w_out[i, 0, :m])
