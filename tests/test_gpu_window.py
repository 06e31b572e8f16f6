"""GPU tests of sliding-window attention with sinks: forward and backward in bf16 and fp32 and the
one-token form, against float64 with element-wise error bounds (window_ref), the layouts against
each other bit for bit, gradients against differences, repeats, streams and graphs."""
import pytest
import torch

from dadgpt_amd import attention as A
from tests import window_ref as R

BF, F32 = torch.bfloat16, torch.float32


def _inputs(BH, S, D, dtype, seed, n=4):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn((BH, S, D), generator=gen, device="cuda").to(dtype) for _ in range(n)]


def _run(q, k, v, g, scale, window, sinks, stream=None):
    BH, S, D = q.shape
    out, dq, dk, dv = (torch.full_like(q, float("nan")) for _ in range(4))
    lse, delta = (torch.full((BH, S), float("nan"), device="cuda") for _ in range(2))
    ws = A.window_workspace(BH, S, D, window, sinks)
    if ws is not None:
        ws.fill_(0xFF)  # whatever the workspace held before (NaN patterns) must not matter
    f, b = ((A.flash_attention_window_forward_bf16, A.flash_attention_window_backward_bf16)
            if q.dtype == BF else
            (A.flash_attention_window_forward, A.flash_attention_window_backward))
    f(out, lse, q, k, v, BH, S, D, scale, window, sinks, stream)
    b(dq, dk, dv, delta, g, out, lse, q, k, v, BH, S, D, scale, window, sinks, ws, stream)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


# (BH, S, D, window, sinks): one token; windows of one key, inside a chunk, across tiles, of almost
# the whole sequence; sinks none, one, across a chunk, a tile and a key block, more than the
# window, more than the sequence; lengths off every tile; sums of sink keys in one and in many
# pieces (sequences of 8 tiles and more), on small grids (two waves a row group) and large ones
CASES = [
    (2, 1, 64, 1, 0), (3, 2, 32, 1, 1), (2, 33, 64, 1, 0), (2, 64, 32, 7, 3), (5, 65, 64, 64, 0),
    (3, 129, 64, 31, 1), (3, 130, 32, 33, 40), (2, 200, 64, 199, 4), (2, 257, 64, 100, 300),
    (4, 300, 64, 16, 65), (2, 511, 32, 130, 64), (7, 600, 64, 1, 5), (3, 777, 32, 100, 3),
    (2, 777, 64, 100, 3), (2, 1024, 64, 256, 4), (40, 650, 64, 65, 33), (130, 530, 64, 40, 2),
    (300, 300, 32, 90, 4), (1, 1500, 64, 3, 130), (2, 2100, 64, 1000, 4), (1, 2300, 32, 900, 200),
    (1, 1800, 64, 17, 1024), (240, 1100, 64, 80, 4), (240, 1100, 32, 80, 4), (240, 1100, 64, 80, 0),
    (20, 2100, 64, 1000, 4), (20, 2100, 32, 1000, 0), (260, 200, 64, 33, 2), (24, 1024, 32, 200, 40),
    (12, 1024, 64, 250, 4), (5, 2100, 64, 1000, 4), (6, 1300, 64, 40, 300),
    (2, 4500, 64, 30, 40), (1, 6000, 32, 100, 130), (9, 6500, 64, 60, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("BH,S,D,window,sinks", CASES)
def test_window_attention(gpu, dtype, BH, S, D, window, sinks):
    scale = D ** -0.5
    q, k, v, g = _inputs(BH, S, D, dtype, seed=S + window)
    got = _run(q, k, v, g, scale, window, sinks)
    # float64 scores of every slice at once take BH S^2 8 bytes a matrix: sampled for large grids
    pick = slice(0, BH) if BH * S * S < 2e7 else slice(0, BH, max(1, BH // 8))
    ref = R.attention(q[pick], k[pick], v[pick], g[pick], scale, window, sinks, dtype)
    R.assert_within({n: x[pick] for n, x in got.items()}, ref, (BH, S, D, window, sinks))
    assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.125, 1.0, 0.0, 1e-20])
def test_window_scales(gpu, dtype, scale):
    """A negative scale, and one that makes the softmax sharp."""
    q, k, v, g = _inputs(2, 333, 64, dtype, seed=5)
    got = _run(q, k, v, g, scale, 70, 9)
    R.assert_within(got, R.attention(q, k, v, g, scale, 70, 9, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_window_large_scores(gpu, dtype):
    """Scores that differ by hundreds between a row's chunks: the running maximum has to move, and
    rows that see nothing of their wave's first chunk start later than the others."""
    q, k, v, g = _inputs(3, 400, 64, dtype, seed=6)
    k = (k * torch.linspace(0.05, 12.0, 400, device="cuda")[None, :, None]).to(dtype)
    q = (q * 3).to(dtype)
    got = _run(q, k, v, g, 0.125, 50, 2)
    R.assert_within(got, R.attention(q, k, v, g, 0.125, 50, 2, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(64, 0), (200, 4)])
@pytest.mark.parametrize("BH", [4, 120])
def test_window_gradients_carry_ds_in_two_values(gpu, BH, window, sinks):
    """dQ and dK in bf16 are off by little more than their own rounding. dS in one bf16 value would
    add an error of the same size and independent of it (in all 2^0.5 times the rounding's); in two
    it adds 2^-8 of that, and what is left beside the rounding is delta's error, a sum over d_head
    of the output's, which is shared by a row's keys and a fraction of either."""
    q, k, v, g = _inputs(BH, 900, 64, BF, seed=21)
    got = _run(q, k, v, g, 0.125, window, sinks)
    pick = slice(0, 4)
    ref = R.attention(q[pick], k[pick], v[pick], g[pick], 0.125, window, sinks, BF)
    for name in ("dq", "dk"):
        exact = ref[name][0]
        own = (exact.to(BF).double() - exact).norm()
        assert (got[name][pick].double() - exact).norm() <= 1.25 * own, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("S,window", [(1, 1), (100, 100), (321, 4000), (1024, 2 ** 31 - 1)])
def test_a_window_of_the_sequence_is_the_causal_call(gpu, dtype, S, window):
    q, k, v, g = _inputs(4, S, 64, dtype, seed=7)
    got = _run(q, k, v, g, 0.125, window, 3)
    out, lse = A.attention_forward(q, k, v, 0.125)
    dq, dk, dv, _ = A.attention_backward(g, out, lse, q, k, v, 0.125)
    for name, x in {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}.items():
        assert torch.equal(got[name], x), name


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,S,D,window,sinks", [(2, 3, 777, 64, 100, 3), (1, 4, 1300, 32, 1100, 70),
                                                  (16, 12, 300, 64, 64, 4), (3, 2, 63, 64, 9, 1),
                                                  (20, 12, 1100, 64, 80, 4), (20, 12, 1100, 32, 80, 0),
                                                  (2, 4, 1300, 64, 200, 0)])
def test_token_major_and_strided_give_the_contiguous_bits(gpu, B, H, S, D, window, sinks):
    d, scale = H * D, D ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(B + S)
    qkv = torch.randn((B * S, 3 * d), generator=gen, device="cuda").to(BF)
    dout = torch.randn((B * S, d), generator=gen, device="cuda").to(BF)

    def heads(x):
        return x.view(B, S, H, D).transpose(1, 2).reshape(B * H, S, D).contiguous()

    q, k, v = (qkv[:, i * d:(i + 1) * d] for i in range(3))
    want = _run(heads(q.contiguous()), heads(k.contiguous()), heads(v.contiguous()), heads(dout),
                scale, window, sinks)
    ws = A.window_workspace(B * H, S, D, window, sinks)
    out, dqkv = torch.empty_like(dout), torch.empty_like(qkv)
    lse, delta = (torch.empty((B * H, S), device="cuda") for _ in range(2))
    dq, dk, dv = (dqkv[:, i * d:(i + 1) * d] for i in range(3))
    A.flash_attention_window_forward_bf16_tokens(out, d, lse, q, k, v, 3 * d, B, H, S, D, scale,
                                                 window, sinks)
    A.flash_attention_window_backward_bf16_tokens(dq, dk, dv, 3 * d, delta, dout, out, d, lse, q, k,
                                                  v, 3 * d, B, H, S, D, scale, window, sinks, ws)
    assert torch.equal(lse, want["lse"])
    for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.equal(heads(x.contiguous()), want[name]), name

    # rows of a wider buffer, the gaps left as they were
    def view(n=1):
        big = torch.full((B, H, S + 3, D + 8), 7.0, device="cuda").to(BF)
        return big, big[:, :, 1:S + 1, :D]

    views = {}
    for name, x in (("q", q), ("k", k), ("v", v), ("dout", dout)):
        views[name] = view()
        views[name][1].copy_(x.reshape(B, S, H, D).transpose(1, 2))
    for name in ("out", "dq", "dk", "dv"):
        views[name] = view()
    w = {n: x[1] for n, x in views.items()}
    A.flash_attention_window_forward_bf16_strided(w["out"], lse, w["q"], w["k"], w["v"], scale,
                                                  window, sinks)
    A.flash_attention_window_backward_bf16_strided(w["dq"], w["dk"], w["dv"], delta, w["dout"],
                                                   w["out"], lse, w["q"], w["k"], w["v"], scale,
                                                   window, sinks, ws)
    for name in ("out", "dq", "dk", "dv"):
        big, rows = views[name]
        assert torch.equal(rows.reshape(B * H, S, D), want[name]), name
        rows.fill_(7.0)
        assert (big == 7.0).all(), name


@pytest.mark.gpu
def test_window_gradients_against_differences(gpu):
    """d/dt of sum(out dout) along a direction, by central differences of the fp32 forward: the
    difference's own error is h^2/6 of the third derivative (below 1e-4 of the value at this h and
    size) and the forward's rounding over h."""
    BH, S, D, window, sinks, h = 2, 150, 32, 40, 5, 2.0 ** -7
    q, k, v, g, a, b, c = _inputs(BH, S, D, F32, seed=11, n=7)
    grads = _run(q, k, v, g, 0.2, window, sinks)

    def loss(t):
        r = _run(q + t * a, k + t * b, v + t * c, g, 0.2, window, sinks)
        return (r["out"].double() * g.double()).sum().item()

    num = (loss(h) - loss(-h)) / (2 * h)
    ana = sum((grads[n].double() * x.double()).sum().item()
              for n, x in (("dq", a), ("dk", b), ("dv", c)))
    size = sum((grads[n].double() * x.double()).norm().item()
               for n, x in (("dq", a), ("dk", b), ("dv", c)))
    assert abs(num - ana) <= 2e-3 * size, (num, ana, size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("BH", [6, 60])
def test_window_repeats_streams_and_graph_replays(gpu, dtype, BH):
    """The same bits on every call, on another stream, and on every replay of a captured graph with
    eager work between, for backwards of several pieces on a small and a large grid."""
    S, D, window, sinks = 1400, 64, 90, 20
    q, k, v, g = _inputs(BH, S, D, dtype, seed=13)
    want = {n: x.clone() for n, x in _run(q, k, v, g, 0.125, window, sinks).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, g, 0.125, window, sinks)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse, delta = (torch.empty((BH, S), device="cuda") for _ in range(2))
    ws = A.window_workspace(BH, S, D, window, sinks)
    f, b = ((A.flash_attention_window_forward_bf16, A.flash_attention_window_backward_bf16)
            if dtype == BF else
            (A.flash_attention_window_forward, A.flash_attention_window_backward))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f(out, lse, q, k, v, BH, S, D, 0.125, window, sinks)
        b(dq, dk, dv, delta, g, out, lse, q, k, v, BH, S, D, 0.125, window, sinks, ws)
    for _ in range(3):
        for x in (out, dq, dk, dv, lse, ws):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for n, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
            assert torch.equal(x, want[n]), n
        _run(q, k, v, g, 0.125, window, sinks)


@pytest.mark.gpu
def test_window_backward_leaves_the_end_of_its_workspace(gpu):
    BH, S, D, window, sinks = 3, 2000, 64, 100, 40
    q, k, v, g = _inputs(BH, S, D, BF, seed=17)
    need = A.window_workspace_bytes(BH, S, D, window, sinks)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse, delta = (torch.empty((BH, S), device="cuda") for _ in range(2))
    A.flash_attention_window_forward_bf16(out, lse, q, k, v, BH, S, D, 0.125, window, sinks)
    A.flash_attention_window_backward_bf16(dq, dk, dv, delta, g, out, lse, q, k, v, BH, S, D, 0.125,
                                           window, sinks, ws[:need])
    torch.cuda.synchronize()
    assert (ws[need:] == 0x5A).all()


# ----------------------------------------------------------------------- one token

def _decode_ref(q, k, v, lens, window, sinks, scale):
    """float64 outputs, and what half a step of the output and the fp32 sums may change."""
    out, bound = [], []
    for i, end in enumerate(lens.tolist()):
        j = torch.arange(end, device="cuda")
        j = j[(j >= end - window) | (j < sinks)]
        kk, vv = k[i][:, j].double(), v[i][:, j].double()
        if len(j) == 0:
            out.append(torch.zeros_like(q[i], dtype=torch.float64))
            bound.append(torch.zeros_like(out[-1]))
            continue
        s = (kk * q[i].double()[:, None]).sum(-1) * scale
        e = (kk.abs() * q[i].double().abs()[:, None]).sum(-1) * abs(scale) * 72 * R.F32_HALF
        p = torch.softmax(s, -1)[..., None]
        o = (p * vv).sum(1)
        u = R.BF16_HALF if q.dtype == BF else R.F32_HALF
        # exponents off by e (own and the normaliser's) and a few fp32 roundings, sums over the keys
        rel = 2 * e.amax(-1)[:, None] + 2.0 ** -19 + len(j) / 8 * R.F32_HALF
        out.append(o)
        bound.append(rel * (p * vv.abs()).sum(1) + u * o.abs())
    return torch.stack(out), torch.stack(bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D,window,sinks", [
    (3, 2, 1, 64, 1, 0), (5, 3, 40, 32, 1, 0), (6, 4, 300, 64, 7, 3), (8, 3, 1024, 64, 256, 4),
    (4, 2, 1025, 32, 700, 1024), (3, 2, 5000, 64, 1500, 64), (2, 3, 9001, 64, 8000, 600),
    (2, 1, 3000, 32, 2 ** 31 - 1, 5),
])
def test_window_decode(gpu, dtype, n, H, L, D, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(L)
    q = torch.randn((n, H, D), generator=gen, device="cuda").to(dtype)
    k, v = (torch.randn((n, H, L, D), generator=gen, device="cuda").to(dtype) for _ in range(2))
    # no row, one, the window's edges, the end, and past the end (clamped)
    lens = [0, 1, min(L, window), min(L, window + sinks), min(L, window + sinks + 1), L, L + 9, L // 2]
    lens = torch.tensor(lens[:n] if n >= 4 else lens[-n:], dtype=torch.int32, device="cuda")
    seen = lens.clamp(0, L)
    # what the last row does not see is never read: NaN there changes nothing
    j = torch.arange(L, device="cuda")[None, :]
    hidden = (j >= seen[:, None]) | ((j < seen[:, None] - window) & (j >= sinks))
    ref, bound = _decode_ref(q, k, v, seen, window, sinks, D ** -0.5)
    for x in (k, v):
        x.masked_fill_(hidden[:, None, :, None], float("nan"))
    out = torch.full_like(q, float("nan"))
    ws = A.decode_workspace(n, H, min(L, window + sinks), D)
    for _ in range(2):  # the second call finds the workspace as the first left it
        A.decode_attention_window(out, q, k, v, lens, n, H, L, D, D ** -0.5, window, sinks, ws)
        off = (out.double() - ref).abs()
        assert (off <= bound).all(), (off / (bound + 1e-30)).max().item()


@pytest.mark.gpu
def test_window_decode_is_the_windowed_forward_of_the_last_row(gpu):
    """The two forms agree: the forward's last row, and a decode over the same keys (each within
    its bf16 rounding: two half steps of the output and one of the probabilities)."""
    B, H, S, D, window, sinks = 2, 3, 600, 64, 130, 4
    q, k, v, g = _inputs(B * H, S, D, BF, seed=19)
    got = _run(q, k, v, g, 0.125, window, sinks)["out"][:, -1].double()
    out = torch.empty((B, H, D), dtype=BF, device="cuda")
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    A.decode_attention_window(out, q[:, -1].reshape(B, H, D).contiguous(), k, v, lens, B, H, S, D,
                              0.125, window, sinks, None)
    ref = R.attention(q, k, v, g, 0.125, window, sinks, BF)["out"]
    o, e = ref[0][:, -1], ref[1][:, -1]
    assert ((out.view(B * H, D).double() - got).abs() <= 2 * e).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_window_over_a_long_sequence(gpu, dtype):
    """30,000 tokens with a gradient in the first and the last 300 rows only: what those rows give is
    what they give in two short sequences, of the first rows, and of the sinks and the last rows;
    the sink keys' gradients are the sum of both."""
    BH, S, D, window, sinks, n = 3, 30000, 64, 100, 5, 300
    q, k, v, g = _inputs(BH, S, D, dtype, seed=23)
    g[:, n:S - n] = 0
    got = _run(q, k, v, g, 0.125, window, sinks)
    first = [x[:, :n + 200] for x in (q, k, v, g)]
    last = [torch.cat((x[:, :sinks], x[:, S - n - 200:]), 1) for x in (q, k, v, g)]
    last[3] = last[3].clone()
    last[3][:, :sinks] = 0
    a = R.attention(*first, 0.125, window, sinks, dtype)
    b = R.attention(*last, 0.125, window, sinks, dtype)
    R.assert_within({m: got[m][:, :n] for m in ("out", "lse", "dq")},
                    {m: (a[m][0][:, :n], a[m][1][:, :n]) for m in ("out", "lse", "dq")})
    R.assert_within({m: got[m][:, S - n:] for m in got},
                    {m: (b[m][0][:, -n:], b[m][1][:, -n:]) for m in got})
    R.assert_within({m: got[m][:, sinks:n] for m in ("dk", "dv")},
                    {m: (a[m][0][:, sinks:n], a[m][1][:, sinks:n]) for m in ("dk", "dv")})
    # the sums over 30,000 rows: the rows between add nothing but their place in the order of the sum
    slack = 2.0 ** -24 * (S / 16) * (1 if dtype == BF else 6)
    for m in ("dk", "dv"):
        y = a[m][0][:, :sinks] + b[m][0][:, :sinks]
        e = a[m][1][:, :sinks] + b[m][1][:, :sinks] + slack * y.abs().amax()
        assert ((got[m][:, :sinks].double() - y).abs() <= e).all(), m


@pytest.mark.gpu
def test_window_decode_past_32_bit_offsets(gpu):
    """fp32 caches of 16,776,960 rows (the launch limit; 4.3 GB each, so the last rows lie past 2^32
    bytes): the windowed rows only are read."""
    n, H, L, D, window, sinks = 1, 1, 65535 * 256, 64, 700, 4
    k, v = (torch.zeros((n, H, L, D), device="cuda") for _ in range(2))
    rows = torch.cat((torch.arange(sinks), torch.arange(L - window, L))).cuda()
    gen = torch.Generator(device="cuda").manual_seed(29)
    q = torch.randn((n, H, D), generator=gen, device="cuda")
    kk, vv = (torch.randn((len(rows), D), generator=gen, device="cuda") for _ in range(2))
    k[0, 0, rows], v[0, 0, rows] = kk, vv
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    ws = A.decode_workspace(n, H, window + sinks, D)
    A.decode_attention_window(out, q, k, v, lens, n, H, L, D, 0.125, window, sinks, ws)
    ref, bound = _decode_ref(q, kk[None, None], vv[None, None],
                             torch.tensor([len(rows)]), len(rows), 0, 0.125)
    assert ((out.double() - ref).abs() <= bound).all()
