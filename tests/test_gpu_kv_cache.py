"""GPU tests of the bounded caches: the 8-bit append (codes and scales exactly those of the
definition), decode over 8-bit caches, decode that accumulates attention weights, and eviction,
against CPU references (kv_ref); and a loop that uses them together."""
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


def _u8(t):
    return t.view(torch.uint8)


def _filled_cache(n, H, L, D, block, seed):
    """An 8-bit cache with values everywhere: scales of several sizes, every code but NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache = C.kv8_cache(n, H, L, D, block)
    for codes, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
        c = torch.randint(0, 254, codes.shape, generator=gen, device="cuda")
        c = torch.where(c >= 127, c + 1, c)  # 127 (and 255) are NaN
        _u8(codes).copy_(c.to(torch.uint8))
        e = torch.randint(-14, -7, scale.shape, generator=gen, device="cuda")
        scale.copy_(torch.exp2(e.float()))
    return cache


# ------------------------------------------------------------------------ append

@pytest.mark.gpu
def test_append_rounds_every_bf16_value_as_defined(gpu):
    """Every finite bf16 of magnitude up to 448, in blocks whose scale is 1 (each holds a 448): ties
    to even, subnormals, signed zeros; and the same values as fp32."""
    bits = torch.arange(65536, dtype=torch.int32)
    x = (bits << 16).view(torch.float32)
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    D, block = 64, 16
    x = torch.cat([x, torch.zeros(-len(x) % (D - 1))]).view(-1, D - 1)
    x = torch.cat([x, torch.full((len(x), 1), 448.0)], 1)       # a 448 in every row
    rows = (len(x) + block - 1) // block * block
    x = torch.cat([x, torch.full((rows - len(x), D), 448.0)])[None, None]
    for dtype in (BF, F32):
        k8, v8, ks, vs = C.kv8_cache(1, 1, rows, D, block)
        src = x.to("cuda").to(dtype)
        C.kv8_append(k8, v8, ks, vs, src, -src, _int([0]), None, 1, 1, rows, rows, D, block)
        assert (ks == 1).all() and (vs == 1).all()
        assert torch.equal(_u8(k8).cpu(), R.e4m3(x.double()))
        assert torch.equal(_u8(v8).cpu(), R.e4m3(-x.double()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D,block,rows", [
    (1, 1, 1, 32, 16, 1), (3, 2, 70, 64, 32, 1), (4, 3, 100, 32, 16, 37), (5, 2, 300, 64, 128, 200),
    (6, 1, 129, 64, 64, 129), (5, 4, 96, 32, 128, 50), (8, 2, 515, 64, 16, 300),
])
def test_append_codes_and_scales(gpu, dtype, n, H, L, D, block, rows):
    """Ragged starts and counts, blocks that begin full, half full and empty, scales that grow and
    that stay, infinities, NaN, zeros, the smallest and largest magnitudes; rows past the count are
    not looked at, rows outside the append keep their codes and blocks their scales."""
    cache = _filled_cache(n, H, L, D, block, seed=L)
    x = _randn((n, rows, 3, H, D), seed=rows)     # a fused projection's output: q, k, v
    mul = [1.0, 1e-3, 50.0, 1e-38, 1e30, 0.0, 3e4, 1e-12]
    for i in range(n):
        x[i] *= mul[(i + 1) % len(mul)]
    if rows > 20:
        x[0, 3, :, 0, 5] = float("inf")
        x[0, 4, :, 0, 6] = float("nan")
        x[0, 5, :, H - 1] = -float("inf")
        x[1, 10:20] = 0.0
    x = x.to(dtype)
    lens = [0, L // 2 + 1, block, L, L - 1, 3, L + 5, -2][:n]
    counts = [rows, 1, rows - 1, rows, rows + 9, 0, 4, 5][:n]
    for i in range(n):
        x[i, max(0, min(counts[i], rows)):] = float("nan")
    want = [t.cpu().clone() for t in cache]
    k, v = x[:, :, 1].permute(0, 2, 1, 3), x[:, :, 2].permute(0, 2, 1, 3)
    C.kv8_append(*cache, k, v, _int(lens), _int(counts), n, H, rows, L, D, block)
    for j, src in ((0, k), (1, v)):
        R.append(_u8(want[j]), want[2 + j], src.float().cpu(), lens, counts, block)
        assert torch.equal(cache[2 + j].cpu(), want[2 + j])
        assert R.same_codes(_u8(cache[j]).cpu(), _u8(want[j]))


@pytest.mark.gpu
@pytest.mark.parametrize("D,block", [(64, 32), (64, 64), (64, 128), (32, 128)])
def test_append_without_counts_and_token_by_token(gpu, D, block):
    """A prompt appended at once and token by token ends with the same scales, and codes that the
    definition gives for that order."""
    n, H, L, rows = 3, 3, 200, 150
    x = _randn((n, H, rows, D), seed=3) * torch.linspace(0.1, 4, rows, device="cuda")[:, None]
    whole, steps = C.kv8_cache(n, H, L, D, block), C.kv8_cache(n, H, L, D, block)
    C.kv8_append(*whole, x, x, _int([0] * n), None, n, H, rows, L, D, block)
    want = [t.cpu().clone() for t in C.kv8_cache(n, H, L, D, block)]
    for t in range(rows):
        one = x[:, :, t:t + 1]
        C.kv8_append(*steps, one, one, _int([t] * n), None, n, H, 1, L, D, block)
        R.append(_u8(want[0]), want[2], one.cpu(), [t] * n, [1] * n, block)
    assert torch.equal(whole[2], steps[2]) and torch.equal(whole[3], steps[3])
    assert torch.equal(steps[2].cpu(), want[2])
    assert torch.equal(_u8(steps[0]).cpu(), _u8(want[0]))
    assert torch.equal(_u8(steps[0]), _u8(steps[1]))
    assert (_u8(steps[0])[:, :, rows:] == 0).all()
    # re-rounding moves a code by half a step of the new scale at most, on top of its own half step
    a, b = (R.values(_u8(t[0]).cpu()) for t in (whole, steps))
    assert ((a - b).abs() <= a.abs() * 2.0 ** -3 + 2.0 ** -9).all()


# ------------------------------------------------------------------------ 8-bit decode

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D,block,window,sinks", [
    (3, 2, 1, 64, 16, 0, 0), (8, 3, 40, 32, 32, 0, 0), (8, 12, 1024, 64, 32, 0, 0),
    (8, 2, 515, 64, 128, 0, 0), (4, 2, 2050, 32, 64, 0, 0), (3, 3, 9000, 64, 64, 0, 0),
    (8, 3, 700, 64, 16, 1, 0), (8, 2, 1500, 64, 32, 600, 30), (4, 3, 3000, 32, 128, 1100, 7),
    (2, 1, 300, 64, 64, 2 ** 31 - 1, 1024),
])
def test_kv8_decode(gpu, dtype, n, H, L, D, block, window, sinks):
    cache = _filled_cache(n, H, L, D, block, seed=L + 1)
    q = _randn((n, H, D), seed=L, dtype=dtype)
    lens = _int(([L, 0, 1, L // 2, L + 7, min(L, 513), max(L - 1, 0), min(L, block)] * 2)[:n])
    seen = lens.clamp(0, L)
    row = torch.arange(L, device="cuda") // block
    k, v = (R.values(_u8(c)) * s.double()[:, :, row, None] for c, s in
            ((cache[0], cache[2]), (cache[1], cache[3])))
    ref, bound, _, _ = R.decode(q, k, v, seen, D ** -0.5, window, sinks,
                                2.0 ** -8 if dtype == BF else 2.0 ** -24)
    # what is not seen is not read: NaN codes there, and NaN scales where a whole block is hidden
    j = torch.arange(L, device="cuda")[None, :]
    hidden = j >= seen[:, None]
    if window:
        hidden |= (j < seen[:, None] - window) & (j >= sinks)
    for codes in cache[:2]:
        _u8(codes).masked_fill_(hidden[:, None, :, None], 127)
    blocks = cache[2].shape[2]
    some = torch.zeros((n, blocks), device="cuda").index_add_(1, row, (~hidden).float())
    for scale in cache[2:]:
        scale.masked_fill_((some == 0)[:, None, :], float("nan"))
    most = min(L, window + sinks) if window else L
    ws = C.decode_kv8_workspace(n, H, most, D)
    out = torch.full_like(q, float("nan"))
    for _ in range(2):  # the second call finds the workspace as the first left it
        C.decode_attention_kv8(out, q, *cache, lens, n, H, L, D, block, D ** -0.5, window, sinks, ws)
        off = (out.double() - ref).abs()
        assert (off <= bound).all(), (off / (bound + 1e-30)).max().item()


@pytest.mark.gpu
def test_kv8_decode_of_a_nan_row(gpu):
    """A key held as NaN makes its (sequence, head) NaN, as in the bf16 cache, and no other."""
    n, H, L, D, block = 2, 2, 700, 64, 32
    cache = _filled_cache(n, H, L, D, block, seed=9)
    _u8(cache[0])[1, 0, 650, 3] = 127
    q = _randn((n, H, D), seed=2, dtype=BF)
    out = torch.empty_like(q)
    ws = C.decode_kv8_workspace(n, H, L, D)
    C.decode_attention_kv8(out, q, *cache, _int([L, L]), n, H, L, D, block, 0.125, 0, 0, ws)
    bad = torch.isnan(out).any(-1)
    assert bad.tolist() == [[False, False], [True, False]]


# ------------------------------------------------------------------------ weights

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D", [(3, 2, 1, 64), (8, 3, 200, 32), (8, 12, 1024, 64),
                                     (6, 2, 513, 64), (3, 3, 9001, 64), (2, 2, 5000, 32)])
def test_weights_decode(gpu, dtype, n, H, L, D):
    q, k, v = (_randn(s, seed, dtype) for s, seed in
               (((n, H, D), 1), ((n, H, L, D), 2), ((n, H, L, D), 3)))
    lens = _int([L, 0, 1, L // 2, L + 7, min(L, 257), max(L - 1, 0), min(L, 512)][:n])
    before = torch.rand((n, H, L), device="cuda") * 100
    out_half = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    ref, bound, p, e_p = R.decode(q, k.double(), v.double(), lens, D ** -0.5, out_half=out_half)
    hidden = (torch.arange(L, device="cuda")[None, :] >= lens.clamp(0, L)[:, None])
    for x in (k, v):
        x.masked_fill_(hidden[:, None, :, None], float("nan"))
    ws = C.decode_weights_workspace(n, H, L, D)
    if ws is not None:
        ws.fill_(0xFF)  # whatever it held before must not matter
    out, after = torch.full_like(q, float("nan")), torch.full_like(before, float("nan"))
    C.decode_attention_weights(out, after, q, k, v, before, lens, n, H, L, D, D ** -0.5, ws)
    assert ((out.double() - ref).abs() <= bound).all()
    want = before.double() + p
    assert ((after.double() - want).abs() <= e_p + want * 2.0 ** -24).all()
    # in place, twice; and what lies past the length stays
    acc = before.clone()
    for _ in range(2):
        C.decode_attention_weights(out, acc, q, k, v, acc, lens, n, H, L, D, D ** -0.5, ws)
    want = before.double() + 2 * p
    assert ((acc.double() - want).abs() <= 2 * e_p + 2 * want * 2.0 ** -24).all()
    assert torch.equal(acc.masked_select(hidden[:, None]), before.masked_select(hidden[:, None]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("L,m", [(900, 300), (1000, 600), (2500, 1100)])
def test_weights_decode_of_scores_of_minus_infinity(gpu, dtype, L, m):
    """Keys whose score is -inf weigh 0, also where a wave, a chunk or the first of two chunks
    holds nothing else: the answer is that of the other keys alone."""
    n, H, D = 2, 2, 64
    q, k, v = (_randn(s, seed, dtype) for s, seed in
               (((n, H, D), 4), ((n, H, L, D), 5), ((n, H, L, D), 6)))
    q[..., 0] = 1
    lens, rest = _int([L, L - 5]), _int([L - m, L - 5 - m])
    out_half = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    ref, bound, p, e_p = R.decode(q, k[:, :, m:].double(), v[:, :, m:].double(), rest, D ** -0.5,
                                  out_half=out_half)
    k[:, :, :m, 0] = -float("inf")
    before = torch.zeros((n, H, L), device="cuda")
    ws = C.decode_weights_workspace(n, H, L, D)
    out, after = torch.empty_like(q), torch.empty_like(before)
    C.decode_attention_weights(out, after, q, k, v, before, lens, n, H, L, D, D ** -0.5, ws)
    assert ((out.double() - ref).abs() <= bound).all()
    assert (after[..., :m] == 0).all()
    assert ((after[..., m:].double() - p).abs() <= e_p + p * 2.0 ** -24).all()


# ------------------------------------------------------------------------ eviction

def _weights(n, H, L, seed):
    """Weights with many ties, zeros of both signs, infinities, negatives and NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.round(torch.rand((n, H, L), generator=gen, device="cuda").pow(4) * 20) / 4
    r = torch.rand((n, H, L), generator=gen, device="cuda")
    w = torch.where(r < 0.05, -0.0, w)
    w = torch.where((r > 0.05) & (r < 0.08), float("nan"), w)
    w = torch.where((r > 0.08) & (r < 0.1), float("inf"), w)
    return torch.where((r > 0.1) & (r < 0.15), -w, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,H,L,D,budget,sinks,recent", [
    (3, 2, 1, 64, 1, 0, 0), (8, 2, 50, 32, 7, 2, 3), (8, 3, 300, 64, 100, 4, 32),
    (8, 2, 300, 64, 36, 4, 32), (8, 1, 257, 32, 256, 0, 1), (8, 2, 2500, 64, 600, 1, 0),
    (8, 2, 4100, 32, 2100, 16, 500), (3, 2, 40, 64, 90, 4, 32), (2, 1, 9000, 64, 5000, 0, 0),
    (2, 150, 2300, 32, 900, 2, 30), (3, 100, 4500, 32, 900, 2, 30),
    (4, 1, 20000, 32, 7000, 4, 100), (8, 2, 8192, 32, 80, 4, 20),
])
def test_evict(gpu, dtype, n, H, L, D, budget, sinks, recent):
    k, v = (_randn((n, H, L, D), s, dtype) for s in (1, 2))
    w = _weights(n, H, L, seed=L)
    lens_l = [L, 0, 1, L // 2, L + 7, min(L, budget), min(L, budget + 1), max(L - 1, 0)][:n]
    lens = _int(lens_l)
    most = min(budget, L)
    k_out, v_out = (torch.full((n, H, most + 3, D), 7.0, device="cuda").to(dtype) for _ in range(2))
    w_out = torch.full((n, H, most + 3), 7.0, device="cuda")
    kept = torch.full((n, H, budget), -9, dtype=torch.int32, device="cuda")
    lens_out = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    C.kv_evict(k_out, v_out, w_out, kept, lens_out, k, v, w, lens, n, H, L, most + 3, D, budget,
               sinks, recent)
    wc, kept_c = w.cpu(), kept.cpu()
    for i in range(n):
        end = min(max(lens_l[i], 0), L)
        assert lens_out[i].item() == min(end, budget)
        for h in range(H):
            want = R.evict(wc[i, h], end, budget, sinks, recent)
            assert kept_c[i, h].tolist() == want + [-1] * (budget - len(want)), (i, h)
            at = torch.tensor(want, dtype=torch.long, device="cuda")
            m = len(want)
            assert torch.equal(k_out[i, h, :m], k[i, h, at]) and (k_out[i, h, m:] == 7).all()
            assert torch.equal(v_out[i, h, :m], v[i, h, at]) and (v_out[i, h, m:] == 7).all()
            assert torch.equal(w_out[i, h, :m].view(torch.int32), w[i, h, at].view(torch.int32))
            assert (w_out[i, h, m:] == 7).all()
    # in place, lens too
    k2, v2, w2, lens2, kept2 = (t.clone() for t in (k, v, w, lens, kept))
    C.kv_evict(k2, v2, w2, kept2, lens2, k2, v2, w2, lens2, n, H, L, L, D, budget, sinks, recent)
    assert torch.equal(kept2, kept) and torch.equal(lens2, lens_out)
    for i in range(n):
        m = lens_out[i].item()
        assert torch.equal(k2[i, :, :m], k_out[i, :, :m]) and torch.equal(k2[i, :, most:], k[i, :, most:])
        assert torch.equal(v2[i, :, :m], v_out[i, :, :m])
        assert torch.equal(w2[i, :, :m].view(torch.int32), w_out[i, :, :m].view(torch.int32))


# ------------------------------------------------------------------------ together

@pytest.mark.gpu
def test_a_serving_loop_over_bounded_caches(gpu):
    """Prompts through the windowed forward, their keys and values into an 8-bit cache, then tokens
    one by one: each step appends and attends with the same window. Beside it a bf16 cache that
    accumulates weights and is cut back whenever it passes its budget. Every step's output is
    checked against the same steps in float64 on the rows that the caches hold."""
    n, H, D, L, block, window, sinks, scale = 3, 4, 64, 200, 32, 48, 4, 0.125
    budget, recent = 64, 16
    prompts = [90, 1, 60]
    S = max(prompts)
    qkv = _randn((n, S, 3, H, D), seed=21, dtype=BF)
    heads = [qkv[:, :, i].permute(0, 2, 1, 3) for i in range(3)]
    out = torch.empty((n, H, S, D), dtype=BF, device="cuda")
    lse = torch.empty((n * H, S), device="cuda")
    A.flash_attention_window_forward_bf16_strided(out, lse, *heads, scale, window, sinks)
    lens = _int(prompts)
    cache = C.kv8_cache(n, H, L, D, block)
    C.kv8_append(*cache, heads[1], heads[2], _int([0] * n), lens, n, H, S, L, D, block)
    k, v = (torch.zeros((n, H, L, D), dtype=BF, device="cuda") for _ in range(2))
    k[:, :, :S], v[:, :, :S] = heads[1], heads[2]
    w = torch.zeros((n, H, L), device="cuda")
    blens = lens.clone()
    kept = torch.empty((n, H, budget), dtype=torch.int32, device="cuda")
    ws8, wsw = C.decode_kv8_workspace(n, H, L, D), C.decode_weights_workspace(n, H, L, D)
    row = torch.arange(L, device="cuda") // block
    evictions = 0
    for step in range(40):
        q1, k1, v1 = (_randn((n, H, 1, D), seed=100 + 3 * step + i, dtype=BF) for i in range(3))
        C.kv8_append(*cache, k1, v1, lens, None, n, H, 1, L, D, block)
        lens += 1
        o = torch.empty((n, H, D), dtype=BF, device="cuda")
        C.decode_attention_kv8(o, q1[:, :, 0].contiguous(), *cache, lens, n, H, L, D, block, scale,
                               window, sinks, ws8)
        kk, vv = (R.values(_u8(c)) * s.double()[:, :, row, None] for c, s in
                  ((cache[0], cache[2]), (cache[1], cache[3])))
        ref, bound, _, _ = R.decode(q1[:, :, 0], kk, vv, lens, scale, window, sinks, 2.0 ** -8)
        assert ((o.double() - ref).abs() <= bound).all(), step
        # the codes stand for the rows to half a step of e4m3 (2^-4), twice where re-rounded, and
        # for small ones half of its least step
        for i in range(n):
            at = int(lens[i]) - 1
            s = cache[2][i, :, at // block, None].double()
            assert ((kk[i, :, at] - k1[i, :, 0].double()).abs()
                    <= k1[i, :, 0].double().abs() * 2.0 ** -4 + s * 2.0 ** -10).all()

        for i in range(n):  # the bf16 cache's own append
            k[i, :, int(blens[i])], v[i, :, int(blens[i])] = k1[i, :, 0], v1[i, :, 0]
        blens += 1
        C.decode_attention_weights(o, w, q1[:, :, 0].contiguous(), k, v, w, blens, n, H, L, D,
                                   scale, wsw)
        ref, bound, p, _ = R.decode(q1[:, :, 0], k.double(), v.double(), blens, scale,
                                    out_half=2.0 ** -8)
        assert ((o.double() - ref).abs() <= bound).all(), step
        if int(blens.max()) > budget + 8:
            C.kv_evict(k, v, w, kept, blens, k, v, w, blens, n, H, L, L, D, budget, sinks, recent)
            for i in range(n):  # a row that was not there yet starts from nothing
                w[i, :, int(blens[i]):] = 0
            evictions += 1
    assert evictions >= 3 and int(blens.max()) <= budget + 8


@pytest.mark.gpu
def test_cache_calls_repeat_on_streams_and_in_graphs(gpu):
    """One decode step captured (append, both decodes, eviction into another cache) and replayed,
    with eager work between, gives the eager bits every time; so does another stream."""
    n, H, D, L, block, budget = 4, 3, 64, 1500, 32, 300
    cache0 = _filled_cache(n, H, L, D, block, seed=31)
    q, k1, v1 = (_randn((n, H, 1, D), seed=s, dtype=BF) for s in (1, 2, 3))
    q = q[:, :, 0].contiguous()
    k, v = (_randn((n, H, L, D), s, BF) for s in (4, 5))
    w = torch.rand((n, H, L), device="cuda")
    lens = _int([L - 1, 700, 0, 1])
    ws8, wsw = C.decode_kv8_workspace(n, H, L, D), C.decode_weights_workspace(n, H, L, D)

    def buffers():
        return {"o8": torch.empty_like(q), "ow": torch.empty_like(q), "w": torch.empty_like(w),
                "k": torch.zeros((n, H, budget, D), dtype=BF, device="cuda"),
                "v": torch.zeros((n, H, budget, D), dtype=BF, device="cuda"),
                "we": torch.zeros((n, H, budget), device="cuda"),
                "kept": torch.empty((n, H, budget), dtype=torch.int32, device="cuda"),
                "lens": torch.empty_like(lens), "cache": [t.clone() for t in cache0]}

    def step(b):
        C.kv8_append(*b["cache"], k1, v1, lens, None, n, H, 1, L, D, block)
        C.decode_attention_kv8(b["o8"], q, *b["cache"], lens, n, H, L, D, block, 0.125, 0, 0, ws8)
        C.decode_attention_weights(b["ow"], b["w"], q, k, v, w, lens, n, H, L, D, 0.125, wsw)
        C.kv_evict(b["k"], b["v"], b["we"], b["kept"], b["lens"], k, v, b["w"], lens, n, H, L, budget,
                   D, budget, 4, 100)

    def flat(b):
        return [t.view(torch.uint8) for t in [x for key, x in b.items() if key != "cache"] + b["cache"]]

    eager = buffers()
    step(eager)
    want = [t.clone() for t in flat(eager)]
    side = torch.cuda.Stream()
    other = buffers()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(other)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(flat(other), want))
    b = buffers()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for _ in range(3):
        for t in flat(b)[:-4]:
            t.zero_()
        for t, x in zip(b["cache"], cache0):
            t.view(torch.uint8).copy_(x.view(torch.uint8))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, x) for a, x in zip(flat(b), want))
        step(eager)


@pytest.mark.gpu
def test_kv8_past_32_bit_offsets(gpu):
    """Five 8-bit caches of 16,776,960 rows (1.07 GB of codes each, so the last ones lie past 2^32
    bytes): rows appended at the very end and read back through a window."""
    n, H, L, D, block, window = 5, 1, 65535 * 256, 64, 64, 40
    cache = C.kv8_cache(n, H, L, D, block)
    x = _randn((n, H, window, D), seed=41, dtype=BF)
    y = _randn((n, H, window, D), seed=42, dtype=BF)
    q = _randn((n, H, D), seed=43, dtype=BF)
    C.kv8_append(*cache, x, y, _int([L - window] * n), None, n, H, window, L, D, block)
    want = torch.zeros((1, H, 2 * block, D), dtype=torch.uint8), torch.zeros((1, H, 2))
    at = 2 * block - window
    for i in (0, n - 1):
        codes, scale = want[0].clone(), want[1].clone()
        R.append(codes, scale, x[i:i + 1].float().cpu(), [at], [window], block)
        assert torch.equal(_u8(cache[0])[i, :, L - window:].cpu(), codes[0, :, at:])
        assert torch.equal(cache[2][i, :, -1].cpu(), scale[0, :, -1])
    out = torch.empty_like(q)
    C.decode_attention_kv8(out, q, *cache, _int([L] * n), n, H, L, D, block, 0.125, window, 0, None)
    k, v = (R.values(_u8(c)[:, :, L - window:].contiguous()) * s[:, :, -1:, None].double()
            for c, s in ((cache[0], cache[2]), (cache[1], cache[3])))
    ref, bound, _, _ = R.decode(q, k, v, [window] * n, 0.125, out_half=2.0 ** -8)
    assert ((out.double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("L,budget,sinks,recent", [(6000, 700, 3, 50), (3000, 1500, 0, 0),
                                                   (9000, 4000, 10, 10)])
def test_evict_of_many_equal_weights(gpu, L, budget, sinks, recent):
    """More rows of one weight than are ranked against each other: the edge is among them, and the
    lowest rows of it stay."""
    n, H, D = 3, 2, 32
    k, v = (_randn((n, H, L, D), s) for s in (1, 2))
    w = torch.zeros((n, H, L), device="cuda")
    w[1] = (torch.arange(L, device="cuda") % 7 == 0).float()      # two weights
    w[2] = -0.0
    w[2, 1, ::3] = float("nan")
    out = [torch.empty((n, H, budget, D), device="cuda") for _ in range(2)]
    w_out = torch.empty((n, H, budget), device="cuda")
    kept = torch.empty((n, H, budget), dtype=torch.int32, device="cuda")
    lens_out = torch.empty(n, dtype=torch.int32, device="cuda")
    C.kv_evict(*out, w_out, kept, lens_out, k, v, w, _int([L, L, L - 1]), n, H, L, budget, D, budget,
               sinks, recent)
    for i, end in enumerate((L, L, L - 1)):
        for h in range(H):
            assert kept[i, h].tolist() == R.evict(w[i, h].cpu(), end, budget, sinks, recent), (i, h)
            assert torch.equal(out[0][i, h], k[i, h, kept[i, h].long()])


@pytest.mark.gpu
def test_kv8_append_of_rows_with_odd_strides(gpu):
    """Rows read out of wider buffers, K and V with strides of their own, and a single head or row
    whose stride torch leaves arbitrary."""
    n, H, L, D, block, rows = 2, 3, 64, 32, 16, 9
    big = _randn((rows, n, H, 48), seed=51)            # row-major in tokens, gaps after each head
    k = big[..., 8:40].permute(1, 2, 0, 3)
    v = _randn((H, n, rows, D), seed=52).permute(1, 0, 2, 3)
    a, b = C.kv8_cache(n, H, L, D, block), C.kv8_cache(n, H, L, D, block)
    C.kv8_append(*a, k, v, _int([3, 11]), None, n, H, rows, L, D, block)
    C.kv8_append(*b, k.contiguous(), v.contiguous(), _int([3, 11]), None, n, H, rows, L, D, block)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    one = torch.as_strided(k.contiguous()[:1, :1, :1], (1, 1, 1, D), (5, 3, 1, 1))
    c = C.kv8_cache(1, 1, L, D, block)
    C.kv8_append(*c, one, one, _int([0]), None, 1, 1, 1, L, D, block)
    want = torch.zeros((1, 1, L, D), dtype=torch.uint8), torch.zeros((1, 1, L // block))
    R.append(*want, one.cpu(), [0], [1], block)
    assert torch.equal(_u8(c[0]).cpu(), want[0]) and torch.equal(c[2].cpu(), want[1])


@pytest.mark.gpu
def test_cache_wrappers_refuse_what_does_not_fit(gpu):
    n, H, L, D, block = 2, 2, 32, 32, 16
    cache = C.kv8_cache(n, H, L, D, block)
    x, lens = _randn((n, H, 3, D), seed=1), _int([0, 0])
    with pytest.raises(ValueError, match="contiguous rows"):
        C.kv8_append(*cache, x.transpose(2, 3), x, lens, None, n, H, 3, L, D, block)
    with pytest.raises(TypeError, match="v must be"):
        C.kv8_append(*cache, x, x.to(BF), lens, None, n, H, 3, L, D, block)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        C.kv8_append(*cache, x.half(), x.half(), lens, None, n, H, 3, L, D, block)
    with pytest.raises(ValueError, match="k_cache has"):
        C.kv8_append(cache[0][:1], *cache[1:], x, x, lens, None, n, H, 3, L, D, block)
    with pytest.raises(TypeError, match="float8"):
        C.kv8_append(_u8(cache[0]), *cache[1:], x, x, lens, None, n, H, 3, L, D, block)
    with pytest.raises(ValueError, match="block"):
        C.kv8_append(*cache, x, x, lens, None, n, H, 3, L, D, 24)
    k = _randn((n, H, L, D), seed=2)
    w = torch.zeros((n, H, L), device="cuda")
    kept = torch.empty((n, H, 8), dtype=torch.int32, device="cuda")
    with pytest.raises(A.AttentionError, match="in place"):
        C.kv_evict(k, k.clone(), w, kept, lens, k, k.clone(), w, lens, n, H, L, L, D, 8, 0, 0)
    with pytest.raises(ValueError, match="kept has"):
        C.kv_evict(k, k, w, kept[:1], lens, k, k, w, lens, n, H, L, L, D, 8, 0, 0)
