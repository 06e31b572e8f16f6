"""GPU tests of the sampling: tokens equal to the definition's (serving_ref, sums in extended precision) for
rows whose decisions lie further from a border than the sums are off, and probabilities to fp32."""
import math

import numpy as np
import pytest
import torch

from dadgpt_amd import sampling
from tests import serving_ref as S

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
# Weights are multiples of 2^-44 of the largest: a sum of n is off by less than n 2^-45 of it, and the
# exponentials by 1e-14 of each weight.
MARGIN = 1e-8


def _sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = logits.shape[0]

    def dev(x, dtype=F32):
        return None if x is None else torch.tensor(x, dtype=dtype).cuda()
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((rows,), -7.0, device="cuda")
    sampling.sample(tokens, probs, logits.cuda() if not logits.is_cuda else logits, dev(u),
                    dev(temperature), dev(top_k, torch.int32), dev(top_p), dev(min_p))
    torch.cuda.synchronize()
    return tokens.cpu().tolist(), probs.cpu().tolist()


def _check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    tokens, probs = _sample(logits, u, temperature, top_k, top_p, min_p)
    x, checked = logits.float().cpu().numpy(), 0
    for r in range(len(u)):
        want, p, margin = S.sample(x[r], np.float32(u[r]), 1.0 if temperature is None else temperature[r],
                                   0 if top_k is None else top_k[r], 1.0 if top_p is None else top_p[r],
                                   0.0 if min_p is None else min_p[r])
        if margin < MARGIN:
            continue
        checked += 1
        assert tokens[r] == want, (r, tokens[r], want, margin)
        assert abs(probs[r] - p) <= 2.0 ** -23 * p + 1e-30
    assert checked >= 0.9 * len(u)


def _logits(rows, vocab, seed, dtype, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=gen) * spread).to(dtype)


def _uniforms(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 1000, 4096, 4097, 8193, 50257, 70001])
def test_settings(gpu, vocab, dtype):
    rows = 24
    x, u = _logits(rows, vocab, vocab, dtype), _uniforms(rows, vocab + 1)
    pick = [(t, k, p, m) for t in (0.7, 1.0, 1.7) for k, p, m in
            ((0, 1.0, 0.0), (1, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05),
             (200, 0.8, 0.01), (5000, 0.5, 0.0), (3, 0.999, 0.3))]
    assert len(pick) == rows
    _check(x, u, *(list(z) for z in zip(*pick)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [7, 1000, 9001])
def test_more_rows_than_cus(gpu, vocab, dtype):
    rows = 320
    x, u = _logits(rows, vocab, 100 + vocab, dtype), _uniforms(rows, vocab + 2)
    pick = [((0.6, 1.0, 1.9)[r % 3], *((0, 1.0, 0.0), (1, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0),
                                       (0, 1.0, 0.05), (200, 0.8, 0.01), (0, 0.999, 0.0))[r % 7])
            for r in range(rows)]
    _check(x, u, *(list(z) for z in zip(*pick)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_defaults_and_draws(gpu, dtype):
    """No settings; the draw follows the probabilities (4096 draws of one row: each of the likeliest
    tokens within five standard deviations)."""
    x = _logits(1, 300, 3, dtype, 1.5)
    rows = 4096
    u = ((torch.arange(rows) + 0.5) / rows).tolist()
    tokens, _ = _sample(x.expand(rows, 300), u)
    p = torch.softmax(x[0].double(), 0)
    n = torch.bincount(torch.tensor(tokens), minlength=300).double()
    assert ((n - rows * p).abs() <= 1.0 + 1e-6).all()  # evenly spaced numbers: within one
    _check(x.expand(64, 300).contiguous(), _uniforms(64, 4))


def test_edges_of_the_settings(gpu):
    x = _logits(1, 777, 5, F32)
    inf, nan = math.inf, math.nan
    rows = [  # u, temperature, top_k, top_p, min_p
        (0.5, 0.0, 0, 1.0, 0.0), (0.5, -1.0, 7, 0.5, 0.1), (0.5, nan, 0, 1.0, 0.0),
        (0.5, inf, 0, 1.0, 0.0), (0.5, 1e-30, 0, 1.0, 0.0), (0.9, 1e-3, 50, 0.9, 0.0),
        (0.5, 1.0, -3, 1.0, 0.0), (0.5, 1.0, 776, 1.0, 0.0), (0.5, 1.0, 777, 1.0, 0.0),
        (0.5, 1.0, 10000, 1.0, 0.0), (0.5, 1.0, 0, 0.0, 0.0), (0.5, 1.0, 0, -1.0, 0.0),
        (0.5, 1.0, 0, nan, 0.0), (0.5, 1.0, 0, 1.5, 0.0), (0.5, 1.0, 0, 1.0, 1.0),
        (0.5, 1.0, 0, 1.0, 2.0), (0.5, 1.0, 0, 1.0, nan), (0.5, 1.0, 0, 1.0, -0.5),
        (0.0, 1.0, 0, 1.0, 0.0), (nan, 1.0, 0, 1.0, 0.0), (-0.5, 1.0, 0, 1.0, 0.0),
        (1.0, 1.0, 0, 1.0, 0.0), (2.0, 1.0, 5, 1.0, 0.0), (0.99999994, 1.0, 0, 0.95, 0.0),
        (0.3, 100.0, 0, 0.9, 0.0), (0.3, 1e4, 20, 0.9, 0.5)]
    _check(x.expand(len(rows), 777).contiguous(), *(list(z) for z in zip(*rows)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties(gpu, dtype):
    """Equal logits: the lowest indices stay. 3000 ties are more than are compared each with each."""
    for vocab, at in ((50, [3, 9, 20, 21, 40]), (50257, list(range(100, 50257, 16)))):
        x = torch.full((1, vocab), -2.0)
        x[0, at] = 1.5
        x[0, at[1]] = 4.0
        x[0, 0], x[0, 1] = 0.0, -0.0  # equal
        x = x.to(dtype)
        rows = [(u, 1.0, k, p, m) for u in (0.0, 0.41, 0.77, 0.9999) for k, p, m in
                ((2, 1.0, 0.0), (4, 1.0, 0.0), (0, 0.31, 0.0), (len(at) + 1, 1.0, 0.0),
                 (len(at) + 1, 0.97, 0.0), (3, 0.6, 0.01), (0, 0.5, 0.0), (0, 1.0, 0.05))]
        _check(x.expand(len(rows), vocab).contiguous(), *(list(z) for z in zip(*rows)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_all_equal(gpu, dtype):
    rows = [(u, 1.0, k, p, 0.0) for u in (0.0, 0.3, 0.70001) for k, p in
            ((0, 1.0), (17, 1.0), (0, 0.25003), (5000, 0.50007))]
    _check(torch.full((len(rows), 50257), 2.5, dtype=dtype), *(list(z) for z in zip(*rows)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_special_logits(gpu, dtype):
    """NaN and -inf are never picked, +inf alone is where there is one, nothing left: -1."""
    inf, nan = math.inf, math.nan
    V, rows = 90, []
    for x in ([nan] * V, [-inf] * V, [nan, -inf] * (V // 2), [-inf] * 50 + [1.0] + [nan] * 39,
              [1.0] * 40 + [inf] + [2.0] * 48 + [inf], [inf] * V, [nan, inf, 3.0] * 30,
              [3.0e38] + [-3.0e38] * 88 + [1.0], [0.0] + [nan] * 80 + [-1e30] * 9):
        rows += [x] * 4
    u = [0.0, 0.4, 0.6, 0.999] * 9
    x = torch.tensor(rows).to(dtype)
    _check(x, u)
    _check(x, u, [0.8] * 36, [3] * 36, [0.9] * 36, [0.1] * 36)
    _check(x, u, [0.0] * 36)


def _edge(t, distance, place):
    per = np.float32(255) / (np.float32(31) * np.float32(t))
    assert np.float32(distance) * per == place and distance * float(per) < place


def _check_flat(t, row, ps, dtype):
    row = torch.tensor(row)[torch.randperm(len(row), generator=torch.Generator().manual_seed(5))]
    x = row.to(dtype).repeat(2 * len(ps), 1)
    _check(x, _uniforms(len(x), 6), [t] * len(x), [0] * len(ps) + [len(row) - 50] * len(ps), ps + ps)


@pytest.mark.parametrize("many", [300, 20000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_at_a_buckets_edge(gpu, dtype, many):
    """More candidates than the list holds, `many` of them at a logit whose distance from the largest, in
    buckets, rounds up to the edge of one: 11.75 * 255 / (31 t) in fp32 is 73 and exactly a little less."""
    t = 1.324016809463501
    _edge(t, 11.75, 73)
    row = [0.0] + [-11.75] * many + [-11.8125] * 12000 + [-20.0] * 100
    w = np.exp(np.array([0.0, -11.75, -11.8125]) / t) * [1, many, 12000]
    ends = np.cumsum(w) / w.sum()
    ps = [float(ends[i] + f * (ends[i + 1] - ends[i])) for i in range(2) for f in (0.3, 0.6, 0.9)]
    _check_flat(t, row, ps, dtype)


@pytest.mark.parametrize("many", [300, 4000])
def test_ties_at_the_edge_of_a_buckets_part(gpu, many):
    """The same at the edge of one of the 256 parts of a bucket of more than the list holds."""
    t = 1.1700055599212646
    _edge(t, 11.5, 80 + 218 / 256)
    row = [0.0] + [-11.4375] * 9000 + [-11.5] * many + [-11.5004] * 3000 + [-20.0] * 100
    w = np.exp(np.array([0.0, -11.4375, -11.5, -11.5004]) / t) * [1, 9000, many, 3000]
    ends = np.cumsum(w) / w.sum()
    ps = [float(ends[i] + f * (ends[i + 1] - ends[i])) for i in (1, 2) for f in (0.3, 0.6, 0.9)]
    _check_flat(t, row, ps, F32)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(gpu, dtype):
    """Rows at any pitch and alignment: slices of a wider buffer, one row expanded."""
    rows, vocab = 6, 1003
    wide = _logits(rows, vocab + 13, 9, dtype).cuda()
    u, k = _uniforms(rows, 10), [0, 1, 20, 0, 300, 2]
    for lo in range(5):
        x = wide[:, lo:lo + vocab]
        _check(x, u, None, k, [0.9] * rows)


def test_largest_vocabulary(gpu):
    x = _logits(3, sampling.MAX_VOCAB, 11, F32)
    _check(x, [0.2, 0.5, 0.9], [1.0, 0.9, 1.1], [0, 1000, 0], [1.0, 1.0, 0.9], [0.0, 0.0, 0.0])


def test_no_probabilities_and_graph(gpu):
    x = _logits(8, 5000, 12, F32).cuda()
    u = torch.tensor(_uniforms(8, 13)).cuda()
    p = torch.full((8,), 0.9, device="cuda")
    tokens, probs = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda")
    sampling.sample(tokens, None, x, u, top_p=p)
    got = torch.zeros_like(tokens)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        sampling.sample(got, probs, x, u, top_p=p)
    for i in range(3):
        sampling.sample(tokens, None, x, u, top_p=p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, tokens)
        x.add_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
        u.copy_(torch.tensor(_uniforms(8, 20 + i)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [16, 320])
def test_a_bucket_that_top_k_leaves_a_part_of(gpu, rows, dtype):
    """top-p ends in a bucket of which top-k left fewer elements than the candidate list holds and which has
    many more: the list is given up for the row itself. Every call and every row of equal settings answers the
    same."""
    x = torch.full((rows, 50257), 2.5)
    x[1::2, :300] = 3.0
    x, p = x.to(dtype), [0.50007] * rows
    u, k = [0.03, 0.37, 0.71, 0.96] * (rows // 4), [5000, 8000, 8000, 5000] * (rows // 4)
    if rows == 16:
        _check(x, u, None, k, p)
    x = x[:4].repeat(rows // 4, 1).cuda()
    first = _sample(x, u, None, k, p)
    for got in first:
        assert got == got[:4] * (rows // 4)
    for _ in range(3):
        assert _sample(x, u, None, k, p) == first


@pytest.mark.parametrize("dtype", [BF, F32])
def test_distances_that_overflow(gpu, dtype):
    """Logits further apart than fp32 reaches, at temperatures where the lower ones still weigh something: fewer
    candidates than the list holds, in a row that is longer. At an infinite temperature, and of the first 3000 of
    4000 equal ones, all weights are 2^44 units: sums and their parts by fp32 numbers are exact, also at a
    border. Otherwise sums of 4000 largest weights and more are off by 6000 * 2^-45 / 4000 and 1e-14 of
    themselves, less than 1e-12, and no decision lies as near a border."""
    x = torch.full((9000,), -math.inf)
    at = torch.randperm(9000, generator=torch.Generator().manual_seed(7))
    x[at[:4000]], x[at[4000:6000]] = 2.0e38, -2.0e38
    inf = math.inf
    rows = [(u, t, k, p, 0.0) for u in (0.2, 0.6, 0.99) for t in (1.0e38, inf)
            for k, p in ((5000, 1.0), (5000, 0.93), (0, 0.95), (6000, 1.0), (3000, 1.0), (0, 1.0))]
    x = x.to(dtype).repeat(len(rows), 1)
    tokens, probs = _sample(x, *(list(z) for z in zip(*rows)))
    for r, (u, t, k, p, _) in enumerate(rows):
        want, prob, margin = S.sample(x[r].float().numpy(), np.float32(u), t, k, p)
        assert margin >= 1e-12 or t == inf or k == 3000
        assert tokens[r] == want and abs(probs[r] - prob) <= 2.0 ** -23 * prob, r


@pytest.mark.parametrize("vocab", [40, 5000, 9001])
def test_uniforms_far_outside(gpu, vocab):
    """What is outside [0, 1) counts as the nearest end, however far: above, the last token that stayed."""
    x, u = _logits(1, vocab, 21, F32), [1.0, 2.0, 1e10, 3.0e38, math.inf, -1e-30, -3.0e38, -math.inf]
    for k, p in ((0, 1.0), (30, 1.0), (0, 0.99), (3000, 0.9999)):
        tokens, probs = _sample(x.expand(8, vocab).contiguous(), u, None, [k] * 8, [p] * 8)
        for i in range(8):
            want, prob, _ = S.sample(x[0].numpy(), np.float32(min(max(u[i], 0.0), 1.0)), 1.0, k, p)
            assert tokens[i] == want and abs(probs[i] - prob) <= 2.0 ** -23 * prob, (k, p, u[i])
