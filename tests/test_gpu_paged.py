"""GPU tests of the paged caches: append (with rotary positions) and attention over pages, against
references in 64 bits (serving_ref) with bounds counted from their roundings."""
import math

import pytest
import torch

from dadgpt_amd import paged as P
from dadgpt_amd import rope as R
from tests import serving_ref as S

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _attend(st, max_rows=None, scale=None, workspace="own", out=None, q=None):
    scale = 1.0 / math.sqrt(st.D) if scale is None else scale
    q = st.cuda("q") if q is None else q
    out = torch.full_like(q, 7.0) if out is None else out
    kp, vp, table = (st.cuda(x) for x in ("k_pages", "v_pages", "table"))
    max_rows = max_rows or max(1, *st.counts)
    ws = P.paged_workspace(q, kp, table, max_rows) if isinstance(workspace, str) else workspace
    P.paged_attention(out, q, kp, vp, table, st.cuda("starts"), st.cuda("lens"), max_rows, scale, ws)
    torch.cuda.synchronize()
    if ws is not None:  # the counters are back at zero
        assert int(ws[:4 * len(st.counts) * st.Hkv].max()) == 0
    return out


def _check(st, out, max_rows=None, scale=None):
    scale = 1.0 / math.sqrt(st.D) if scale is None else scale
    want, bound = st.attention(scale, max_rows)
    used = ~torch.isnan(want)
    got = out.cpu().double()[:st.rows]
    assert (got[~used] == 7.0).all()  # rows that are no one's are left as they were
    err = (got - want).abs()
    assert (err[used] <= bound[used]).all(), float((err[used] / bound[used].clamp(min=1e-30)).max())


SHAPES = [  # lens, counts, H, Hkv, D, page
    ([1], [1], 1, 1, 32, 16),
    ([5, 17, 64, 65, 300], [1, 1, 1, 1, 1], 4, 4, 64, 16),
    ([5, 17, 64, 65, 300], [1, 1, 1, 1, 1], 6, 2, 64, 32),
    ([1, 16, 33, 700], [1, 1, 1, 1], 8, 1, 32, 16),
    ([40, 100, 7], [40, 3, 0], 2, 2, 64, 32),
    ([129, 64, 65], [129, 33, 65], 3, 3, 64, 64),
    ([500, 90, 260], [31, 32, 33], 4, 2, 32, 128),
    ([777, 200], [200, 133], 8, 2, 32, 16),
    ([600, 2000, 1], [64, 130, 1], 4, 4, 64, 16),
    ([1500], [257], 12, 4, 64, 64),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{s[1]}-{s[2]}-{s[3]}-{s[4]}-{s[5]}")
def test_attention(gpu, shape, dtype):
    st = S.Step(*shape, dtype, seed=1, pad=3)
    _check(st, _attend(st))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hkv,G,D,len_", [(2, 1, 64, 4000), (1, 3, 64, 5000), (2, 4, 32, 3000),
                                          (1, 16, 64, 2100), (1, 130, 32, 900)])
def test_long_caches_split(gpu, dtype, Hkv, G, D, len_):
    """Few rows over long caches: chunks of keys, merged by the last workgroup to arrive; and the same
    again into a workspace that other shapes used."""
    st = S.Step([len_, 1, 300], [1, 1, 1], G * Hkv, Hkv, D, 16, dtype, seed=2)
    out = _attend(st)
    _check(st, out)
    big = S.Step([len_, 1, 300, 40], [5, 1, 1, 2], G * Hkv, Hkv, D, 16, dtype, seed=3)
    kp, table, q = big.cuda("k_pages"), big.cuda("table"), big.cuda("q")
    ws = P.paged_workspace(q, kp, table, 5)
    _check(big, _attend(big, workspace=ws))
    for _ in range(3):
        assert torch.equal(_attend(st, workspace=ws), out)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_workspace_of_prompts_and_tokens(gpu, dtype):
    """One workspace for a step of prompts' chunks and a step of single tokens in turn, whose partials are
    fewer and larger than those of the tokens: each gets the bits it gets with one of its own. The caches are
    long; their pages are shared, as prefixes are."""
    n, Hkv, D, page, max_pages = 64, 4, 64, 128, 128
    gen = torch.Generator().manual_seed(9)
    kp, vp = (torch.randn((24, Hkv, page, D), generator=gen).to(dtype).cuda() for _ in range(2))
    table = torch.randint(0, 24, (n, max_pages), generator=gen).int().cuda()
    lens = torch.randint(9000, page * max_pages, (n,), generator=gen).int().cuda()
    q = torch.randn((n * 48, Hkv, D), generator=gen).to(dtype).cuda()
    ws = P.paged_workspace(q, kp, table, 48)

    def step(rows, ws):
        start = (torch.arange(n + 1) * rows).int().cuda()
        out = torch.empty_like(q[:n * rows])
        P.paged_attention(out, q[:n * rows], kp, vp, table, start, lens, rows, 0.125,
                          torch.zeros_like(ws) if ws is own else ws)
        torch.cuda.synchronize()
        return out
    own = ws.clone()
    assert P.paged_workspace(q[:n], kp, table, 1).numel() < ws.numel()
    want = {rows: step(rows, own) for rows in (48, 1, 20)}
    for rows in (48, 1, 20, 1, 48):
        assert torch.equal(step(rows, ws), want[rows]), rows


@pytest.mark.parametrize("dtype", [BF, F32])
def test_chunk_equals_one_token_at_a_time(gpu, dtype):
    """A chunk's rows are the rows of its tokens alone, up to both forms' bounds."""
    st = S.Step([150, 70], [50, 70], 4, 2, 64, 32, dtype, seed=4)
    whole = _attend(st).cpu()
    _, bound = st.attention(1.0 / math.sqrt(64))
    for s, row, tok in list(st.new_rows())[::7]:
        one = S.Step([tok + 1], [1], 4, 2, 64, 32, dtype, seed=4)
        one.k_pages, one.v_pages, one.n_pages = st.k_pages, st.v_pages, st.n_pages
        one.table, one.max_pages, one.q = st.table[s:s + 1], st.max_pages, st.q[row:row + 1]
        got = _attend(one).cpu()[0].double()
        assert ((got - whole[row].double()).abs() <= 2 * bound[row]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_missing_pages_and_empty_rows(gpu, dtype):
    """Tokens in pages that do not exist are not seen; a row that sees nothing gets zeros; counts of
    zero, lengths of zero, counts above the length, lengths above the table."""
    st = S.Step([200, 90, 0, 3, 64, 500], [30, 90, 0, 5, 1, 1], 4, 2, 64, 16, dtype, seed=5, pad=2,
                max_pages=20)
    st.table[0, 2], st.table[0, 5], st.table[1, :] = -1, st.n_pages, 1 << 30
    st.table[4, :4] = torch.tensor([-5, st.n_pages + 3, -1, -1])
    st.table[5, :20] = torch.arange(20) % st.n_pages  # lens 500 > 20 * 16: clamped
    out = _attend(st)
    _check(st, out)
    assert (out[st.starts[1]:st.starts[2]] == 0).all() and (out[st.starts[4]] == 0).all()
    assert (out[st.starts[3]:st.starts[3] + 2] == 0).all()  # two rows before token 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_left_out(gpu, dtype):
    """What a sequence has beyond max_rows is left as it was; the rows before keep their tokens."""
    st = S.Step([100, 60], [40, 8], 2, 2, 64, 16, dtype, seed=6)
    out = _attend(st, max_rows=16)
    _check(st, out, max_rows=16)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(gpu, dtype, scale):
    st = S.Step([100, 33], [20, 1], 4, 2, 32, 16, dtype, seed=7)
    _check(st, _attend(st, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_unseen_values_do_not_matter(gpu, dtype):
    """NaN in slots past the length, in pages that no table names and in rows behind the last: never
    read. NaN in a key: its row is NaN, rows before it and other sequences are not."""
    st = S.Step([37, 100], [5, 1], 2, 1, 64, 16, dtype, seed=8, pad=4)
    want = _attend(st)
    used = torch.zeros(st.n_pages, st.page, dtype=torch.bool)
    for s, n in enumerate(st.lens):
        for j in range(n):
            used[st.place(s, j)] = True
    for x in (st.k_pages, st.v_pages):
        x.transpose(1, 2)[~used] = math.nan
    st.q[st.starts[-1]:] = math.nan
    assert torch.equal(_attend(st), want)
    page, slot = st.place(0, 35)  # seen by the last two of the first sequence's five rows
    st.k_pages[page, :, slot] = math.nan
    got = _attend(st)
    assert torch.isnan(got[3:5]).all()
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[5:], want[5:])


def test_minus_infinite_scores_bf16(gpu):
    """Keys that score -inf weigh nothing; rows with no other key get zeros."""
    st = S.Step([130, 40], [3, 1], 2, 2, 64, 16, BF, seed=9)
    st.q[:, :, 0] = 1.0
    for s, n, skip in ((0, 130, 64), (1, 40, 40)):
        for j in range(skip):
            page, slot = st.place(s, j)
            st.k_pages[page, :, slot, 0] = -math.inf
    out = _attend(st)
    assert (out[3] == 0).all()
    less = S.Step([130, 40], [3, 1], 2, 2, 64, 16, BF, seed=9)
    less.q, less.k_pages, less.v_pages = st.q, st.k_pages, st.v_pages
    less.table[0, :4] = -1  # tokens 0 .. 63 are not there
    _check_rows, bound = less.attention(1.0 / 8)
    got = out.cpu().double()[:3]
    assert ((got - _check_rows[:3]).abs() <= bound[:3]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_in_place_and_shared_pages(gpu, dtype):
    """Queries out of a fused projection, output over them, and sequences that share their first pages."""
    st = S.Step([80, 96, 50], [16, 1, 30], 6, 2, 64, 16, dtype, seed=10)
    st.table[1, :2], st.table[2, :2] = st.table[0, :2], st.table[0, :2]
    want = _attend(st)
    _check(st, want)
    fused = torch.zeros((st.rows, 6 + 4, 64), dtype=dtype, device="cuda")
    fused[:, :6] = st.cuda("q")
    q = fused[:, :6]
    assert torch.equal(_attend(st, q=q), want)
    assert torch.equal(_attend(st, q=q, out=q), want)
    assert (fused[:, 6:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_sequences(gpu, dtype):
    """More sequences than the lanes of a wave, most without rows."""
    n = 150
    counts = [0] * n
    for s, c in ((3, 40), (63, 1), (64, 200), (65, 2), (128, 129), (149, 7)):
        counts[s] = c
    lens = [c + (7 * s) % 50 for s, c in enumerate(counts)]
    st = S.Step(lens, counts, 4, 4, 32, 16, dtype, seed=11, pad=1)
    _check(st, _attend(st))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_sequences_in_chunks(gpu, dtype):
    """More sequences than the lanes of a wave, some of whose caches are cut and some not."""
    n = 100
    counts = [0] * n
    for s, c in ((0, 150), (1, 33), (62, 140), (63, 2), (64, 1), (65, 300), (98, 129), (99, 64)):
        counts[s] = c
    lens = [c + (0, 3000, 100, 5000)[s % 4] if c else 5 for s, c in enumerate(counts)]
    st = S.Step(lens, counts, 2, 2, 32, 64, dtype, seed=13)
    _check(st, _attend(st))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129])
def test_rows_of_every_kernel(gpu, dtype, rows):
    """The numbers of rows at which another kernel or another share of the waves takes over, over caches of
    one and of several chunks; D alternates."""
    D = 64 if rows % 2 else 32
    for group in (1, rows) if rows < 64 else (1,):
        count = rows // group
        st = S.Step([count + 1400, count, count + 40], [count] * 3, group, 1, D, 16, dtype, seed=14)
        _check(st, _attend(st))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_far_pages(gpu, dtype):
    """Pages behind the element 2^32 of a cache: the bits of the same pages at its start, read and written."""
    n_pages, Hkv, page, D = (1 << 32) // (8 * 128 * 64) + 24, 8, 128, 64
    far = n_pages - 20
    kp, vp = (torch.empty((n_pages, Hkv, page, D), dtype=dtype, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(15)
    for x in (kp, vp):
        x[:20] = torch.randn((20, Hkv, page, D), generator=gen).to(dtype)
    lens, freqs = [1200, 1100], R.rope_frequencies(64)
    table = torch.arange(20).view(2, 10).int()
    for rows in (1, 3, 40):  # of a KV head: the three kernels
        counts = torch.tensor([0, rows, 2 * rows]).int().cuda()
        new = torch.randn((2 * rows, 3 * Hkv, D), generator=gen).to(dtype).cuda()
        outs = []
        for start in (0, far):
            if start:
                kp[far:], vp[far:] = kp[:20], vp[:20]
            at = (table + start).cuda()
            q, k, v = new.clone().split(Hkv, 1)
            length = torch.tensor(lens).int().cuda()
            P.paged_append(kp, vp, q, q, k, v, at, counts, length, rows, freqs, False)
            out = torch.empty((2 * rows, Hkv, D), dtype=dtype, device="cuda")
            P.paged_attention(out, q, kp, vp, at, counts, length, rows, 0.125,
                              P.paged_workspace(q, kp, at, rows))
            outs.append(out)
        torch.cuda.synchronize()
        assert torch.equal(*outs), rows
        assert torch.equal(kp[far:], kp[:20]) and torch.equal(vp[far:], vp[:20])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_graph_of_a_prompts_step_replays(gpu, dtype):
    """The same graph for chunks that are cut and that are not, and for sequences that have none."""
    st = S.Step([4000, 200, 90], [100, 60, 90], 2, 1, 64, 32, dtype, seed=16, max_pages=125)
    q, kp, vp, table, starts, lens = (st.cuda(x) for x in ("q", "k_pages", "v_pages", "table", "starts",
                                                           "lens"))
    ws, out = P.paged_workspace(q, kp, table, 100), torch.zeros_like(q)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        P.paged_attention(out, q, kp, vp, table, starts, lens, 100, 0.125, ws)
    for i, (now, rows) in enumerate((([4000, 200, 90], [100, 60, 90]), ([300, 200, 4000], [50, 100, 100]),
                                     ([4000, 0, 1], [99, 0, 1]), ([4000, 200, 90], [100, 60, 90]))):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        starts.copy_(torch.tensor([0, rows[0], rows[0] + rows[1], sum(rows)], dtype=torch.int32))
        table[:, 63:].copy_(table[:, :62])  # (a place for every token)
        graph.replay()
        got = out.clone()
        want = torch.zeros_like(q)
        P.paged_attention(want, q, kp, vp, table, starts, lens, 100, 0.125, ws)
        torch.cuda.synchronize()
        assert torch.equal(got[:sum(rows)], want[:sum(rows)]), i


@pytest.mark.parametrize("dtype", [BF, F32])
def test_graph_replays(gpu, dtype):
    """A captured step follows lengths, rows and pages in device memory."""
    st = S.Step([900, 40, 300], [1, 1, 1], 4, 2, 64, 16, dtype, seed=12, max_pages=64)
    q, kp, vp, table, starts, lens = (st.cuda(x) for x in ("q", "k_pages", "v_pages", "table", "starts",
                                                           "lens"))
    ws, out = P.paged_workspace(q, kp, table, 1), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        P.paged_attention(out, q, kp, vp, table, starts, lens, 1, 0.125, ws)
    for i, now in enumerate(([900, 40, 300], [17, 1, 288], [880, 33, 5])):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        q.add_(0.25)
        graph.replay()
        want = torch.zeros_like(q)
        P.paged_attention(want, q, kp, vp, table, starts, lens, 1, 0.125, ws)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


# ------------------------------------------------------------------------ append

def _append(st, max_rows=None, freqs=None, interleaved=False, magnitude=1.0, fused=True, with_q=True):
    H, Hkv, D = st.H, st.Hkv, st.D
    if fused:
        x = torch.cat((st.q, st.k, st.v), 1).cuda()
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    else:
        q, k, v = (st.cuda(x) for x in "qkv")
    kp, vp = st.cuda("k_pages"), st.cuda("v_pages")
    qo = torch.full((st.rows, H, D), 7.0, dtype=st.dtype, device="cuda")
    P.paged_append(kp, vp, qo if with_q else None, q if with_q else None, k, v, st.cuda("table"),
                   st.cuda("starts"), st.cuda("lens"), max_rows or max(1, *st.counts),
                   None if freqs is None else freqs.cuda(), interleaved, magnitude)
    torch.cuda.synchronize()
    return qo, kp, vp


APPENDS = [  # lens, counts, H, Hkv, D, page, rot, interleaved
    ([1], [1], 1, 1, 32, 16, 8, False),
    ([1, 16, 17, 300], [1, 1, 1, 1], 12, 12, 64, 16, 64, False),
    ([40, 100, 7, 5], [40, 3, 0, 5], 6, 2, 64, 32, 48, True),
    ([500, 129], [31, 129], 4, 1, 32, 128, 0, False),
    ([700, 20], [640, 20], 12, 4, 64, 64, 32, True),
    ([700, 20], [640, 20], 3, 3, 32, 16, 24, False),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c)))
def test_append(gpu, case, dtype):
    lens, counts, H, Hkv, D, page, rot, inter = case
    st = S.Step(lens, counts, H, Hkv, D, page, dtype, seed=20, pad=2)
    freqs = R.rope_frequencies(rot, device="cpu") if rot else None
    qo, kp, vp = (x.cpu() for x in _append(st, None, freqs, inter, 1.2 if rot else 1.0))
    want_k, want_v = st.k_pages.clone().double(), st.v_pages.clone()
    bound_k = torch.zeros_like(want_k)
    none = torch.zeros(0, dtype=torch.float64)
    f, mag = (none, 1.0) if freqs is None else (freqs, 1.2)
    seen = torch.zeros(st.rows, dtype=torch.bool)
    for s, row, tok in st.new_rows():
        pos, (page_, slot) = torch.tensor([tok]), st.place(s, tok)
        seen[row] = True
        want_k[page_, :, slot] = S.rotate(st.k[row], pos, f, inter, mag)
        bound_k[page_, :, slot] = S.rotate_bound(st.k[row], pos, f, dtype, inter, mag)
        want_v[page_, :, slot] = st.v[row]
        d = (qo[row].double() - S.rotate(st.q[row], pos, f, inter, mag)).abs()
        assert (d <= S.rotate_bound(st.q[row], pos, f, dtype, inter, mag)).all()
    assert torch.equal(vp, want_v)
    assert ((kp.double() - want_k).abs() <= bound_k).all()
    assert (qo[~seen] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_edges(gpu, dtype):
    """Pages that do not exist, counts above the length, rows past max_rows, k and v alone, tensors of
    their own."""
    st = S.Step([64, 3, 30], [40, 5, 20], 4, 2, 64, 16, dtype, seed=21)
    st.table[0, 2] = -1
    st.table[2, 0] = st.n_pages
    qo, kp, vp = _append(st, max_rows=18, fused=False)
    want_k, want_v = st.k_pages.clone(), st.v_pages.clone()
    want_q = torch.full_like(st.q, 7.0)
    for s, row, tok in st.new_rows(18):
        if tok < 0:
            continue
        want_q[row] = st.q[row]
        if st.place(s, tok) is not None:
            page, slot = st.place(s, tok)
            want_k[page, :, slot], want_v[page, :, slot] = st.k[row], st.v[row]
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)
    assert torch.equal(qo.cpu(), want_q)
    qo, kp2, vp2 = _append(st, max_rows=18, with_q=False)
    assert torch.equal(kp2, kp) and torch.equal(vp2, vp) and (qo == 7.0).all()


def test_append_in_place_query(gpu):
    st = S.Step([20, 50], [20, 1], 4, 2, 64, 16, BF, seed=22)
    freqs = R.rope_frequencies(64)
    qo, kp, vp = _append(st, freqs=freqs)
    x = torch.cat((st.q, st.k, st.v), 1).cuda()
    kp2, vp2 = st.cuda("k_pages"), st.cuda("v_pages")
    P.paged_append(kp2, vp2, x[:, :4], x[:, :4], x[:, 4:6], x[:, 6:], st.cuda("table"),
                   st.cuda("starts"), st.cuda("lens"), 20, freqs)
    assert torch.equal(x[:, :4], qo) and torch.equal(kp2, kp) and torch.equal(vp2, vp)
    assert torch.equal(x[:, 4:], torch.cat((st.k, st.v), 1).cuda())


def _without(st, skip):
    """The same step, without the tokens 0 .. skip[s] - 1 (whole pages) of sequence s."""
    less = S.Step(st.lens, st.counts, st.H, st.Hkv, st.D, st.page, st.dtype, seed=0)
    less.q, less.k_pages, less.v_pages, less.n_pages = st.q, st.k_pages, st.v_pages, st.n_pages
    less.table = st.table.clone()
    for s, n in enumerate(skip):
        less.table[s, :n // st.page] = -1
    return less


# rows of a KV head: the kernels of a few rows, of up to 32, and the tiles, whose waves share 32 rows by four
# and by two
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 4, 5, 20, 40])
@pytest.mark.parametrize("how", ["infinite", "overflow", "far overflow"])
def test_scores_of_minus_infinity(gpu, dtype, rows, how):
    """Keys that score -inf (an infinite element, or finite ones whose product overflows) weigh nothing,
    wherever the first of them are; a row that has no other key gets zeros. The scores of a far overflow differ
    by enough that parts of a product overflow to either side."""
    st = S.Step([900, 192 + rows, 130], [rows, rows, 1], 2, 2, 64, 64, dtype, seed=30)
    skip = [704, 128, 192]  # of 900 (into the second chunk), of some, of all of the third's 130
    big = {"infinite": (1.0, -math.inf), "overflow": (2.0 ** 70, -1.234 * 2.0 ** 70),
           "far overflow": (1.377 * 2.0 ** 100, -1.234 * 2.0 ** 100)}[how]
    st.q[:, :, 5] = big[0]
    st.k_pages[..., 5] = 0.0  # (of what is seen: the large element of q must not matter)
    for s, n in enumerate(skip):
        for j in range(min(n, st.lens[s])):
            page, slot = st.place(s, j)
            st.k_pages[page, :, slot, 5] = big[1]
    out = _attend(st)
    assert (out[-1] == 0).all()
    want, bound = _without(st, skip).attention(1.0 / 8)
    got = out.cpu().double()[:-1]
    assert ((got - want[:-1]).abs() <= bound[:-1]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 4, 5, 20, 40])
def test_infinite_values(gpu, dtype, rows):
    """An infinite value makes its column of the rows that see it infinite, two of unlike signs or a NaN make it
    NaN; other columns are what they were."""
    st = S.Step([700 + rows, 60 + rows], [rows, rows], 2, 1, 64, 16, dtype, seed=31)
    before = _attend(st).cpu()
    for s, j, col, x in ((0, 3, 7, math.inf), (0, 600, 40, -math.inf), (0, 5, 41, math.inf),
                         (0, 650, 41, -math.inf), (0, 9, 42, math.nan), (1, 50, 0, -math.inf)):
        page, slot = st.place(s, j)
        st.v_pages[page, :, slot, col] = x
    got = _attend(st).cpu()
    a, b = got[:rows], got[rows:]
    assert (a[..., 7] == math.inf).all() and (a[..., 40] == -math.inf).all()
    assert torch.isnan(a[..., 41:43]).all() and (b[..., 0] == -math.inf).all()
    left = [c for c in range(64) if c not in (7, 40, 41, 42)]
    want, bound = st.attention(1.0 / 8)
    assert torch.equal(b[..., 1:], before[rows:, :, 1:])
    assert ((a.double() - want[:rows]).abs() <= bound[:rows])[..., left].all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [65535, (65535 - 769 - 60000) * 128])
def test_largest_grids(gpu, dtype, rows):
    """A token of each of 65535 sequences, and as many tiles as a grid has room for, over shared pages: some of
    the first, last and other sequences against the same sequence in a step of its own."""
    gen = torch.Generator().manual_seed(32)
    n, page, D, max_pages = (65535 if rows == 65535 else 60000), 16, 32, 64
    kp, vp = (torch.randn((90, 2, page, D), generator=gen).to(dtype).cuda() for _ in range(2))
    table = torch.randint(0, 90, (n, max_pages), generator=gen).int().cuda()
    counts = torch.ones(n, dtype=torch.long)
    more = rows - n
    at = torch.randperm(n - 1, generator=gen)[:more // 999]
    counts[at] += 999
    counts[-1] += more - 999 * len(at)  # (the last one too)
    assert int(counts.sum()) == rows and int(counts.max()) <= 1000
    lens = torch.minimum(counts + torch.randint(0, 1000, (n,), generator=gen), torch.tensor(1024))
    starts = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0)))
    q = torch.randn((rows, 2, D), generator=gen).to(dtype).cuda()
    out, most = torch.full_like(q, 7.0), int(counts.max())
    P.paged_attention(out, q, kp, vp, table, starts.int().cuda(), lens.int().cuda(), most, 0.25,
                      P.paged_workspace(q, kp, table, most))
    torch.cuda.synchronize()
    for s in [0, 1, n // 2, n - 2, n - 1, *(at[:3].tolist())]:
        a, b = int(starts[s]), int(starts[s + 1])
        st = S.Step([int(lens[s])], [b - a], 2, 2, D, page, dtype, seed=0)
        st.q, st.k_pages, st.v_pages, st.n_pages = q[a:b].cpu(), kp.cpu(), vp.cpu(), 90
        st.table, st.max_pages = table[s:s + 1].cpu(), max_pages
        some = torch.arange(0, b - a, max(1, (b - a) // 20))
        want, bound = st.attention(0.25)
        assert ((out[a:b].cpu().double() - want).abs() <= bound)[some].all(), s


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [([9000, 3000, 8500], [1, 1, 1], 4, 4), ([9000, 700, 4000], [2, 1, 0], 2, 1),
                                   ([9000, 8000], [8, 3], 2, 2), ([9000, 200], [300, 200], 2, 2)],
                         ids=["one row", "four rows", "eight rows", "tiles"])
def test_all_counters_return_to_zero(gpu, dtype, shape):
    """Counters lie in front and partials against the end: in a workspace of twice the size everything in the
    front half is zero after a call."""
    lens, counts, H, Hkv = shape
    st = S.Step(lens, counts, H, Hkv, 64, 128, dtype, seed=33)
    q, kp, table = st.cuda("q"), st.cuda("k_pages"), st.cuda("table")
    size = P.paged_workspace(q, kp, table, max(counts)).numel()
    ws = torch.zeros(2 * size, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    for _ in range(2):
        P.paged_attention(out, q, kp, st.cuda("v_pages"), table, st.cuda("starts"), st.cuda("lens"),
                          max(counts), 0.125, ws)
        torch.cuda.synchronize()
        assert int(ws[:size].max()) == 0 and int(ws[size:].max()) > 0
    _check(st, out)


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 16, 17, 32])
@pytest.mark.parametrize("D", [32, 64])
def test_weights_of_a_few_bf16_rows(gpu, rows, D):
    """Steps of up to 32 rows of a KV head round nothing to bf16 but the result: weights are fp32, or two bf16
    numbers (the first cut off, which leaves less than 2^-7 of the weight, that rounded by 2^-8 of itself, and
    2^-20 added), and what fp32 arithmetic leaves is the bound of the fp32 step."""
    st = S.Step([2000 + rows, rows, 300 + rows], [rows] * 3, 1, 1, D, 16, BF, seed=34)
    out = _attend(st).cpu().double()
    st.dtype = F32
    want, bound = st.attention(D ** -0.5)
    st.v_pages = st.v_pages.abs()
    bound = bound + (2.0 ** -15 + 2.0 ** -20) * st.attention(D ** -0.5)[0]
    err = (out - want).abs() - (bound + 2.0 ** -8 * (want.abs() + bound))
    assert (err <= 0).all(), float(err.max())
