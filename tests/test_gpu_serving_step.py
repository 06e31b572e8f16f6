"""GPU tests of the serving operators as a server runs them together: prompts enter in chunks beside
sequences that decode, every step rotates and appends, attends and picks; against one pass over
each whole sequence in 64 bits; and a decode step captured into a graph."""
import math

import pytest
import torch

from dadgpt_amd import paged as P
from dadgpt_amd import rope as R
from dadgpt_amd import sampling as Z
from tests import serving_ref as S

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
H, HKV, D, PAGE, VOCAB = 4, 2, 64, 16, 200
WIDTH = (H + 2 * HKV) * D


class Server:
    """One layer over a vocabulary: token -> fused projection row (a table), attention, logits."""

    def __init__(self, n_seq, max_pages, dtype, seed):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.n_seq = dtype, n_seq
        self.rows = torch.randn((VOCAB, WIDTH), generator=gen).to(dtype).cuda()
        self.head = (torch.randn((H * D, VOCAB), generator=gen) * 0.2).to(dtype).cuda()
        self.freqs = R.rope_frequencies(D, 10000.0, "parts", 4.0, 64)
        self.magnitude = R.rope_magnitude(4.0)
        self.k, self.v = P.paged_cache(n_seq * max_pages + 3, HKV, PAGE, D, dtype)
        order = torch.randperm(n_seq * max_pages + 3, generator=gen)[:n_seq * max_pages]
        self.table = order.view(n_seq, max_pages).to(torch.int32).cuda()

    def step(self, tokens, starts, lens, max_rows, u, last, buffers=None):
        """tokens [rows] on the device; last: the rows whose logits count."""
        rows = tokens.numel()
        b = buffers or {}
        x = self.rows[tokens].view(rows, H + 2 * HKV, D)
        q = b.get("q", torch.empty((rows, H, D), dtype=self.dtype, device="cuda"))
        P.paged_append(self.k, self.v, q, x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], self.table, starts,
                       lens, max_rows, self.freqs, False, self.magnitude)
        if "ws" not in b:
            b["ws"] = P.paged_workspace(q, self.k, self.table, max_rows)
        P.paged_attention(q, q, self.k, self.v, self.table, starts, lens, max_rows, 1 / math.sqrt(D),
                          b["ws"])
        logits = (q[last].reshape(len(last), H * D) @ self.head).float()
        picked = torch.empty(len(last), dtype=torch.int32, device="cuda")
        Z.sample(picked, None, logits, u, None, None, torch.full((len(last),), 0.9, device="cuda"))
        return picked, logits, q

    def whole(self, tokens):
        """Attention of every row of one sequence, float64, on the CPU."""
        x = self.rows[torch.tensor(tokens)].cpu().view(-1, H + 2 * HKV, D)
        pos = torch.arange(len(tokens))[:, None]
        f = self.freqs.cpu()
        # the rotated rows are rounded to the cache's type, as the append does
        q, k = (S.rotate(t, pos, f, False, self.magnitude).to(self.dtype).double()
                for t in (x[:, :H], x[:, H:H + HKV]))
        v = x[:, H + HKV:].double()
        q = q.view(-1, HKV, H // HKV, D)
        s = torch.einsum("ihgd,jhd->hgij", q, k) / math.sqrt(D)
        hidden = torch.ones(s.shape[-2:], dtype=torch.bool).triu(1)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        return torch.einsum("hgij,jhd->ihgd", p, v).reshape(-1, H, D)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_chunks_and_tokens_together(gpu, dtype):
    """Three prompts of unlike lengths enter in chunks of up to 24 while the others already decode."""
    sv = Server(3, 8, dtype, 1)
    gen = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in (70, 5, 33)]
    seqs, done, outs = [list(p) for p in prompts], [0, 0, 0], [[], [], []]
    u = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(12):
        counts = [min(24, len(s) - d) for s, d in zip(seqs, done)]
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        tokens = [t for s, d, c in zip(seqs, done, counts) for t in s[d:d + c]]
        done = [d + c for d, c in zip(done, counts)]
        last = [starts[i + 1] - 1 for i in range(3)]
        picked, _, q = sv.step(torch.tensor(tokens, device="cuda"), _int(starts), _int(done), 24,
                               torch.rand(3, device="cuda", generator=u), last)
        for i in range(3):
            outs[i].append(q[starts[i]:starts[i + 1]].double().cpu())
            if done[i] == len(seqs[i]):
                seqs[i].append(int(picked[i]))
                assert 0 <= seqs[i][-1] < VOCAB
    for i in range(3):
        got, want = torch.cat(outs[i]), sv.whole(seqs[i][:done[i]])
        # A rotated element may round to the other side of a half step: q and k then differ by 2^-8 (bf16),
        # a score by 2 * 2^-8 of its 64 products at most (|q||k| / 8, below 25 here), so a weight by
        # e^0.2; on top the kernel's own roundings. In norm, over sums of many: 2^-5 and 2^-17.
        err = (got - want).norm() / want.norm()
        assert err <= (2.0 ** -5 if dtype == BF else 2.0 ** -17), err


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_decode_step(gpu, dtype):
    """Append, attention and pick in one graph, replayed against the eager step over the same state."""
    n = 4
    sv, eager = Server(n, 40, dtype, 5), Server(n, 40, dtype, 5)
    starts = _int(list(range(n + 1)))
    lens = _int([300, 1, 17, 600])
    for s in (sv, eager):
        gen = torch.Generator(device="cuda").manual_seed(6)
        s.k.copy_(torch.randn(s.k.shape, generator=gen, device="cuda"))
        s.v.copy_(torch.randn(s.v.shape, generator=gen, device="cuda"))
    row = torch.randn((n, H + 2 * HKV, D), device="cuda").to(dtype)
    q = torch.empty((n, H, D), dtype=dtype, device="cuda")
    ws = P.paged_workspace(q, sv.k, sv.table, 1)
    logits = torch.empty((n, VOCAB), device="cuda")
    u, p = torch.rand(n, device="cuda"), torch.full((n,), 0.8, device="cuda")
    picked, probs = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")

    def step(s, q, picked, probs):
        P.paged_append(s.k, s.v, q, row[:, :H], row[:, H:H + HKV], row[:, H + HKV:], s.table, starts,
                       lens, 1, s.freqs, True, 1.1)
        P.paged_attention(q, q, s.k, s.v, s.table, starts, lens, 1, 0.125, ws)
        logits.copy_(q.reshape(n, H * D)[:, :VOCAB])
        Z.sample(picked, probs, logits, u, top_p=p)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step(sv, q, picked, probs)
    for i in range(4):
        lens.add_(1)
        row.copy_(torch.randn(row.shape, device="cuda"))
        u.copy_(torch.rand(n, device="cuda"))
        graph.replay()
        q2, picked2, probs2 = torch.empty_like(q), torch.zeros_like(picked), torch.zeros_like(probs)
        step(eager, q2, picked2, probs2)
        torch.cuda.synchronize()
        assert torch.equal(q, q2) and torch.equal(picked, picked2) and torch.equal(probs, probs2), i
        assert torch.equal(sv.k, eager.k) and torch.equal(sv.v, eager.v)
