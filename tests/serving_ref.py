"""CPU references of the rotary positions, the paged caches and the sampling, from their definitions, in
64 bits (the sampling's sums in extended precision), and the bounds of the kernels' roundings."""
import math

import numpy as np
import torch

F8 = torch.float64
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative to the value


# ------------------------------------------------------------------------ rotary positions

def rotate(x, pos, freqs, interleaved=False, magnitude=1.0, back=False):
    """x [..., D] with its first 2 * len(freqs) elements turned; pos broadcasts against x's rows."""
    x, half = x.to(F8), freqs.numel()
    angle = pos.to(F8)[..., None] * freqs.to(F8).cpu()
    c, s = torch.cos(angle), torch.sin(angle) * (-1.0 if back else 1.0)
    y = x.clone()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[..., a] = magnitude * (x[..., a] * c - x[..., b] * s)
    y[..., b] = magnitude * (x[..., a] * s + x[..., b] * c)
    return y


def rotate_bound(x, pos, freqs, dtype, interleaved=False, magnitude=1.0, back=False):
    """What rotate's fp32 form may be off: each pair's sines and cosines are good to 2^-21 (the angle's
    rounding to fp32 is pi 2^-24 at most, the library's functions 2 ulp, the magnitude one more) and the
    double product pos * f to 2^-51 of itself; two products and a sum, three half steps of fp32; and the
    result's rounding."""
    x, half = x.to(F8), freqs.numel()
    far = (pos.to(F8)[..., None] * freqs.to(F8).cpu()).abs() * 2.0 ** -51
    y = rotate(x, pos, freqs, interleaved, magnitude, back)
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    size = torch.zeros_like(x)
    pair = abs(magnitude) * (x[..., a].abs() + x[..., b].abs()) * (2.0 ** -21 + 3 * 2.0 ** -24 + far)
    size[..., a], size[..., b] = pair, pair
    return size + HALF[dtype] * y.abs() * (1.0 + 2.0 ** -8)


# ------------------------------------------------------------------------ paged caches

class Step:
    """A step over a paged cache on the CPU: random rows, pages in random order, and what each row sees."""

    def __init__(self, lens, counts, H, Hkv, D, page, dtype, seed, max_pages=None, pad=0, spare=2,
                 size=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.counts = list(lens), list(counts)
        self.H, self.Hkv, self.D, self.page, self.dtype = H, Hkv, D, page, dtype
        n = len(lens)
        used = [(max(x, 0) + page - 1) // page for x in lens]
        self.max_pages = max_pages or max(1, *used)
        used = [min(u, self.max_pages) for u in used]
        self.n_pages = sum(used) + spare
        order = torch.randperm(self.n_pages, generator=gen).tolist()
        self.table = torch.full((n, self.max_pages), -1, dtype=torch.int32)
        for s, u in enumerate(used):
            for j in range(u):
                self.table[s, j] = order.pop()
        self.starts = [0]
        for c in counts:
            self.starts.append(self.starts[-1] + c)
        self.rows = self.starts[-1] + pad

        def normal(*shape):
            return (torch.randn(shape, generator=gen) * size).to(dtype)
        self.k_pages = normal(self.n_pages, Hkv, page, D)
        self.v_pages = normal(self.n_pages, Hkv, page, D)
        self.q = normal(max(self.rows, 1), H, D)
        self.k, self.v = (normal(max(self.rows, 1), Hkv, D) for _ in range(2))

    def cuda(self, name):
        x = getattr(self, name)
        if isinstance(x, list):
            x = torch.tensor(x, dtype=torch.int32)
        return x.cuda()

    def place(self, s, j):
        """(page, slot) of token j, None where it has none."""
        p = int(self.table[s, j // self.page])
        return (p, j % self.page) if 0 <= p < self.n_pages else None

    def new_rows(self, max_rows=None):
        """(sequence, row, token) of every row that the step handles."""
        most = self.max_pages * self.page
        for s, c in enumerate(self.counts):
            length = min(max(self.lens[s], 0), most)
            for t in range(min(c, max_rows or c)):
                yield s, self.starts[s] + t, length - c + t

    def attention(self, scale, max_rows=None):
        """float64 output, and the bound of each element, for the rows in use; others NaN."""
        out = torch.full((self.rows, self.H, self.D), math.nan, dtype=F8)
        bound = torch.zeros_like(out)
        G, bf16 = self.H // self.Hkv, self.dtype == torch.bfloat16
        kp, vp = self.k_pages.to(F8), self.v_pages.to(F8)
        cache = {}
        for s, row, tok in self.new_rows(max_rows):
            if s not in cache:
                last = tok + self.counts[s]
                places = [(j, self.place(s, j)) for j in range(max(last, 0))]
                places = [(j, p) for j, p in places if p is not None]
                at = torch.tensor([j for j, _ in places], dtype=torch.long)
                pg = torch.tensor([p[0] for _, p in places], dtype=torch.long)
                sl = torch.tensor([p[1] for _, p in places], dtype=torch.long)
                cache[s] = at, kp[pg, :, sl], vp[pg, :, sl]      # [keys, Hkv, D]
            at, K, V = cache[s]
            n = int((at <= tok).sum())
            if n == 0:
                out[row] = 0.0
                continue
            q = self.q[row].to(F8).view(self.Hkv, G, self.D)
            x = torch.einsum("hgd,nhd->hgn", q, K[:n]) * scale
            w = torch.softmax(x, -1)
            o = torch.einsum("hgn,nhd->hgd", w, V[:n])
            A = torch.einsum("hgn,nhd->hgd", w, V[:n].abs())
            # sum |q k| |scale|: a score's products are summed in fp32 (fp32: six bf16 products each)
            mass = torch.einsum("hgd,nhd->hgn", q.abs(), K[:n].abs()).amax(-1, keepdim=True) * abs(scale)
            e = (self.D + 8) * 2.0 ** -24 * mass + 2.0 ** -21    # a weight's relative error
            b = A * (2 * e + (n + 8) * 2.0 ** -23)               # of numerator and sum, and their sums
            if bf16:
                b = b + 2.0 ** -8 * A                            # weights rounded to bf16
            b = b + HALF[self.dtype] * (o.abs() + b)
            out[row], bound[row] = o.reshape(self.H, self.D), b.reshape(self.H, self.D)
        return out, bound


# ------------------------------------------------------------------------ sampling

LD = np.longdouble


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability, margin) for one row (numpy float32): margin is the distance of the decisions
    to their borders, relative to the weights' sum."""
    x = np.asarray(logits, np.float32)
    ok = x > -np.inf  # (NaN: False)
    if not ok.any():
        return -1, 0.0, 1.0
    top = x[ok].max()
    if np.isinf(top):
        ok &= x == top
    at = np.flatnonzero(ok)
    if not temperature > 0 or min_p > 1:
        return int(at[np.argmax(x[at])]), 1.0, 1.0
    d = np.zeros(len(at), LD) if np.isinf(top) else (x[at].astype(LD) - LD(top))
    w = np.exp(d / LD(np.float32(temperature)))
    order = np.argsort(-d, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    margin = 1.0
    if top_p < 1:
        c = np.cumsum(w[order])
        target = LD(np.float32(max(top_p, 0.0))) * c[-1]
        n = min(int(np.searchsorted(c, target)) + 1, len(order))
        near = np.abs(c - target) / c[-1]
        margin = min(margin, float(near[near > 1e-15].min(initial=1.0)))
        order = order[:n]
    if min_p > 0:
        keep = w[order] >= LD(np.float32(min_p))
        keep[0] = True
        margin = min(margin, float(np.abs(w[order] - LD(np.float32(min_p)))[1:].min(initial=1.0)))
        order = order[keep]
    order = np.sort(order)
    c = np.cumsum(w[order])
    u = LD(min(max(float(u), 0.0), 1.0)) if u == u else LD(0)
    target = u * c[-1]
    j = min(int(np.searchsorted(c, target, side="right")), len(order) - 1)
    if u > 0:
        margin = min(margin, float((np.abs(c[:-1] - target) / c[-1]).min(initial=1.0)))
    return int(at[order[j]]), float(w[order[j]] / c[-1]), margin
