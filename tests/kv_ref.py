"""CPU references of the bounded caches, from their definitions: e4m3 rounding by the table of its
values, the 8-bit append, attention over rows in float64, and eviction by sorting."""
import math

import torch

_CODES = torch.arange(256, dtype=torch.uint8)
# The finite non-negative e4m3 values, ascending (codes 0 .. 126; 127 is NaN).
TABLE = _CODES[:127].view(torch.float8_e4m3fn).double()


def e4m3(x):
    """Codes (uint8) of float64 x: the nearest value, ties to the even code; NaN for what is not
    finite. |x| <= 448."""
    a = x.abs().clamp(max=448.0)
    a = torch.where(torch.isfinite(x), a, 0.0)
    hi = torch.searchsorted(TABLE, a).clamp(max=126)       # first value >= a
    lo = (hi - 1).clamp(min=0)
    up = (TABLE[hi] - a) - (a - TABLE[lo])                 # < 0: the upper one is nearer
    code = torch.where(up < 0, hi, lo)
    code = torch.where(up == 0, torch.where(hi % 2 == 0, hi, lo), code)
    code = torch.where(a == TABLE[hi], hi, code)
    code = code + torch.where(torch.signbit(x), 128, 0)
    return torch.where(torch.isfinite(x), code, 127).to(torch.uint8)


def values(codes):
    """float64 values of e4m3 codes (uint8)."""
    return codes.view(torch.float8_e4m3fn).double()


def scale_of(amax: float) -> float:
    """The least 2^e >= 2^-100 with amax <= 448 * 2^e."""
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scale, x, lens, counts, block):
    """Appends x [n, H, rows, D] (CPU, any float) to codes uint8 [n, H, L, D] and scale, in place."""
    n, H, rows, D = x.shape
    L = codes.shape[2]
    for s in range(n):
        at = min(max(int(lens[s]), 0), L)
        end = min(L, at + min(max(int(counts[s]), 0), rows))
        for b in range(at // block, (end - 1) // block + 1 if end > at else 0):
            lo, hi = max(at, b * block), min(end, (b + 1) * block)
            for h in range(H):
                new = x[s, h, lo - at:hi - at].double()
                fin = new[torch.isfinite(new)].abs()
                to = scale_of(fin.max().item() if fin.numel() else 0.0)
                if b * block < at:
                    was = scale[s, h, b].item()
                    if was >= to:
                        to = was
                    else:
                        held = codes[s, h, b * block:at]
                        codes[s, h, b * block:at] = e4m3(values(held) * (was / to))
                codes[s, h, lo:hi] = e4m3(new / to)
                scale[s, h, b] = to


def same_codes(a, b):
    """Equal codes, NaN codes of either sign alike."""
    nan_a, nan_b = (a & 127) == 127, (b & 127) == 127
    return bool((nan_a == nan_b).all() and ((a == b) | nan_a).all())


def decode(q, k, v, lens, scale, window=0, sinks=0, out_half=2.0 ** -24):
    """float64 out [n, H, D], its bound, and probabilities [n, H, L] of one query per (sequence,
    head) over float64 k, v [n, H, L, D]. The bound: fp32 score sums (72 steps of 2^-24 of the
    absolute terms, own and the normaliser's), a few fp32 roundings of the exponent and of each
    product, fp32 sums over the keys (one addition in eight in sequence), and half a step of the
    output."""
    n, H, L, D = k.shape
    out = torch.zeros((n, H, D), dtype=torch.float64, device=k.device)
    bound, probs = torch.zeros_like(out), torch.zeros((n, H, L), dtype=torch.float64, device=k.device)
    e_probs = torch.zeros_like(probs)
    for i in range(n):
        end = min(max(int(lens[i]), 0), L)
        j = torch.arange(end, device=k.device)
        if window:
            j = j[(j >= end - window) | (j < sinks)]
        if len(j) == 0:
            continue
        kk, vv, qq = k[i][:, j], v[i][:, j], q[i].double()[:, None]
        s = (kk * qq).sum(-1) * scale
        e = (kk.abs() * qq.abs()).sum(-1) * abs(scale) * 72 * 2.0 ** -24 + s.abs() * 2.0 ** -22
        p = torch.softmax(s, -1)
        rel = 2 * e.amax(-1, keepdim=True) + 2.0 ** -19 + len(j) / 8 * 2.0 ** -24
        out[i] = (p[..., None] * vv).sum(1)
        bound[i] = rel * (p[..., None] * vv.abs()).sum(1) + out_half * out[i].abs()
        probs[i][:, j] = p
        e_probs[i][:, j] = p * rel
    return out, bound, probs, e_probs


def evict(weights, L, budget, sinks, recent):
    """Kept rows of one (sequence, head) with `L` rows and weights [>= L]."""
    if L <= budget:
        return list(range(L))
    first, last = min(sinks, L), max(min(sinks, L), L - recent)
    w = [(-math.inf if math.isnan(x) else x) for x in weights[first:last].tolist()]
    nan = [math.isnan(x) for x in weights[first:last].tolist()]
    order = sorted(range(first, last), key=lambda i: (nan[i - first], -w[i - first], i))
    most = budget - first - (L - last)
    return sorted(list(range(first)) + order[:most] + list(range(last, L)))
