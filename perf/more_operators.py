"""The calls of a serving step over paged caches (rotary positions, append, attention, sampling), and
the rotary positions of a training step, in two forms: elementary torch operations (``own`` false),
and this framework's kernels (``own`` true).

Kinds of case:

- ``rope``: q and k of a training step rotated by their positions, and the gradients of the rotated
  rotated back. Pair i of a head's first `rot` elements turns by position * freqs[i]; the pairs are
  (i, i + rot / 2), or (2i, 2i + 1) where interleaved; a magnitude multiplies the rotated elements.
- ``append``: the new tokens of ragged sequences out of a fused projection's rows: q and k rotated, k
  and v written into the pages that the block table names.
- ``attend``: new tokens against the pages: token t of a sequence's last `count` sees its keys up to
  its own. One token for each sequence is a decode step, hundreds a chunk of a prompt.
- ``sample``: a token for each row of logits from a given uniform number, with temperature, top-k,
  top-p and min-p for each row.

Queries, keys and values are N(0, 1); lengths are uniform; pages lie in the pool in random order.
Logits fall off with the logarithm of a random rank, as those of a language model do.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
BF16, F32 = "bf16", "f32"


def _rope(name, dtype, B, H, HK, S, D, rot, interleaved=False, factor=1.0, layout="tokens"):
    return {"name": name, "kind": "rope", "dtype": dtype, "B": B, "H": H, "HK": HK, "S": S, "D": D,
            "rot": rot, "interleaved": interleaved, "factor": factor, "layout": layout}


def _paged(name, kind, dtype, n, H, HK, D, page, max_len, max_rows, rows, pad=0, **more):
    return {"name": name, "kind": kind, "dtype": dtype, "n": n, "H": H, "HK": HK, "D": D,
            "page": page, "max_len": max_len, "max_rows": max_rows, "rows": rows, "pad": pad, **more}


def _sample(name, dtype, rows, vocab, mode):
    return {"name": name, "kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab,
            "mode": mode}


def listed():
    return [
        # the GPT-2 124M training layer (B16 H12 T1024 D64) on a fused QKV projection
        _rope("rope_train_gpt2_bf16", BF16, 16, 12, 12, 1024, 64, 64),
        # one long document in fp32 with shared KV heads, half of each head rotated, scaled for
        # eight times the context
        _rope("rope_train_long_f32", F32, 1, 8, 2, 32768, 64, 32, True, 8.0, "heads"),
        # 16 prompts of 512 tokens on average enter the cache
        _paged("append_prompts_bf16", "append", BF16, 16, 12, 12, 64, 32, 1024, 1024, 8192,
               rot=64, interleaved=False),
        # the append of every decode step: one token for each of 32 sequences
        _paged("append_token_bf16", "append", BF16, 32, 12, 12, 64, 16, 1024, 1, 32,
               rot=64, interleaved=False),
        # a decode step of 32 ragged sequences: the smallest attention, where latency counts
        _paged("attend_token_ragged_bf16", "attend", BF16, 32, 12, 12, 64, 16, 1024, 1, 32),
        # long contexts of a few users, three query heads to a KV head: bound by reading the pages
        _paged("attend_token_long_bf16", "attend", BF16, 8, 12, 4, 64, 64, 32768, 1, 8),
        # chunks of 8 prompts under a budget of 2048 tokens, behind up to 7680 cached ones
        _paged("attend_chunk_bf16", "attend", BF16, 8, 12, 12, 64, 32, 8192, 512, 2048),
        # a mixed step: a chunk of one prompt beside 15 sequences of one token each
        _paged("attend_mixed_bf16", "attend", BF16, 16, 12, 12, 64, 16, 4096, 512, 527),
        # the reference's own precision at its smaller head, nothing a multiple of a tile
        _paged("attend_chunk_odd_f32", "attend", F32, 3, 8, 2, 32, 16, 777, 200, 333, 5),
        # the pick of a decode step: 32 rows of GPT-2's vocabulary, every row its own settings
        _sample("sample_step_f32", F32, 32, 50257, "mixed"),
        # one user, top-k: the smallest pick
        _sample("sample_one_f32", F32, 1, 50257, "top_k"),
        # many continuations at once, top-p, logits in bf16 (with many ties)
        _sample("sample_batch_bf16", BF16, 512, 50257, "top_p"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the ranges the listed ones stand for: sequences of 1 to 32768 tokens in
    training, caches of 1 to 32768, chunks of 1 to 1024 tokens, batches of 1 to 64, 1 to 8 query
    heads to a KV head, pages of 16 to 128 tokens, vocabularies of 100 to 131072."""
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "sample"])
    dtype = rng.choice([BF16, BF16, F32])
    if kind == "sample":
        vocab = _log_int(rng, 100, 131072)
        rows = min(_log_int(rng, 1, 512), 512 * 50257 // vocab)
        return _sample("", dtype, rows, vocab, rng.choice(["mixed", "top_k", "top_p", "plain"]))
    HK, G = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 8])
    if HK * G > 32:
        G = 1
    H, D = HK * G, rng.choice([32, 64, 64])
    rot = rng.choice([D, D, D // 2, 8, 24])
    if kind == "rope":
        S = _log_int(rng, 1, 32768)
        B = _log_int(rng, 1, 32)
        while B > 1 and B * S * (H + HK) * D > 16 * 1024 * 24 * 64:
            B //= 2
        while S * (H + HK) * D * B > 32768 * 10 * 64:
            S = S // 2 + 1
        return _rope("", dtype, B, H, HK, S, D, rot, rng.random() < 0.5,
                     rng.choice([1.0, 1.0, 4.0, 16.0]), rng.choice(["tokens", "heads"]))
    n, page = _log_int(rng, 1, 64), rng.choice([16, 32, 64, 128])
    max_len = _log_int(rng, 1, 32768)
    max_rows = rng.choice([1, min(max_len, _log_int(rng, 1, 1024))])
    most = 8 * 12 * 512 * 8192 if kind == "attend" else 1 << 40
    while n > 1 and (n * HK * max_len * D > 8 * 4 * 32768 * 64 or n * H * max_rows * max_len > most):
        n //= 2
    while H * max_rows * max_len > most // 2 or max_rows * max_len * H * D > 3 << 31:
        max_rows = (max_rows + 1) // 2
    rows = rng.randint(n, n * max_rows)
    more = {} if kind == "attend" else {"rot": rot, "interleaved": rng.random() < 0.5}
    return _paged("", kind, dtype, n, H, HK, D, page, max_len, max_rows, rows,
                  rng.choice([0, 0, 3, 64]), **more)


# ------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float32 if case["dtype"] == F32 else torch.bfloat16


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def _frequencies(rot, factor, trained=4096):
    """Radians a position for each pair: 10000^(-2i / rot); scaled, those that turn less than once
    over the trained context by 1 / factor, those that turn 32 times or more not, a ramp between."""
    f = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    if factor != 1.0:
        keep = ((trained * f / (2.0 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f.to(DEVICE)


def _counts(rng, n, most, total):
    """n counts of 1 to `most` with the given sum, skewed as arrivals are."""
    counts, left = [1] * n, total - n
    order = list(range(n))
    rng.shuffle(order)
    for i, s in enumerate(order):
        others = (n - 1 - i) * (most - 1)
        lo, hi = max(0, left - others), min(most - 1, left)
        take = hi if i == n - 1 else min(hi, max(lo, int(2.0 * rng.random() * left / (n - i))))
        counts[s] += take
        left -= take
    return counts


def _prepare_rope(case, gen, s):
    B, H, HK, S, D, dt = *(case[x] for x in ("B", "H", "HK", "S", "D")), _dtype(case)
    s["freqs"] = _frequencies(case["rot"], case["factor"])
    s["magnitude"] = 1.0 + 0.1 * math.log(case["factor"])
    if case["layout"] == "tokens":  # q, k and v of every token side by side
        for x, y in (("qkv", "rotated"), ("grad", "dqkv")):
            s[x] = _normal(gen, (B, S, H + 2 * HK, D), dt)
            s[y] = torch.zeros((B, S, H + HK, D), dtype=dt, device=DEVICE)
    else:
        for x, y in (("qkv", "rotated"), ("grad", "dqkv")):
            s[x] = _normal(gen, (B, H + HK, S, D), dt)
            s[y] = torch.zeros_like(s[x])


def _prepare_sample(case, gen, s, rng):
    rows, vocab, dt, mode = case["rows"], case["vocab"], _dtype(case), case["mode"]
    rank = torch.rand((rows, vocab), generator=gen, device=DEVICE).mul_(vocab).add_(1.0)
    noise = torch.randn((rows, vocab), generator=gen, device=DEVICE)
    s["logits"] = (8.0 - 1.2 * torch.log(rank) + noise.mul_(0.7)).to(dt)
    s["uniforms"] = torch.rand((rows,), generator=gen, device=DEVICE)
    t = [rng.uniform(0.6, 1.3) for _ in range(rows)]
    k, p, m = [0] * rows, [1.0] * rows, [0.0] * rows
    if mode in ("mixed", "top_k"):
        k = [rng.choice([0, 1, 40, 200, 5000]) if mode == "mixed" else 40 for _ in range(rows)]
    if mode in ("mixed", "top_p"):
        p = [rng.choice([1.0, 0.95, rng.uniform(0.3, 1.0)]) if mode == "mixed"
             else rng.uniform(0.8, 0.99) for _ in range(rows)]
    if mode == "mixed":
        t = [rng.choice([0.0, x, x, x, x, x]) for x in t]
        m = [rng.choice([0.0, 0.0, rng.uniform(0.001, 0.2)]) for _ in range(rows)]
    for name, x in (("temperature", t), ("top_p", p), ("min_p", m)):
        s[name] = torch.tensor(x, dtype=torch.float32).to(DEVICE)
    s["top_k"] = _int32(k)
    s["tokens"] = torch.zeros((rows,), dtype=torch.int32, device=DEVICE)
    s["probs"] = torch.zeros((rows,), dtype=torch.float32, device=DEVICE)


def prepare(case, seed):
    """Inputs, and the buffers that a program keeps: pages, tables, outputs, gradients."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": case}
    if case["kind"] == "rope":
        _prepare_rope(case, gen, s)
        return s
    if case["kind"] == "sample":
        _prepare_sample(case, gen, s, rng)
        return s
    n, H, HK, D, page, dt = *(case[x] for x in ("n", "H", "HK", "D", "page")), _dtype(case)
    max_pages = (case["max_len"] + page - 1) // page
    counts = _counts(rng, n, case["max_rows"], case["rows"])
    lens = [c + rng.randint(0, case["max_len"] - case["max_rows"]) for c in counts]
    pool = list(range(n * max_pages))
    rng.shuffle(pool)
    table = torch.full((n, max_pages), -1, dtype=torch.int32)
    for i, length in enumerate(lens):
        used = (length + page - 1) // page
        table[i, :used] = torch.tensor(pool[i * max_pages:i * max_pages + used])
    s["table"], s["lens"] = table.to(DEVICE), _int32(lens)
    s["row_start"] = _int32(np.concatenate(([0], np.cumsum(counts))).tolist())
    for x in ("k_pages", "v_pages"):
        s[x] = _normal(gen, (n * max_pages, HK, page, D), dt)
    total = case["rows"] + case["pad"]
    if case["kind"] == "append":
        s["qkv"] = _normal(gen, (total, H + 2 * HK, D), dt)
        s["freqs"] = _frequencies(case["rot"], 1.0)
    else:
        s["q"] = _normal(gen, (total, H, D), dt)
    s["out"] = torch.zeros((total, H, D), dtype=dt, device=DEVICE)
    return s


# ------------------------------------------------------------------------------ the plain forms

def _rotate(x, angle, magnitude, interleaved, back=False):
    """x [..., D] fp32 with its first 2 * angle.shape[-1] elements turned by angle (float64)."""
    half = angle.shape[-1]
    c = (torch.cos(angle) * magnitude).float()
    s = (torch.sin(angle) * (-magnitude if back else magnitude)).float()
    r = x[..., :2 * half]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    turned = (a * c - b * s, a * s + b * c)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rope(s, case):
    S, heads, dt = case["S"], case["H"] + case["HK"], _dtype(case)
    angle = torch.arange(S, device=DEVICE, dtype=torch.float64)[:, None] * s["freqs"]
    if case["layout"] == "tokens":
        x, g, angle = s["qkv"][:, :, :heads], s["grad"][:, :, :heads], angle[:, None]
    else:
        x, g = s["qkv"], s["grad"]
    y = _rotate(x.float(), angle, s["magnitude"], case["interleaved"])
    d = _rotate(g.float(), angle, s["magnitude"], case["interleaved"], True)
    return {"rotated": y.to(dt), "dqkv": d.to(dt)}


def _places(s, case):
    """Of every row in use: its sequence and its position there; and which rows are in use."""
    row = torch.arange(case["rows"], device=DEVICE)
    start, lens = s["row_start"].long(), s["lens"].long()
    seq = torch.searchsorted(start, row, right=True) - 1
    return seq, lens[seq] - start[seq + 1] + row


def _plain_append(s, case):
    H, HK, dt, page, rows = case["H"], case["HK"], _dtype(case), case["page"], case["rows"]
    seq, pos = _places(s, case)
    x = s["qkv"][:rows].float()
    angle = (pos.double()[:, None] * s["freqs"])[:, None]
    turned = _rotate(x[:, :H + HK], angle, 1.0, case["interleaved"])
    at = s["table"].long()[seq, pos // page]
    s["k_pages"][at, :, pos % page] = turned[:, H:].to(dt)
    s["v_pages"][at, :, pos % page] = x[:, H + HK:].to(dt)
    s["out"][:rows] = turned[:, :H].to(dt)
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s, case):
    n, H, HK, D, R, dt = *(case[x] for x in ("n", "H", "HK", "D", "max_rows")), _dtype(case)
    G, page, L = H // HK, case["page"], s["table"].shape[1] * case["page"]
    start, lens = s["row_start"].long(), s["lens"].long()
    counts = start[1:] - start[:-1]
    t = torch.arange(R, device=DEVICE)
    row = (start[:-1, None] + t).clamp(max=case["rows"] - 1)                     # [n, R]
    q = s["q"][row].float().view(n, R, HK, G, D).permute(0, 2, 3, 1, 4).reshape(n * HK, G * R, D)
    at = s["table"].long().clamp(min=0)
    k, v = (s[x][at].float().transpose(1, 2).reshape(n * HK, L, D) for x in ("k_pages", "v_pages"))
    last = (lens - counts)[:, None] + t                                         # [n, R]
    hidden = torch.arange(L, device=DEVICE) > last[..., None]                   # [n, R, L]
    p = torch.bmm(q, k.transpose(1, 2)).mul_(1.0 / math.sqrt(D))
    p.view(n, HK * G, R, L).masked_fill_(hidden[:, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    v = v.masked_fill_((torch.arange(L, device=DEVICE) >= lens[:, None])[:, None, :, None]
                       .expand(n, HK, L, 1).reshape(n * HK, L, 1), 0.0)
    o = torch.bmm(p, v).view(n, H, R, D).transpose(1, 2)                        # [n, R, H, D]
    seq, pos = _places(s, case)
    s["out"][:case["rows"]] = o[seq, pos - (lens - counts)[seq]].to(dt)
    return {"out": s["out"]}


def _plain_sample(s, case):
    x, vocab = s["logits"].double(), case["vocab"]
    T, p = s["temperature"].double()[:, None], s["top_p"].double()[:, None]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    k = torch.where(T > 0, k, 1)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(vocab, device=DEVICE)
    w = torch.where(rank < k, w, 0.0)
    upto = torch.cumsum(w, -1)
    before = torch.nn.functional.pad(upto[:, :-1], (1, 0))
    keep = (p >= 1.0) | (before < p * upto[:, -1:])
    keep = (keep & (w >= s["min_p"].double()[:, None]) & (rank < k)) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = torch.cumsum(kept, -1)
    target = s["uniforms"].double()[:, None] * upto[:, -1:]
    token = (upto <= target).sum(-1)
    token = torch.minimum(token, torch.where(kept > 0, rank, 0).amax(-1))
    prob = kept.gather(1, token[:, None]) / upto[:, -1:]
    return {"tokens": token.to(torch.int32), "probs": prob[:, 0].float()}


def _run_plain(s, case):
    kind = case["kind"]
    if kind == "rope":
        return _plain_rope(s, case)
    if kind == "append":
        return _plain_append(s, case)
    if kind == "attend":
        return _plain_attend(s, case)
    return _plain_sample(s, case)


# ------------------------------------------------------------------------------ the framework's

def _own_rope(s, case):
    from dadgpt_amd import rope as R
    H, heads = case["H"], case["H"] + case["HK"]
    tokens = case["layout"] == "tokens"

    def parts(x):  # q and k as [B, heads, S, D] views
        x = x.transpose(1, 2) if tokens else x
        return x[:, :H], x[:, H:heads]
    (q, k), (qo, ko), (gq, gk), (dq, dk) = (parts(s[x]) for x in ("qkv", "rotated", "grad", "dqkv"))
    R.rope(qo, ko, q, k, s["freqs"], None, case["interleaved"], s["magnitude"])
    R.rope_backward(dq, dk, gq, gk, s["freqs"], None, case["interleaved"], s["magnitude"])
    return {"rotated": s["rotated"], "dqkv": s["dqkv"]}


def _own_append(s, case):
    from dadgpt_amd import paged as P
    H, HK, qkv = case["H"], case["HK"], s["qkv"]
    P.paged_append(s["k_pages"], s["v_pages"], s["out"], qkv[:, :H], qkv[:, H:H + HK],
                   qkv[:, H + HK:], s["table"], s["row_start"], s["lens"], case["max_rows"],
                   s["freqs"], case["interleaved"])
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attend(s, case):
    from dadgpt_amd import paged as P
    if "workspace" not in s:  # one for the step's shape, kept as a serving loop keeps it
        s["workspace"] = P.paged_workspace(s["q"], s["k_pages"], s["table"], case["max_rows"])
    P.paged_attention(s["out"], s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"],
                      s["lens"], case["max_rows"], 1.0 / math.sqrt(case["D"]), s["workspace"])
    return {"out": s["out"]}


def _own_sample(s, case):
    from dadgpt_amd import sampling
    sampling.sample(s["tokens"], s["probs"], s["logits"], s["uniforms"], s["temperature"],
                    s["top_k"], s["top_p"], s["min_p"])
    return {"tokens": s["tokens"], "probs": s["probs"]}


def _run_own(s, case):
    kind = case["kind"]
    if kind == "rope":
        return _own_rope(s, case)
    if kind == "append":
        return _own_append(s, case)
    if kind == "attend":
        return _own_attend(s, case)
    return _own_sample(s, case)


def run(state):
    case = state["case"]
    return _run_own(state, case) if own else _run_plain(state, case)


# ------------------------------------------------------------------------------ the floor

def work(case):
    size, kind = 4 if case["dtype"] == F32 else 2, case["kind"]
    if kind == "sample":
        elements = case["rows"] * case["vocab"]
        return {"bytes": elements * size + 28 * case["rows"], "flops": elements}
    H, HK, D = case["H"], case["HK"], case["D"]
    if kind == "rope":  # q and k in and out, gradients in and out
        elements = case["B"] * case["S"] * (H + HK) * D
        rotated = elements // D * case["rot"]
        return {"bytes": 4 * elements * size + 8 * case["rot"], "flops": 6 * rotated}
    n, rows, page = case["n"], case["rows"], case["page"]
    past = (case["max_len"] - case["max_rows"]) / 2
    pages = n * (past / page + 1) + rows / page
    io = 2 * rows * H * D * size + 4 * pages + 8 * n
    if kind == "append":
        return {"bytes": io + 4 * rows * HK * D * size + 4 * case["rot"],
                "flops": 3 * rows * (H + HK) * case["rot"]}
    keys, mean = n * past + rows, rows / n
    return {"bytes": io + 2 * keys * HK * D * size,
            "flops": 4 * D * H * rows * (past + (mean + 1) / 2)}


# ------------------------------------------------------------------------------ float64

def _turn(x, pos, freqs, magnitude, interleaved):
    """x [..., D] with pair i times magnitude e^(i pos freqs[i]), as complex numbers; pos [...]."""
    half = freqs.numel()
    x = x.to(torch.float64)
    r = x[..., :2 * half]
    if interleaved:
        z = torch.view_as_complex(r.unflatten(-1, (half, 2)).contiguous())
    else:
        z = torch.complex(r[..., :half].contiguous(), r[..., half:].contiguous())
    z = z * torch.polar(torch.full_like(freqs, magnitude).expand(*pos.shape, half).contiguous(),
                        pos.to(torch.float64)[..., None] * freqs)
    z = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((z, x[..., 2 * half:]), -1)


def _exact_rope(s, case):
    heads = case["H"] + case["HK"]
    pos = torch.arange(case["S"], device=DEVICE)
    if case["layout"] == "tokens":
        x, g, pos = s["qkv"][:, :, :heads], s["grad"][:, :, :heads], pos[None, :, None]
    else:
        x, g, pos = s["qkv"], s["grad"], pos[None, None, :]
    pos = pos.expand(x.shape[:-1])
    return {"rotated": _turn(x, pos, s["freqs"], s["magnitude"], case["interleaved"]),
            "dqkv": _turn(g, -pos, s["freqs"], s["magnitude"], case["interleaved"])}


def _exact_append(s, case):
    H, HK, page = case["H"], case["HK"], case["page"]
    k, v, q = (s[x].to(torch.float64) for x in ("k_pages", "v_pages", "out"))
    starts, table = s["row_start"].tolist(), s["table"].cpu()
    for i, length in enumerate(s["lens"].tolist()):
        a, b = starts[i], starts[i + 1]
        pos = torch.arange(length - (b - a), length)
        pages, slots = table[i, pos // page].long().to(DEVICE), (pos % page).to(DEVICE)
        x, pos = s["qkv"][a:b], pos.to(DEVICE)[:, None].expand(-1, H + HK)
        y = _turn(x[:, :H + HK], pos, s["freqs"], 1.0, case["interleaved"])
        q[a:b], k[pages, :, slots] = y[:, :H], y[:, H:]
        v[pages, :, slots] = x[:, H + HK:].to(torch.float64)
    return {"q": q, "k_pages": k, "v_pages": v}


def _exact_attend(s, case):
    H, HK, D, page = (case[x] for x in ("H", "HK", "D", "page"))
    out = s["out"].to(torch.float64)
    starts = s["row_start"].tolist()
    for i, length in enumerate(s["lens"].tolist()):
        a, b = starts[i], starts[i + 1]
        ids = s["table"][i, :(length + page - 1) // page].long()
        k, v = (s[x][ids].transpose(0, 1).reshape(HK, -1, D)[:, :length].to(torch.float64)
                for x in ("k_pages", "v_pages"))
        for r in range(a, b, 256):
            e = min(b, r + 256)
            seen = length - (b - a) + (e - a)  # keys that the last of these rows sees
            q = s["q"][r:e].to(torch.float64).view(e - r, HK, H // HK, D).permute(1, 2, 0, 3)
            x = torch.matmul(q, k[:, None, :seen].mT.contiguous()) / math.sqrt(D)
            late = torch.ones((e - r, seen), dtype=torch.bool, device=DEVICE).triu(
                seen - (e - r) + 1)
            P = torch.softmax(torch.where(late, -math.inf, x), -1)
            out[r:e] = torch.matmul(P, v[:, None, :seen]).permute(2, 0, 1, 3).reshape(e - r, H, D)
    return {"out": out}


def _exact_sample(s, case):
    """Row by row on the host, sums in extended precision."""
    logits = s["logits"].float().cpu().numpy().astype(np.longdouble)
    t, p, m, u = (s[x].cpu().numpy().astype(np.longdouble)
                  for x in ("temperature", "top_p", "min_p", "uniforms"))
    ks, tokens, probs = s["top_k"].tolist(), [], []
    for i, x in enumerate(logits):
        if not t[i] > 0:
            tokens.append(int(np.argmax(x)))
            probs.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        if ks[i] > 0:
            order = order[:ks[i]]
        w = np.exp((x[order] - x[order[0]]) / t[i])
        if p[i] < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p[i] * w.sum()))]
        w = w[:len(order)]
        order = np.sort(order[:max(1, int((w >= m[i]).sum()))])
        w = np.exp((x[order] - x.max()) / t[i])
        c = np.cumsum(w)
        j = min(int(np.searchsorted(c, u[i] * c[-1], side="right")), len(order) - 1)
        tokens.append(int(order[j]))
        probs.append(float(w[j] / c[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=DEVICE),
            "probs": torch.tensor(probs, dtype=torch.float64, device=DEVICE)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(s, case)
    if kind == "append":
        return _exact_append(s, case)
    if kind == "attend":
        return _exact_attend(s, case)
    return _exact_sample(s, case)
