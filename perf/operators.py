"""The calls that the bounded-attention and bounded-cache operators are timed on, each in two
forms: elementary torch operations in fp32 (``own`` false), and this framework's kernels
(``own`` true).

Kinds of case:

- ``window_train``: one layer's attention with a sliding window and sinks in a training step,
  forward and backward. Query i sees key j when j <= i and (j > i - window or j < sinks).
- ``window_decode``: one query token per sequence (the cache's last row) under the same mask,
  over ragged bf16 or fp32 caches.
- ``kv8_append``: new K and V rows into a cache held in e4m3 with a power-of-two scale for each
  block of tokens and head; a block that already has rows and needs a larger scale is re-rounded.
- ``kv8_decode``: one query token per sequence over such a cache, whole or windowed.
- ``weights_decode``: one query token per sequence; the probability of every key is added to
  that key's accumulated weight.
- ``evict``: each (sequence, head) keeps `budget` rows: its first `sinks`, its last `recent`, and
  those of the largest accumulated weight between, in order.

Queries, keys and values are N(0, 1); the keys and values of the 8-bit cache vary in size from
channel to channel, as projected keys do; lengths are uniform. Accumulated weights are those of a
skewed attention (a power of a uniform variable, many of them equal to the last bit: rounded to
1/64, so that ties are met).
"""
import math

import torch

own = False

DEVICE = "cuda"
BF16, F32 = "bf16", "f32"
E4M3 = torch.float8_e4m3fn


def _train(name, dtype, B, H, S, D, window, sinks, layout="heads"):
    return {"name": name, "kind": "window_train", "dtype": dtype, "B": B, "H": H, "S": S, "D": D,
            "window": window, "sinks": sinks, "layout": layout}


def _cache(name, kind, dtype, n, H, max_len, D, **more):
    return {"name": name, "kind": kind, "dtype": dtype, "n": n, "H": H, "max_len": max_len,
            "D": D, **more}


def listed():
    return [
        # the GPT-2 124M training layer (B16 H12 T1024 D64) with a window of a quarter of its
        # context, on the buffers of a fused QKV projection
        _train("window_train_gpt2_bf16", BF16, 16, 12, 1024, 64, 256, 4, layout="tokens"),
        # a long document at batch 1, the case the window is for
        _train("window_train_long_bf16", BF16, 1, 12, 8192, 64, 1024, 4),
        # the reference's own precision at its smaller head, nothing a multiple of a tile
        _train("window_train_odd_f32", F32, 3, 8, 777, 32, 100, 3),
        # serving 32 ragged sequences with a small window: the smallest call, all latency
        _cache("window_decode_ragged_bf16", "window_decode", BF16, 32, 12, 1024, 64,
               window=256, sinks=4),
        # long fp32 caches under a window of a few thousand keys
        _cache("window_decode_long_f32", "window_decode", F32, 8, 12, 16384, 64,
               window=4096, sinks=16),
        # a batch of 16 prompts of 1 to 1024 tokens quantised out of a fused QKV projection
        _cache("kv8_append_prompts", "kv8_append", BF16, 16, 12, 1024, 64, block=32, rows=1024,
               start=0),
        # the append of every decode step: one token for each of 32 ragged sequences
        _cache("kv8_append_token", "kv8_append", BF16, 32, 12, 1024, 64, block=32, rows=1,
               start=1023),
        # the ragged decode of 32 sequences over 8-bit caches
        _cache("kv8_decode_ragged", "kv8_decode", BF16, 32, 12, 1024, 64, block=32, window=0,
               sinks=0),
        # long contexts of a few users, bound by reading the caches
        _cache("kv8_decode_long", "kv8_decode", BF16, 8, 12, 32768, 64, block=64, window=0,
               sinks=0),
        # the ragged decode while weights are accumulated for a later eviction
        _cache("weights_decode_ragged_bf16", "weights_decode", BF16, 32, 12, 1024, 64),
        # the same over longer caches, where the weights need a second pass
        _cache("weights_decode_long_bf16", "weights_decode", BF16, 16, 12, 8192, 64),
        # 32 sequences of up to 2048 rows cut back to a budget of 512
        _cache("evict_bf16", "evict", BF16, 32, 12, 2048, 64, budget=512, sinks=4, recent=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the ranges the listed ones stand for: sequences of 16 to 8192 tokens
    (fp32 to 2048), caches of 1 to 32768 rows, batches of 1 to 64, windows from a few keys to the
    whole sequence, up to 64 sinks, blocks of 16 to 128 tokens. (A row that sees itself alone has
    gradients of zero for its query and key, and nothing but rounding to compare.)"""
    kind = rng.choice(["window_train", "window_train", "window_train", "window_decode",
                       "kv8_append", "kv8_decode", "weights_decode", "evict"])
    H = rng.choice([1, 3, 4, 8, 12])
    D = rng.choice([32, 64, 64])
    dtype = rng.choice([BF16, BF16, F32])
    if kind == "window_train":
        S = _log_int(rng, 16, 8192 if dtype == BF16 else 2048)
        B = _log_int(rng, 1, 16)
        most = 12 * 8192 ** 2 if dtype == BF16 else 24 * 2048 ** 2
        while B > 1 and B * H * S * S > most:
            B //= 2
        layout = rng.choice(["heads", "tokens"]) if dtype == BF16 else "heads"
        return _train("", dtype, B, H, S, D, _log_int(rng, 4, S),
                      rng.choice([0, 1, 4, _log_int(rng, 1, 64)]), layout)
    max_len = _log_int(rng, 1, 32768)
    n = _log_int(rng, 1, 64)
    while n > 1 and n * H * max_len * D > 6 * 12 * 32768 * 64:
        n //= 2
    if kind == "evict":
        max_len = min(max_len, 8192)
        sinks, recent = rng.choice([0, 1, 4, 16]), _log_int(rng, 1, max(1, max_len // 8))
        budget = sinks + recent + _log_int(rng, 1, max(1, max_len // 2))
        return _cache("", kind, dtype, n, H, max_len, D, budget=budget, sinks=sinks, recent=recent)
    if kind == "kv8_append":
        rows = rng.choice([1, 1, _log_int(rng, 1, min(max_len, 2048))])
        return _cache("", kind, dtype, n, H, max_len, D, block=rng.choice([16, 32, 64, 128]),
                      rows=rows, start=rng.randint(0, max_len - rows))
    c = _cache("", kind, dtype, n, H, max_len, D)
    if kind == "window_decode":
        c.update(window=_log_int(rng, 1, max_len), sinks=rng.choice([0, 1, 4, 64]))
    elif kind == "kv8_decode":
        window = rng.choice([0, _log_int(rng, 1, max_len)])
        c.update(block=rng.choice([16, 32, 64, 128]), window=window,
                 sinks=rng.choice([0, 1, 4, 64]) if window else 0)
    return c


# ------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float32 if case["dtype"] == F32 else torch.bfloat16


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _lens(seed, n, lo, hi):
    gen = torch.Generator().manual_seed(seed * 2 + 1)
    return torch.randint(lo, hi + 1, (n,), generator=gen).to(torch.int32).to(DEVICE)


def _channels(gen, n, H, D):
    """The size of each channel: e^N(0, 1/2)."""
    return torch.exp(0.5 * torch.randn((n, H, 1, D), generator=gen, device=DEVICE))


def _e4m3_cache(gen, case):
    """An 8-bit cache that appends have filled: values in every row, a scale in every block."""
    n, H, L, D, block = (case[x] for x in ("n", "H", "max_len", "D", "block"))
    blocks = (L + block - 1) // block
    amax = 16.0 * torch.rand((n, H, blocks), generator=gen, device=DEVICE) + 1e-3
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
    x = torch.randn((n, H, L, D), generator=gen, device=DEVICE).mul_(_channels(gen, n, H, D))
    row = torch.arange(L, device=DEVICE) // block
    x.mul_((amax / 8.0)[:, :, row, None]).clamp_(-1e4, 1e4)
    limit = (448.0 * scale)[:, :, row, None]
    x = torch.minimum(torch.maximum(x, -limit), limit).div_(scale[:, :, row, None])
    return x.to(E4M3), scale


def prepare(case, seed):
    """Inputs, and the buffers that a program keeps: caches, outputs, gradients."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dt, H, D = case["kind"], _dtype(case), case["H"], case["D"]
    s = {"case": case, "scale": 1.0 / math.sqrt(D)}
    if kind == "window_train":
        B, S = case["B"], case["S"]
        if case["layout"] == "tokens":
            s["qkv"] = _normal(gen, (B * S, 3 * H * D), dt)
            s["dout"] = _normal(gen, (B * S, H * D), dt)
            s["dqkv"] = torch.empty_like(s["qkv"])
        else:
            for x in ("q", "k", "v", "dout"):
                s[x] = _normal(gen, (B * H, S, D), dt)
            for x in ("dq", "dk", "dv"):
                s[x] = torch.empty_like(s["q"])
        s["out"] = torch.empty_like(s["dout"])
        s["lse"] = torch.empty((B * H, S), dtype=torch.float32, device=DEVICE)
        s["delta"] = torch.empty_like(s["lse"])
        return s
    n, L = case["n"], case["max_len"]
    if kind == "kv8_append":
        s["k8"], s["k_scale"] = _e4m3_cache(gen, case)
        s["v8"], s["v_scale"] = _e4m3_cache(gen, case)
        rows = case["rows"]
        # the projection's output for the new tokens: q, k and v of every head side by side
        qkv = torch.randn((n, rows, 3, H, D), generator=gen, device=DEVICE)
        s["qkv"] = (qkv * _channels(gen, 1, H, D)[:, None, :, 0]).to(dt)
        s["lens"] = _lens(seed, n, 0, case["start"])
        s["counts"] = _lens(seed + 1, n, 1, rows)
        return s
    s["lens"] = _lens(seed, n, 1, L)
    if kind == "evict":
        for x in ("k", "v"):
            s[x] = _normal(gen, (n, H, L, D), dt)
            s[x + "_out"] = torch.zeros((n, H, case["budget"], D), dtype=dt, device=DEVICE)
        w = torch.rand((n, H, L), generator=gen, device=DEVICE).pow_(6).mul_(64.0)
        s["weights"] = torch.round(w * 64.0) / 64.0
        s["weights_out"] = torch.zeros((n, H, case["budget"]), device=DEVICE)
        s["kept"] = torch.empty((n, H, case["budget"]), dtype=torch.int32, device=DEVICE)
        s["lens_out"] = torch.empty_like(s["lens"])
        return s
    s["q"] = _normal(gen, (n, H, D), dt)
    s["out"] = torch.empty_like(s["q"])
    if kind == "kv8_decode":
        s["k8"], s["k_scale"] = _e4m3_cache(gen, case)
        s["v8"], s["v_scale"] = _e4m3_cache(gen, case)
        return s
    s["k"] = _normal(gen, (n, H, L, D), dt)
    s["v"] = _normal(gen, (n, H, L, D), dt)
    if kind == "weights_decode":
        s["weights"] = torch.rand((n, H, L), generator=gen, device=DEVICE)
        s["weights_out"] = torch.empty_like(s["weights"])
    return s


# ------------------------------------------------------------------------------ the plain forms

def _heads(x, case):
    """[B*S, H*D] -> [B*H, S, D]."""
    B, H, S, D = (case[x] for x in ("B", "H", "S", "D"))
    return x.reshape(B, S, H, D).transpose(1, 2).reshape(B * H, S, D)


def _tokens(x, case):
    B, H, S, D = (case[x] for x in ("B", "H", "S", "D"))
    return x.view(B, H, S, D).transpose(1, 2).reshape(B * S, H * D)


def _plain_train(s, case):
    tokens, dt, scale = case["layout"] == "tokens", _dtype(case), s["scale"]
    d = case["H"] * case["D"]
    if tokens:
        q, k, v = (_heads(s["qkv"][:, i * d:(i + 1) * d].float(), case) for i in range(3))
        g = _heads(s["dout"].float(), case)
    else:
        q, k, v, g = (s[x].float() for x in ("q", "k", "v", "dout"))
    i = torch.arange(case["S"], device=DEVICE)
    back = i[:, None] - i[None, :]
    seen = (back >= 0) & ((back < case["window"]) | (i[None, :] < case["sinks"]))
    p = torch.bmm(q, k.transpose(1, 2)).mul_(scale).masked_fill_(~seen, float("-inf"))
    m = p.amax(-1, keepdim=True)
    p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + torch.log(l)).squeeze(-1)
    p.div_(l)
    out = torch.bmm(p, v)
    dv = torch.bmm(p.transpose(1, 2), g)
    ds = torch.bmm(g, v.transpose(1, 2)).sub_((g * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.bmm(ds, k), torch.bmm(ds.transpose(1, 2), q)
    if tokens:
        return {"out": _tokens(out, case).to(dt), "lse": lse,
                "dqkv": torch.cat([_tokens(x, case) for x in (dq, dk, dv)], 1).to(dt)}
    return {"out": out.to(dt), "lse": lse, "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


def _plain_decode(q, k, v, lens, scale, window, sinks):
    """out and the probabilities of one query per (sequence, head) over fp32 caches."""
    key = torch.arange(k.shape[2], device=DEVICE)
    end = lens[:, None]
    seen = key < end
    if window:
        seen = seen & ((key >= end - window) | (key < sinks))
    seen = seen[:, None, :]
    p = (k * q[:, :, None, :]).sum(-1).mul_(scale).masked_fill_(~seen, float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return (p[..., None] * v).sum(2), p


def _plain_append_one(x, codes, scale, lens, counts, block):
    """Appends x [n, H, rows, D] to one 8-bit cache, looking at the blocks that can be touched."""
    n, H, rows, D = x.shape
    L, blocks = codes.shape[2], scale.shape[2]
    touched = (rows + block - 2) // block + 1
    first = lens.long()[:, None] // block
    b = (first + torch.arange(touched, device=DEVICE)).clamp_(max=blocks - 1)      # [n, touched]
    pos = (b[:, :, None] * block + torch.arange(block, device=DEVICE)).clamp_(max=L - 1)
    begin = lens.long()[:, None, None]
    end = begin + counts.long()[:, None, None].clamp(max=rows)
    old, new = pos < begin, (pos >= begin) & (pos < end)                      # [n, touched, block]
    ni = torch.arange(n, device=DEVICE)[:, None, None]
    # (indexed along n and the row, the heads end up last but one)
    raw = codes.view(torch.uint8)[ni, :, pos]                              # [n, touched, block, H, D]
    was = raw.view(E4M3).float()
    src = x.float()[ni, :, (pos - begin).clamp(0, rows - 1)]
    size = torch.where(new[..., None, None] & torch.isfinite(src), src.abs(), 0.0).amax((2, 4))
    mant, exp = torch.frexp(size)                                          # size = mant 2^exp
    exp = torch.where(mant > 0.875, exp - 8, exp - 9)                      # 448 = 0.875 2^9
    need = torch.ldexp(torch.ones_like(size), torch.where(size > 0, exp, -100).clamp(min=-100))
    had = scale[ni[:, :, 0], :, b]                                         # [n, touched, H]
    any_old, any_new = old.any(-1)[..., None], new.any(-1)[..., None]
    now = torch.where(any_new, torch.where(any_old, torch.maximum(had, need), need), had)
    by = now[:, :, None, :, None]
    src = torch.where(torch.isfinite(src), src, float("nan"))
    fresh = (src / by).to(E4M3).view(torch.uint8)
    again = (was * (had[:, :, None, :, None] / by)).to(E4M3).view(torch.uint8)
    again = torch.where(any_new[:, :, None, :, None] & old[..., None, None], again, raw)
    codes.view(torch.uint8)[ni, :, pos] = torch.where(new[..., None, None], fresh, again)
    scale[ni[:, :, 0], :, b] = now


def _new_rows(s):
    """K and V of the new tokens as [n, H, rows, D] views of the projection's output."""
    return s["qkv"][:, :, 1].permute(0, 2, 1, 3), s["qkv"][:, :, 2].permute(0, 2, 1, 3)


def _whole(codes, scale, block):
    """The fp32 values of an 8-bit cache."""
    row = torch.arange(codes.shape[2], device=DEVICE) // block
    return codes.float().mul_(scale[:, :, row, None])


def _plain_evict(s, case):
    budget, L = case["budget"], case["max_len"]
    w = s["weights"]
    at = torch.arange(L, device=DEVICE)
    end = s["lens"].long()[:, None, None]
    stays = (at < case["sinks"]) | (at >= end - case["recent"])
    order = torch.where(stays, float("inf"), w)
    order = torch.where(at < end, order, float("-inf"))
    best = torch.sort(order, dim=-1, descending=True, stable=True)[1][..., :budget]
    rank = torch.arange(best.shape[-1], device=DEVICE)
    some = rank < end
    best = torch.sort(torch.where(some, best, L), dim=-1)[0]
    idx = torch.where(some, best, 0)
    r = {"kept": torch.full_like(s["kept"], -1),
         "lens": torch.minimum(s["lens"], torch.full_like(s["lens"], budget))}
    m = idx.shape[-1]
    r["kept"][..., :m] = torch.where(some, best, -1)
    s["weights_out"][..., :m] = torch.where(some, torch.gather(w, 2, idx), s["weights_out"][..., :m])
    r["weights"] = s["weights_out"]
    for x in ("k", "v"):
        got = torch.gather(s[x], 2, idx[..., None].expand(-1, -1, -1, case["D"]))
        to = s[x + "_out"]
        to[:, :, :m] = torch.where(some[..., None], got, to[:, :, :m])
        r[x] = to
    return r


def _run_plain(s, case):
    kind, dt = case["kind"], _dtype(case)
    if kind == "window_train":
        return _plain_train(s, case)
    if kind == "kv8_append":
        k, v = _new_rows(s)
        _plain_append_one(k, s["k8"], s["k_scale"], s["lens"], s["counts"], case["block"])
        _plain_append_one(v, s["v8"], s["v_scale"], s["lens"], s["counts"], case["block"])
        return {"k": s["k8"], "v": s["v8"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "evict":
        return _plain_evict(s, case)
    q = s["q"].float()
    if kind == "kv8_decode":
        k = _whole(s["k8"], s["k_scale"], case["block"])
        v = _whole(s["v8"], s["v_scale"], case["block"])
    else:
        k, v = s["k"].float(), s["v"].float()
    out, p = _plain_decode(q, k, v, s["lens"], s["scale"], case.get("window", 0),
                           case.get("sinks", 0))
    if kind == "weights_decode":
        return {"out": out.to(dt), "weights": s["weights"] + p}
    return {"out": out.to(dt)}


# ------------------------------------------------------------------------------ the framework's

def _run_train(s, case):
    from dadgpt_amd import attention as A
    B, H, S, D, W, K = (case[x] for x in ("B", "H", "S", "D", "window", "sinks"))
    scale, lse, delta, out = s["scale"], s["lse"], s["delta"], s["out"]
    if "workspace" not in s:  # one for the shape, kept as a training loop keeps it
        s["workspace"] = A.window_workspace(B * H, S, D, W, K)
    if case["layout"] == "tokens":
        d = H * D
        q, k, v = (s["qkv"][:, i * d:] for i in range(3))
        dq, dk, dv = (s["dqkv"][:, i * d:] for i in range(3))
        A.flash_attention_window_forward_bf16_tokens(out, d, lse, q, k, v, 3 * d, B, H, S, D, scale,
                                                     W, K)
        A.flash_attention_window_backward_bf16_tokens(
            dq, dk, dv, 3 * d, delta, s["dout"], out, d, lse, q, k, v, 3 * d, B, H, S, D, scale,
            W, K, s["workspace"])
        return {"out": out, "lse": lse, "dqkv": s["dqkv"]}
    bf16 = case["dtype"] == BF16
    forward = A.flash_attention_window_forward_bf16 if bf16 else A.flash_attention_window_forward
    backward = (A.flash_attention_window_backward_bf16 if bf16
                else A.flash_attention_window_backward)
    q, k, v, dq, dk, dv = (s[x] for x in ("q", "k", "v", "dq", "dk", "dv"))
    forward(out, lse, q, k, v, B * H, S, D, scale, W, K)
    backward(dq, dk, dv, delta, s["dout"], out, lse, q, k, v, B * H, S, D, scale, W, K,
             s["workspace"])
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _run_own(s, case):
    kind = case["kind"]
    if kind == "window_train":
        return _run_train(s, case)
    from dadgpt_amd import attention as A
    from dadgpt_amd import kv_cache as C
    n, H, L, D = (case[x] for x in ("n", "H", "max_len", "D"))
    if kind == "kv8_append":
        k, v = _new_rows(s)
        C.kv8_append(s["k8"], s["v8"], s["k_scale"], s["v_scale"], k, v, s["lens"], s["counts"],
                     n, H, case["rows"], L, D, case["block"])
        return {"k": s["k8"], "v": s["v8"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "evict":
        C.kv_evict(s["k_out"], s["v_out"], s["weights_out"], s["kept"], s["lens_out"], s["k"],
                   s["v"], s["weights"], s["lens"], n, H, L, case["budget"], D, case["budget"],
                   case["sinks"], case["recent"])
        return {"kept": s["kept"], "lens": s["lens_out"], "weights": s["weights_out"],
                "k": s["k_out"], "v": s["v_out"]}
    if kind == "window_decode":
        if "workspace" not in s:  # one for the cache's shape, kept as a serving loop keeps it
            s["workspace"] = A.decode_workspace(n, H, L, D)
        A.decode_attention_window(s["out"], s["q"], s["k"], s["v"], s["lens"], n, H, L, D,
                                  s["scale"], case["window"], case["sinks"], s["workspace"])
        return {"out": s["out"]}
    if kind == "kv8_decode":
        if "workspace" not in s:
            s["workspace"] = C.decode_kv8_workspace(n, H, L, D)
        C.decode_attention_kv8(s["out"], s["q"], s["k8"], s["v8"], s["k_scale"], s["v_scale"],
                               s["lens"], n, H, L, D, case["block"], s["scale"], case["window"],
                               case["sinks"], s["workspace"])
        return {"out": s["out"]}
    if "workspace" not in s:
        s["workspace"] = C.decode_weights_workspace(n, H, L, D)
    C.decode_attention_weights(s["out"], s["weights_out"], s["q"], s["k"], s["v"], s["weights"],
                               s["lens"], n, H, L, D, s["scale"], s["workspace"])
    return {"out": s["out"], "weights": s["weights_out"]}


def run(state):
    case = state["case"]
    return _run_own(state, case) if own else _run_plain(state, case)


# ------------------------------------------------------------------------------ the floor

def _mean_least(hi, most):
    """The mean of min(len, most) over len uniform on [1, hi]."""
    full = min(hi, most)
    return (full * (full + 1) / 2 + (hi - full) * full) / hi


def work(case):
    size = 4 if case["dtype"] == F32 else 2
    H, D, kind = case["H"], case["D"], case["kind"]
    if kind == "window_train":
        B, S, W, K = (case[x] for x in ("B", "S", "window", "sinks"))
        t, stat = B * H * S * D * size, B * H * S * 4
        near = min(S, W)
        pairs = near * (near + 1) // 2 + (S - near) * near
        far = max(0, S - W)  # rows with keys before their window; the j-th of them has j
        k = min(K, far)
        pairs += k * (k + 1) // 2 + (far - k) * k
        # forward: q, k, v in, out and lse out, two products; backward: q, k, v, dout, out, lse
        # in, gradients out, five products
        return {"bytes": 12 * t + 2 * stat, "flops": 14 * D * B * H * pairs}
    n, L = case["n"], case["max_len"]
    if kind == "kv8_append":
        rows = n * H * (case["rows"] + 1) / 2
        return {"bytes": 2 * rows * D * (size + 1) + 8 * n * H * math.ceil(
            (case["rows"] + 1) / 2 / case["block"]) + 8 * n, "flops": 4 * rows * D}
    if kind == "evict":
        rows, keys = n * H * _mean_least(L, case["budget"]), n * H * (L + 1) / 2
        return {"bytes": 4 * keys + 4 * rows * D * size + 4 * rows + 4 * n * H * case["budget"],
                "flops": keys}
    most = case["window"] + case["sinks"] if case.get("window") else L
    keys = n * H * _mean_least(L, most)
    io = 2 * n * H * D * size + 4 * n
    if kind == "kv8_decode":
        return {"bytes": keys * (2 * D + 8 / case["block"]) + io, "flops": 4 * keys * D}
    if kind == "weights_decode":
        io += 8 * keys
    return {"bytes": 2 * keys * D * size + io, "flops": 4 * keys * D}


# ------------------------------------------------------------------------------ float64

def _exact_train(s, case):
    """Row by row over the keys that a row sees: its window, then the sinks before it."""
    B, H, S, D, W, K = (case[x] for x in ("B", "H", "S", "D", "window", "sinks"))
    c = 1.0 / math.sqrt(D)
    if case["layout"] == "tokens":
        parts = s["qkv"].view(B, S, 3, H, D).permute(2, 0, 3, 1, 4).reshape(3, B * H, S, D)
        q, k, v = parts[0], parts[1], parts[2]
        g = s["dout"].view(B, S, H, D).permute(0, 2, 1, 3).reshape(B * H, S, D)
    else:
        q, k, v, g = s["q"], s["k"], s["v"], s["dout"]
    f8 = torch.float64
    out, dq, dk, dv = (torch.zeros((B * H, S, D), dtype=f8, device=DEVICE) for _ in range(4))
    lse = torch.zeros((B * H, S), dtype=f8, device=DEVICE)
    heads = max(1, min(B * H, (1 << 23) // max(1, min(S, 512) * min(S, W + 512 + K))))
    for h in range(0, B * H, heads):
        hs = slice(h, min(B * H, h + heads))
        for a in range(0, S, 512):
            b = min(S, a + 512)
            lo = max(0, a - W + 1)
            keys = torch.cat((torch.arange(0, min(K, lo), device=DEVICE),
                              torch.arange(lo, b, device=DEVICE)))
            i = torch.arange(a, b, device=DEVICE)[:, None]
            hidden = (keys > i) | ((keys <= i - W) & (keys >= K))
            Q, G = q[hs, a:b].to(f8), g[hs, a:b].to(f8)
            KK, V = k[hs][:, keys].to(f8), v[hs][:, keys].to(f8)
            x = torch.matmul(Q, KK.mT.contiguous()) * c
            x = torch.where(hidden, -math.inf, x)
            z = torch.logsumexp(x, -1)
            P = torch.exp(x - z[..., None])
            o = torch.matmul(P, V)
            dP = torch.matmul(G, V.mT.contiguous())
            dS = P * (dP - (P * dP).sum(-1, keepdim=True))
            out[hs, a:b], lse[hs, a:b] = o, z
            dq[hs, a:b] = torch.matmul(dS, KK) * c
            dk[hs].index_add_(1, keys, torch.matmul(dS.mT.contiguous(), Q) * c)
            dv[hs].index_add_(1, keys, torch.matmul(P.mT.contiguous(), G))
    if case["layout"] == "tokens":
        def rows(x):
            return x.view(B, H, S, D).permute(0, 2, 1, 3).reshape(B * S, H * D)
        return {"out": rows(out), "lse": lse, "dqkv": torch.cat((rows(dq), rows(dk), rows(dv)), 1)}
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _e4m3_round(x):
    """The nearest e4m3 value (ties to the even mantissa) of each |x| <= 448, in float64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s, case, x, codes, scale):
    values, scale = codes.to(torch.float64), scale.to(torch.float64)
    block, L = case["block"], case["max_len"]
    for i, (at, count) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
        end = min(L, at + min(count, case["rows"]))
        for b in range(at // block, (end - 1) // block + 1):
            lo, hi = max(at, b * block), min(end, (b + 1) * block)
            new = x[i, :, lo - at:hi - at].to(torch.float64)
            size = new.abs().amax((1, 2))
            to = torch.exp2(torch.ceil(torch.log2((size / 448.0).clamp(min=2.0 ** -100))))
            if b * block < at:
                was = scale[i, :, b]
                to = torch.maximum(to, was)
                held = values[i, :, b * block:at]
                values[i, :, b * block:at] = _e4m3_round(held * (was / to)[:, None, None])
            values[i, :, lo:hi] = _e4m3_round(new / to[:, None, None])
            scale[i, :, b] = to
    return values, scale


def _exact_evict(s, case):
    n, H, budget = case["n"], case["H"], case["budget"]
    r = {"kept": torch.full_like(s["kept"], -1).cpu(), "lens": torch.zeros_like(s["lens"]).cpu(),
         "weights": s["weights_out"].clone(), "k": s["k_out"].clone(), "v": s["v_out"].clone()}
    for i, end in enumerate(s["lens"].tolist()):
        keep = min(end, budget)
        r["lens"][i] = keep
        first = min(case["sinks"], end)
        last = max(first, end - case["recent"])
        for h in range(H):
            if end <= budget:
                kept = list(range(end))
            else:
                w = s["weights"][i, h, first:last].tolist()
                by = sorted(range(first, last), key=lambda j: (-w[j - first], j))
                kept = sorted(list(range(first)) + by[:budget - first - (end - last)]
                              + list(range(last, end)))
            r["kept"][i, h, :keep] = torch.tensor(kept, dtype=torch.int32)
            at = torch.tensor(kept, device=DEVICE)
            r["weights"][i, h, :keep] = s["weights"][i, h, at]
            r["k"][i, h, :keep], r["v"][i, h, :keep] = s["k"][i, h, at], s["v"][i, h, at]
    r["kept"], r["lens"] = r["kept"].to(DEVICE), r["lens"].to(DEVICE)
    return r


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "window_train":
        return _exact_train(s, case)
    if kind == "evict":
        return _exact_evict(s, case) if case["n"] * case["H"] * case["max_len"] < 4e6 else None
    if kind == "kv8_append":
        n, rows, _, H, D = s["qkv"].shape
        if n * (rows / case["block"] + 2) > 8192:
            return None
        k = s["qkv"].select(2, 1).transpose(1, 2)
        v = s["qkv"].select(2, 2).transpose(1, 2)
        kv, ks = _exact_append(s, case, k, s["k8"], s["k_scale"])
        vv, vs = _exact_append(s, case, v, s["v8"], s["v_scale"])
        return {"k": kv, "v": vv, "k_scale": ks, "v_scale": vs}
    f8 = torch.float64
    outs, weights = [], []
    for i, end in enumerate(s["lens"].tolist()):
        keys = torch.arange(end, device=DEVICE)
        if case.get("window"):
            lo = max(0, end - case["window"])
            keys = torch.cat((keys[:min(case["sinks"], lo)], keys[lo:]))
        if kind == "kv8_decode":
            b = keys // case["block"]
            k = s["k8"][i, :, :end].to(f8)[:, keys] * s["k_scale"][i].to(f8)[:, b, None]
            v = s["v8"][i, :, :end].to(f8)[:, keys] * s["v_scale"][i].to(f8)[:, b, None]
        else:
            k, v = s["k"][i][:, keys].to(f8), s["v"][i][:, keys].to(f8)
        x = (k * s["q"][i].to(f8)[:, None]).sum(-1) / math.sqrt(case["D"])
        P = torch.softmax(x, -1)
        outs.append((P[..., None] * v).sum(1))
        if kind == "weights_decode":
            w = s["weights"][i].to(f8)
            w[:, :end] += P
            weights.append(w)
    if kind == "weights_decode":
        return {"out": torch.stack(outs), "weights": torch.stack(weights)}
    return {"out": torch.stack(outs)}
