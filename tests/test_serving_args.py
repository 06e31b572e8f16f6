"""CPU tests of the rotary positions', paged caches' and sampling's C ABI: headers and bindings agree,
frequencies are the definitions', every check answers on the host before any HIP call."""
import ctypes
import math
import os
import re

import pytest
import torch

from dadgpt_amd import attention as A
from dadgpt_amd import paged as P
from dadgpt_amd import rope as R
from dadgpt_amd import sampling as Z

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE, STEP = 0x1000000, 0x10000000  # non-null addresses, far apart; no call below gets past its checks


def _at(i):
    return FAKE + i * STEP


@pytest.mark.parametrize("header,lib,symbols", [("rope", R.lib, R.ROPE_SYMBOLS),
                                                ("paged_cache", P.lib, P.PAGED_SYMBOLS),
                                                ("sampling", Z.lib, Z.SAMPLING_SYMBOLS)])
def test_header_and_binding_agree(header, lib, symbols):
    text = open(os.path.join(ROOT, "include", "dadgpt", header + ".h")).read()
    declared = set(re.findall(r"^(?:int|size_t) (dadgpt_\w+)\s*\(", text, re.M))
    assert declared == set(symbols)
    assert all(hasattr(lib(), s) for s in symbols)


def _refused(call, want, **changes):
    """call(**changes) answers status `want[0]` with `want[1]` in the message."""
    status, text = want
    assert call(**changes) == status, changes
    assert text in A.last_error(), (changes, A.last_error())


# ------------------------------------------------------------------------ rotary positions

def test_frequencies():
    i = torch.arange(32, dtype=torch.float64)
    f = 10000.0 ** (-2 * i / 64)
    near = dict(rtol=1e-14, atol=0.0)
    torch.testing.assert_close(R.rope_frequencies(64, device="cpu"), f, **near)
    torch.testing.assert_close(R.rope_frequencies(64, scaling="linear", factor=4.0, device="cpu"), f / 4,
                               **near)
    b = R.rope_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert b[0] == 1.0 and abs(b[-1] / (f[-1] / 4) - 1) < 1e-12
    p = R.rope_frequencies(64, scaling="parts", factor=4.0, original_len=2048, device="cpu")
    turns = 2048 * f / (2 * math.pi)
    g = ((turns - 1) / 31).clamp(0, 1)
    torch.testing.assert_close(p, f * (g + (1 - g) / 4), rtol=1e-13, atol=0.0)
    assert (p[turns >= 32] == f[turns >= 32]).all()
    assert R.rope_magnitude(1.0) == 1.0 and abs(R.rope_magnitude(8.0) - 1.2079441541679836) < 1e-12


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=-2), dict(base=0.0),
                                dict(base=math.inf), dict(base=math.nan), dict(factor=0.0),
                                dict(factor=-1.0), dict(scaling="base", rot_dim=2),
                                dict(scaling="parts"), dict(scaling="parts", original_len=9, slow=32.0)])
def test_frequency_refusals(kw):
    kw = {"rot_dim": 64, "device": "cpu", **kw}
    with pytest.raises(A.AttentionError) as e:
        R.rope_frequencies(**kw)
    assert e.value.status == 1
    with pytest.raises(KeyError):
        R.rope_frequencies(64, scaling="other", device="cpu")
    assert R.lib().dadgpt_rope_frequencies(FAKE, 64, 1e4, 4, 1.0, 0, 1.0, 32.0) == 1
    assert R.lib().dadgpt_rope_frequencies(None, 64, 1e4, 0, 1.0, 0, 1.0, 32.0) == 1


@pytest.mark.parametrize("name", ["rope_bf16", "rope_f32", "rope_backward_bf16", "rope_backward_f32"])
def test_rope_refusals(name):
    fn = getattr(R.lib(), "dadgpt_" + name)
    size = 2 if name.endswith("bf16") else 4
    B, H, Hkv, S, D = 2, 4, 2, 8, 64
    row = (H + 2 * Hkv) * D  # a fused projection's
    fused = (S * row, D, row)

    def call(ptrs=(_at(0), _at(1), _at(2), _at(2) + H * D * size), strides=None, B=B, H=H, Hkv=Hkv, S=S,
             D=D, freqs=_at(5), rot=32, mag=1.0, pos=None):
        st = [fused, fused, (S * H * 64, S * 64, 64), (S * Hkv * 64, S * 64, 64)]
        for i, x in (strides or {}).items():
            st[i] = x
        flat = (ctypes.c_int64 * 12)(*[y for x in st for y in x])
        return fn(*ptrs, flat, B, H, Hkv, S, D, freqs, rot, 0, mag, pos, None)
    good = (_at(0), _at(1), _at(2), _at(2) + H * D * size)
    for i in range(4):
        bad = list(good)
        bad[i] = None
        _refused(call, (1, "null"), ptrs=bad)
        bad[i] = good[i] + 2
        _refused(call, (1, "aligned"), ptrs=bad)
    assert fn(*good, None, B, H, Hkv, S, D, _at(5), 32, 0, 1.0, None, None) == 1
    _refused(call, (2, "d_head"), D=48)
    _refused(call, (2, "d_head"), D=128)
    for kw in (dict(B=0), dict(H=0), dict(Hkv=0), dict(Hkv=-1), dict(S=0)):
        _refused(call, (1, "positive"), **kw)
    for rot in (0, 4, 12, 72, -8):
        _refused(call, (1, "rot_dim"), rot=rot)
    _refused(call, (1, "freqs is null"), freqs=None)
    _refused(call, (1, "aligned"), freqs=_at(5) + 4)
    _refused(call, (1, "aligned"), pos=_at(6) + 2)
    _refused(call, (1, "magnitude"), mag=math.nan)
    for x in ((-8, 64, row), (S * row, 4, row), (S * row, 64, 12), ((1 << 40) + 8, 64, row)):
        _refused(call, (1, "strides"), strides={0: x})
    _refused(call, (1, "launch limits"), B=1 << 15, S=1 << 14)
    # overlaps: outputs with each other, with inputs in another place, with themselves, with the arrays
    _refused(call, (1, "overlaps"), ptrs=(_at(0), _at(0), good[2], good[3]))
    _refused(call, (1, "overlaps"), ptrs=(good[2], _at(1), good[2], good[3]))   # other strides
    _refused(call, (1, "overlaps"), ptrs=(good[3], _at(1), good[2], good[3]), strides={2: fused})
    _refused(call, (1, "overlaps"), ptrs=(good[2] + 16, _at(1), good[2], good[3]), strides={2: fused})
    _refused(call, (1, "overlap each other"), strides={2: (0, 0, 64)})
    _refused(call, (1, "overlap each other"), strides={2: (S * 64, 32, 64)})
    _refused(call, (1, "overlaps freqs" if "back" not in name else "freqs"), freqs=_at(0))
    _refused(call, (1, "positions"), pos=_at(1) + 64)


# ------------------------------------------------------------------------ paged caches

STEPS = dict(n_seq=3, H=4, Hkv=2, rows=20, max_rows=10, n_pages=9, page=16, max_pages=8, D=64)


def _step(kw):
    s = {**STEPS, **{k: v for k, v in kw.items() if k in STEPS}}
    return [s[k] for k in STEPS]


STEP_REFUSALS = [(dict(n_seq=0), 1, "positive"), (dict(H=0), 1, "positive"), (dict(Hkv=0), 1, "positive"),
                 (dict(rows=0), 1, "positive"), (dict(max_rows=0), 1, "positive"),
                 (dict(n_pages=0), 1, "positive"), (dict(max_pages=-1), 1, "positive"),
                 (dict(H=5), 1, "no multiple"), (dict(page=8), 1, "page=8"), (dict(page=48), 1, "page=48"),
                 (dict(page=256), 1, "page=256"), (dict(D=128), 2, "d_head"), (dict(D=16), 2, "d_head"),
                 (dict(max_pages=65535 * 16 + 1), 1, "tokens"),
                 (dict(n_seq=65536), 1, "launch limits"), (dict(rows=(1 << 24) + 1), 1, "launch limits")]


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_append_refusals(name):
    fn, size = getattr(P.lib(), "dadgpt_paged_append_" + name), 2 if name == "bf16" else 4

    def call(kp=_at(0), vp=_at(1), qo=_at(2), ld_out=256, q=_at(3), ld_q=512, k=_at(3) + 256 * size,
             v=_at(3) + 384 * size, ld_kv=512, table=_at(4), starts=_at(5), lens=_at(6), freqs=_at(7),
             rot=64, mag=1.0, **kw):
        return fn(kp, vp, qo, ld_out, q, ld_q, k, v, ld_kv, table, starts, lens, *_step(kw), freqs, rot, 0,
                  mag, None)
    for x in ("kp", "vp", "k", "v"):
        _refused(call, (1, "null"), **{x: None})
        _refused(call, (1, "aligned"), **{x: _at(9) + 4})
    _refused(call, (1, "together"), q=None)
    _refused(call, (1, "together"), qo=None)
    for x in ("table", "starts", "lens"):
        _refused(call, (1, "null"), **{x: None})
        _refused(call, (1, "aligned"), **{x: _at(9) + 2})
    for kw, status, text in STEP_REFUSALS:
        _refused(call, (status, text), **kw)
    for x in ("ld_out", "ld_q"):
        for ld in (248, 260, (1 << 24) + 8, -8):
            _refused(call, (1, x), **{x: ld})
    for ld in (120, 132, (1 << 24) + 8):
        _refused(call, (1, "ld_kv"), ld_kv=ld)
    _refused(call, (1, "without freqs"), freqs=None)
    for rot in (0, 12, 72):
        _refused(call, (1, "rot_dim"), rot=rot)
    _refused(call, (1, "magnitude"), mag=math.inf)
    _refused(call, (1, "overlaps"), vp=_at(0))
    _refused(call, (1, "overlaps"), vp=_at(0) + 9 * 2 * 16 * 64 * size - 16)
    _refused(call, (1, "k_pages overlaps q_out"), qo=_at(0))
    _refused(call, (1, "v_pages overlaps v"), v=_at(1))
    _refused(call, (1, "overlaps block_table"), table=_at(1) + 64)
    _refused(call, (1, "overlaps lens"), lens=_at(2))
    _refused(call, (1, "overlaps freqs"), freqs=_at(2))
    _refused(call, (1, "q_out overlaps q"), qo=_at(3))                        # another pitch
    _refused(call, (1, "q_out overlaps k"), qo=_at(3) + 16 * size, ld_out=512, q=_at(8))


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_append_in_place_is_of_q_alone(name):
    """q_out may be q; where k or v begin at the same address, the call would overwrite what it reads."""
    fn = getattr(P.lib(), "dadgpt_paged_append_" + name)
    for k, v, what in ((_at(3), _at(2), "k"), (_at(2), _at(3), "v"), (_at(3), _at(3), "k")):
        for H, heads in ((4, 4), (2, 2)):
            status = fn(_at(0), _at(1), _at(3), heads * 64, _at(3), heads * 64, k, v, 256, _at(4), _at(5),
                        _at(6), *_step(dict(H=H)), _at(7), 64, 0, 1.0, None)
            assert status == 1 and "q_out overlaps " + what in A.last_error()


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_attention_refusals(name):
    fn, size = getattr(P.lib(), "dadgpt_paged_attention_" + name), 2 if name == "bf16" else 4

    def call(out=_at(0), ld_out=256, q=_at(1), ld_q=512, kp=_at(2), vp=_at(3), table=_at(4),
             starts=_at(5), lens=_at(6), scale=0.125, ws=_at(7), ws_bytes=1 << 24, **kw):
        return fn(out, ld_out, q, ld_q, kp, vp, table, starts, lens, *_step(kw), scale, ws, ws_bytes, None)
    for x in ("out", "q", "kp", "vp"):
        _refused(call, (1, "null"), **{x: None})
        _refused(call, (1, "aligned"), **{x: _at(9) + 4})
    for x in ("table", "starts", "lens"):
        _refused(call, (1, "null"), **{x: None})
        _refused(call, (1, "aligned"), **{x: _at(9) + 2})
    for kw, status, text in STEP_REFUSALS:
        _refused(call, (status, text), **kw)
    for x in ("ld_out", "ld_q"):
        for ld in (248, 260, (1 << 24) + 8):
            _refused(call, (1, x), **{x: ld})
    _refused(call, (1, "scale"), scale=math.nan)
    _refused(call, (1, "launch limits"), H=4096, Hkv=1, rows=1 << 14, max_rows=1 << 14, ld_q=1 << 18,
             ld_out=1 << 18)
    _refused(call, (1, "out overlaps q"), out=_at(1))                         # another pitch
    _refused(call, (1, "out overlaps q"), out=_at(1) + 64 * size, ld_out=512)
    _refused(call, (1, "out overlaps k_pages"), out=_at(2))
    _refused(call, (1, "out overlaps v_pages"), out=_at(3) + 64)
    _refused(call, (1, "out overlaps block_table"), table=_at(0) + 64)
    split = dict(max_pages=512)  # 8192 tokens: chunks
    assert P.paged_workspace_bytes(*_workspace(split)) > 0
    _refused(call, (4, "workspace"), ws=None, **split)
    _refused(call, (4, "workspace"), ws_bytes=1000, **split)
    _refused(call, (1, "16-byte aligned"), ws=_at(7) + 8, **split)
    for x, what in ((0, "out"), (1, "q"), (2, "k_pages"), (3, "v_pages"), (5, "row_start")):
        _refused(call, (1, "the workspace overlaps " + what), ws=_at(x), **split)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_the_largest_steps(name):
    """Steps are refused for their grid from its limit on, 65535 workgroups of a KV head, not before: a token
    of each of 65535 sequences, and tiles of 128 rows (with up to 2 * 768 / n_kv_heads + 1 places for chunks)."""
    fn = getattr(P.lib(), "dadgpt_paged_attention_" + name)

    def call(n_seq, rows, max_rows):
        step = dict(n_seq=n_seq, H=2, Hkv=2, rows=rows, max_rows=max_rows, n_pages=9, page=16, max_pages=512,
                    D=64)
        status = fn(_at(0), 128, _at(100), 128, _at(200), _at(300), _at(400), _at(500), _at(600),
                    *step.values(), 0.125, None, 0, None)
        return status, A.last_error()
    for n_seq, rows, max_rows in ((65535, 65535, 1), (60000, (65535 - 769 - 60000) * 128, 1000),
                                  (1, 65535 * 128 - 769 * 128, 65535 * 128 - 769 * 128)):
        status, text = call(n_seq, rows, max_rows)
        assert status == 4 and "workspace" in text, text
    status, text = call(60000, (65535 - 769 - 60000 + 1) * 128, 1000)
    assert status == 1 and "launch limits" in text


def _workspace(kw):
    s = {**STEPS, **kw}
    return [s[k] for k in ("n_seq", "H", "Hkv", "rows", "max_rows", "page", "max_pages", "D")]


def test_workspace_sizes():
    """0 where no cache is cut; growing with every one of n_seq, rows, max_rows and max_pages; 0 for a
    shape that is refused."""
    def need(**kw):
        return P.paged_workspace_bytes(*_workspace(kw))
    assert need() == 0
    for key, values in (("max_pages", (17, 64, 512, 4096, 1 << 17)), ("n_seq", (1, 3, 64, 1000, 10000)),
                        ("max_rows", (1, 5, 20)), ("rows", (20, 100, 10000, 1 << 20))):
        base = {"max_pages": 512}
        sizes = [need(**{**base, key: v}) for v in values]
        assert sizes == sorted(sizes) and sizes[0] > 0, (key, sizes)
    for kw in (dict(n_seq=0), dict(page=10), dict(D=65), dict(H=3)):
        assert need(max_pages=512, **{k: v for k, v in kw.items()}) == 0


# ------------------------------------------------------------------------ sampling

@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_sample_refusals(name):
    fn, size = getattr(Z.lib(), "dadgpt_sample_" + name), 2 if name == "bf16" else 4

    def call(tokens=_at(0), probs=_at(1), logits=_at(2), ld=1000, rows=4, vocab=1000, u=_at(3), t=_at(4),
             k=_at(5), p=_at(6), m=_at(7)):
        return fn(tokens, probs, logits, ld, rows, vocab, u, t, k, p, m, None)
    for x in ("tokens", "logits", "u"):
        _refused(call, (1, "null"), **{x: None})
    for x in ("tokens", "probs", "u", "t", "k", "p", "m"):
        _refused(call, (1, "aligned"), **{x: _at(9) + 2})
    _refused(call, (1, "aligned"), logits=_at(2) + size // 2)
    for kw in (dict(rows=0), dict(vocab=0)):
        _refused(call, (1, "positive"), **kw)
    for kw in (dict(vocab=Z.MAX_VOCAB + 1, ld=1 << 20), dict(rows=1 << 21)):
        _refused(call, (1, "limits"), **kw)
    for ld in (999, (1 << 40) + 1):
        _refused(call, (1, "ld="), ld=ld)
    _refused(call, (1, "tokens overlaps probs"), probs=_at(0) + 12)
    _refused(call, (1, "tokens overlaps logits"), tokens=_at(2) + 2000 * size)
    _refused(call, (1, "probs overlaps uniforms"), u=_at(1))
    for x, what in (("t", "temperature"), ("k", "top_k"), ("p", "top_p"), ("m", "min_p")):
        _refused(call, (1, "tokens overlaps " + what), **{x: _at(0)})


# ------------------------------------------------------------------------ Python's checks

def test_python_checks():
    """Tensors that are no device tensors, of another type or of another shape are refused before any
    call."""
    cpu = torch.zeros((4, 2, 64))
    with pytest.raises(TypeError):
        R.rope(cpu[None], None, cpu[None], None, torch.zeros(16, dtype=torch.float64))
    with pytest.raises(TypeError):
        R.rope(cpu[None].half(), None, cpu[None].half(), None, torch.zeros(16, dtype=torch.float64))
    pages, table = torch.zeros((4, 2, 16, 64)), torch.zeros((1, 4), dtype=torch.int32)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        P.paged_append(pages, pages, None, None, cpu, cpu, table, ints, ints, 1)
    with pytest.raises(ValueError):
        P.paged_attention(cpu, cpu, pages, pages, table, ints, ints, 1, 1.0, None)
    with pytest.raises(TypeError):
        P.paged_attention(cpu.half(), cpu.half(), pages, pages, table, ints, ints, 1, 1.0, None)
    with pytest.raises(ValueError):
        P.paged_cache(4, 2, 24, 64, device="cpu")
    with pytest.raises(ValueError):
        Z.sample(ints, None, cpu[0], torch.zeros(2))
