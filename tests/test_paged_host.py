"""Refusals of the rotary and paged entry points, and the frequencies, without a GPU."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from polykernel_amd import _lib, kernels

BF = torch.bfloat16
FAKE = 0x100000  # never dereferenced: every call is refused before a device call


def theta(turns):
    return (turns * 2 * math.pi).tolist()


def plain(dim, base):
    return [base ** (-2 * i / dim) for i in range(dim // 2)]


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (24, 1e6)])
def test_frequencies(dim, base):
    turns, mag = kernels.rotary_frequencies(dim, base, device="cpu")
    assert mag == 1.0 and theta(turns) == pytest.approx(plain(dim, base), rel=1e-14)
    slow, mag = kernels.rotary_frequencies(dim, base, "linear", 4.0, device="cpu")
    assert mag == 1.0 and theta(slow) == pytest.approx([t / 4 for t in plain(dim, base)], rel=1e-14)


def test_frequencies_of_a_stretched_base():
    turns, _ = kernels.rotary_frequencies(128, 10000.0, "base", 8.0, device="cpu")
    assert theta(turns) == pytest.approx(plain(128, 10000.0 * 8.0 ** (128 / 126)), rel=1e-14)
    assert theta(turns)[0] == pytest.approx(1.0) and theta(turns)[-1] == pytest.approx(plain(128, 10000.0)[-1] / 8, rel=1e-13)


def test_frequencies_in_bands():
    f, low, high, n = 8.0, 1.0, 4.0, 8192
    turns, mag = kernels.rotary_frequencies(128, 500000.0, "bands", f, low, high, n, device="cpu")
    assert mag == 1.0
    for t, got in zip(plain(128, 500000.0), theta(turns)):
        wave = 2 * math.pi / t
        if wave < n / high:
            want = t
        elif wave > n / low:
            want = t / f
        else:
            mix = (n / wave - low) / (high - low)
            want = (1 - mix) * t / f + mix * t
        assert got == pytest.approx(want, rel=1e-13)


@pytest.mark.parametrize("dim,n", [(128, 4096), (64, 2048), (128, 2)])
def test_frequencies_on_a_ramp(dim, n):
    base, f, low, high = 10000.0, 16.0, 1.0, 32.0
    turns, mag = kernels.rotary_frequencies(dim, base, "ramp", f, low, high, n, device="cpu")
    assert mag == pytest.approx(0.1 * math.log(f) + 1)
    place = lambda r: dim * math.log(n / (r * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    first, last = max(math.floor(place(high)), 0), min(math.ceil(place(low)), dim - 1)
    for i, (t, got) in enumerate(zip(plain(dim, base), theta(turns))):
        mix = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
        assert got == pytest.approx(t / f * mix + t * (1 - mix), rel=1e-13)


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=3), dict(dim=-2), dict(base=0.0), dict(base=math.inf),
                                dict(scaling="linear", factor=0.0), dict(scaling="linear", factor=math.nan),
                                dict(scaling="bands", factor=2.0), dict(scaling="ramp", factor=2.0, original=10, low=4.0),
                                dict(scaling="bands", factor=2.0, original=10, low=0.0),
                                dict(scaling="base", factor=2.0, dim=2), dict(scaling="ramp", factor=2.0, original=10, base=1.0)])
def test_frequencies_refused(kw):
    with pytest.raises(_lib.PolyKernelError, match="pk_rotary_frequencies"):
        kernels.rotary_frequencies(**{"dim": 64, "device": "cpu", **kw})


def test_unknown_scaling_refused():
    with pytest.raises(ValueError, match="scaling"):
        kernels.rotary_frequencies(64, scaling="other", device="cpu")
    out = (C.c_double * 4)()
    assert _lib.load().pk_rotary_frequencies(8, 10.0, 5, 1.0, 1.0, 2.0, 1.0, out, None) == _lib.PK_ERR_INVALID_ARG
    assert _lib.load().pk_rotary_frequencies(8, 10.0, 0, 1.0, 1.0, 2.0, 1.0, None, None) == _lib.PK_ERR_INVALID_ARG


# ---- the C entries ------------------------------------------------------------------
def rotation(**kw):
    return _lib.Rotary(**{**dict(turns=FAKE, dim=64, interleaved=0, inverse=0, magnitude=1.0), **kw})


def rotary_call(B=1, S=4, H=2, D=64, rot=None, x=FAKE, positions=FAKE, strides=True):
    s = (C.c_int64 * 3)(0, 128, 64) if strides else None
    return _lib.load().launch_rotary(x, s, FAKE, s, positions, 0, B, S, H, D, rot if rot is not None else rotation(), None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), "INVALID_ARG", "shape"), (dict(D=0), "INVALID_ARG", "shape"), (dict(D=1026), "UNSUPPORTED", "1024"),
    (dict(rot=rotation(dim=63)), "INVALID_ARG", "rotated"), (dict(rot=rotation(dim=66)), "INVALID_ARG", "rotated"),
    (dict(rot=rotation(dim=0)), "INVALID_ARG", "rotated"), (dict(rot=rotation(turns=None)), "INVALID_ARG", "turns"),
    (dict(x=None), "INVALID_ARG", "null"), (dict(positions=None), "INVALID_ARG", "null"),
    (dict(strides=False), "INVALID_ARG", "null"), (dict(B=65536, S=65536), "INVALID_ARG", "exceeds"),
    (dict(H=2**25), "INVALID_ARG", "exceeds"), (dict(S=2**27), "UNSUPPORTED", "tokens"),
])
def test_rotary_refused(kw, code, word):
    assert rotary_call(**kw) == getattr(_lib, "PK_ERR_" + code) and word in _lib.last_error()


def paged_cache(**kw):
    return _lib.PagedCache(**{**dict(k=FAKE, v=FAKE, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024,
                                     v_row=64, pages=4, page_size=16, heads=2, dim=64), **kw})


def paged_batch(**kw):
    return _lib.PagedBatch(**{**dict(page_table=FAKE, table_stride=4, table_width=4, q_start=FAKE, kv_len=FAKE,
                                     sequences=2, tokens=2, max_q=1, max_kv=0), **kw})


BAD_PAGED = [
    (dict(cache=paged_cache(k=None)), "INVALID_ARG", "null cache"),
    (dict(cache=paged_cache(page_size=0)), "INVALID_ARG", "invalid cache"),
    (dict(cache=paged_cache(pages=-1)), "INVALID_ARG", "invalid cache"),
    (dict(cache=paged_cache(heads=0)), "INVALID_ARG", "invalid cache"),
    (dict(cache=paged_cache(dim=0)), "INVALID_ARG", "invalid cache"),
    (dict(cache=paged_cache(dim=1025)), "UNSUPPORTED", "1024"),
    (dict(batch=paged_batch(tokens=-1)), "INVALID_ARG", "invalid batch"),
    (dict(batch=paged_batch(max_q=-1)), "INVALID_ARG", "invalid batch"),
    (dict(batch=paged_batch(max_kv=-1)), "INVALID_ARG", "invalid batch"),
    (dict(batch=paged_batch(kv_len=None)), "INVALID_ARG", "null"),
    (dict(batch=paged_batch(page_table=None)), "INVALID_ARG", "null"),
    (dict(batch=paged_batch(q_start=None, tokens=1)), "INVALID_ARG", "without q_start"),
    (dict(batch=paged_batch(table_width=2**27)), "INVALID_ARG", "INT32_MAX"),
    (dict(batch=paged_batch(table_width=2**27 - 256)), "INVALID_ARG", "INT32_MAX"),
    (dict(batch=None), "INVALID_ARG", "null batch"),
    (dict(cache=None), "INVALID_ARG", "null cache"),
]


def tok(data=FAKE):
    return _lib.Tokens(data, 128, 64)


def append_call(cache=paged_cache(), batch=paged_batch(), k=tok(), v=tok(), q=None, q_out=None, q_heads=0, rot=None):
    return _lib.load().launch_paged_kv_append(k, v, q, q_out, q_heads, cache, batch, rot, None)


def attend_call(cache=paged_cache(), batch=paged_batch(), q=tok(), out=tok(), q_heads=4, window=0, ws=None, ws_bytes=0,
                scale=0.125):
    return _lib.load().launch_paged_attention(q, out, q_heads, cache, batch, scale, 1, window, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", BAD_PAGED + [
    (dict(k=None), "INVALID_ARG", "null k or v"), (dict(v=tok(None)), "INVALID_ARG", "null tensor"),
    (dict(q=tok(), q_out=tok(), q_heads=4), "INVALID_ARG", "come together"),
    (dict(q=tok(), rot=rotation(), q_heads=4), "INVALID_ARG", "come together"),
    (dict(q=tok(), q_out=tok(), rot=rotation(), q_heads=0), "INVALID_ARG", "query heads"),
    (dict(rot=rotation(inverse=1)), "INVALID_ARG", "inverse"), (dict(rot=rotation(dim=66)), "INVALID_ARG", "rotated"),
    (dict(q=tok(), q_out=tok(), rot=rotation(), q_heads=2**26), "INVALID_ARG", "heads"),
    (dict(batch=paged_batch(tokens=2**27)), "UNSUPPORTED", "tokens"),
])
def test_append_refused(kw, code, word):
    assert append_call(**kw) == getattr(_lib, "PK_ERR_" + code) and word in _lib.last_error()


@pytest.mark.parametrize("kw,code,word", BAD_PAGED + [
    (dict(q=None), "INVALID_ARG", "null q or out"), (dict(out=tok(None)), "INVALID_ARG", "null tensor"),
    (dict(q_heads=3), "INVALID_ARG", "query heads"), (dict(q_heads=0), "INVALID_ARG", "query heads"),
    (dict(window=-1), "INVALID_ARG", "window"),
    (dict(batch=paged_batch(tokens=2**20), q_heads=2**12), "INVALID_ARG", "exceeds"),
    (dict(cache=paged_cache(dim=20), batch=paged_batch(tokens=2**25)), "UNSUPPORTED", "tokens"),
    (dict(cache=paged_cache(dim=20), q_heads=70000), "UNSUPPORTED", "query heads"),
])
def test_attention_refused(kw, code, word):
    assert attend_call(**kw) == getattr(_lib, "PK_ERR_" + code) and word in _lib.last_error()


def test_nothing_to_do_is_no_error():
    """No tokens or no sequences: no device call."""
    for b in (paged_batch(tokens=0), paged_batch(sequences=0, page_table=None, kv_len=None)):
        assert append_call(batch=b) == _lib.PK_OK and attend_call(batch=b) == _lib.PK_OK
    assert rotary_call(S=0) == _lib.PK_OK and rotary_call(H=0) == _lib.PK_OK


# ---- the torch front end --------------------------------------------------------------
def cpu(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("call,error,word", [
    (lambda: kernels.rotary(cpu(4, 2, 64), i32(4), cpu(32, dtype=torch.float64)), ValueError, "x: tensor must live on a GPU"),
    (lambda: kernels.rotary(cpu(4, 2, 64, dtype=torch.float32), i32(4), None), TypeError, "bfloat16"),
    (lambda: kernels.rotary(cpu(4, 64), i32(4), None), ValueError, "tokens, heads, D"),
    (lambda: kernels.rotary(None, i32(4), None), ValueError, "tokens, heads, D"),
    (lambda: kernels.paged_kv_append(cpu(4, 2, 64), cpu(4, 2, 64), cpu(3, 2, 16, 64), cpu(3, 2, 16, 64), i32(1, 3), i32(2),
                                     i32(1)), ValueError, "k_cache: tensor must live on a GPU"),
    (lambda: kernels.paged_attention(cpu(4, 2, 64), cpu(3, 16, 64), cpu(3, 2, 16, 64), i32(1, 3), i32(2), i32(1)),
     ValueError, "k_cache: expected 4 dimensions"),
    (lambda: kernels.paged_attention(cpu(4, 2, 64), cpu(3, 2, 16, 64, dtype=torch.float16), None, None, None, None),
     TypeError, "k_cache"),
    (lambda: kernels.paged_attention(cpu(4, 2, 64), "cache", None, None, None, None), TypeError, "k_cache"),
])
def test_front_end_refuses(call, error, word):
    with pytest.raises(error, match=word):
        call()


# ---- which kernels take a call ----------------------------------------------------------
def attention_plan(q_heads=32, heads=8, dim=128, page_size=16, table_width=64, tokens=1, sequences=1, max_q=1, window=0,
                   max_kv=0):
    out = _lib.PagedPlan()
    cache = paged_cache(heads=heads, dim=dim, page_size=page_size, pages=1000)
    batch = paged_batch(table_width=table_width, tokens=tokens, sequences=sequences, max_q=max_q, max_kv=max_kv)
    _lib.check(_lib.load().pk_paged_attention_plan(q_heads, cache, batch, window, out), "pk_paged_attention_plan")
    return out


def test_plans():
    p = attention_plan()  # a step on up to 1024 keys
    assert (p.dim, p.whole, p.splits) == (128, 0, 0) and 1 < p.workgroups <= 1024
    p = attention_plan(table_width=20)  # up to 320 keys: items are not cut, and nothing merged
    assert p.whole == 1 and p.workgroups == 8 and p.splits == 0
    long = dict(table_width=512)
    assert attention_plan(q_heads=128, **long).splits == 0 and attention_plan(q_heads=136, **long).workgroups == 0  # 16 and 17 rows
    assert attention_plan(q_heads=256).splits == 0 and attention_plan(q_heads=264).workgroups == 0  # 32 and 33 of a short one
    assert attention_plan(sequences=64, tokens=64, table_width=125).whole == 1  # many items fill the machine uncut
    assert attention_plan(sequences=16, tokens=16, table_width=125).whole == 0
    p = attention_plan(tokens=2048, max_q=2048, table_width=512)
    assert p.workgroups == 0 and p.splits == 1 and p.items == (2048 * 4 // 128 + 1) * 8
    assert attention_plan(tokens=64, max_q=64, table_width=512).splits > 1
    mixed = dict(tokens=600, sequences=40, max_q=500)
    p = attention_plan(**mixed, table_width=512)
    assert p.workgroups > 1 and p.splits >= 1
    assert attention_plan(**mixed, table_width=512, window=512).workgroups == 0  # nobody reaches far
    assert attention_plan(**mixed, table_width=90).workgroups == 0
    assert attention_plan(**mixed, table_width=512, max_kv=1500).workgroups == 0
    assert attention_plan(tokens=600, sequences=4, max_q=150, table_width=512).workgroups == 0  # all as long as the hint
    for general in (dict(dim=20), dict(dim=320), dict(dim=1024)):
        assert attention_plan(**general).dim == 0
    # a line of steps that a 32-bit place cannot hold goes to the general kernel
    assert attention_plan(tokens=1 << 20, sequences=1 << 20, table_width=1 << 20, q_heads=64, heads=64).dim == 0


def test_a_window_needs_no_more_workspace():
    """The size is asked for without the window."""
    for tokens in (1, 40, 300, 3000):
        for width in (30, 100, 1000, 8000):
            for window in (1, 100, 1000, 5000, 50000):
                for dim in (64, 96, 256):
                    a = attention_plan(tokens=tokens, max_q=tokens, table_width=width, dim=dim)
                    b = attention_plan(tokens=tokens, max_q=tokens, table_width=width, dim=dim, window=window)
                    assert b.splits <= a.splits and b.workgroups <= a.workgroups and b.items <= a.items and b.whole == a.whole


def test_workspace_refused():
    c, b = paged_cache(k_page=2048, heads=2, dim=64), paged_batch(table_width=100)
    need = _lib.load().pk_paged_attention_workspace_size(4, c, b)
    assert need > 0
    for ws, room in ((None, 0), (None, need), (FAKE, need - 1), (FAKE + 8, need)):
        assert attend_call(cache=c, batch=b, ws=ws, ws_bytes=room) == _lib.PK_ERR_WORKSPACE
        assert "workspace" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(q_heads=3), dict(q_heads=0), dict(window=-1), dict(sequences=0)])
def test_plan_refused(kw):
    with pytest.raises(_lib.PolyKernelError, match="pk_paged_attention_plan"):
        attention_plan(**kw)


def test_packed_structures_are_the_structures():
    """The bytes that the front end passes are those of the ctypes structures, whose fields are the header's."""
    for cls in (_lib.Rotary, _lib.Tokens, _lib.PagedCache, _lib.PagedBatch):
        values = [0.5 if t is C.c_float else 3 * i + 1 for i, (_, t) in enumerate(cls._fields_)]
        assert cls.pack(*values) == bytes(cls(*values)) and len(cls.pack(*values)) == C.sizeof(cls)
