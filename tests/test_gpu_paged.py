"""Rotary positions, the paged append and paged attention against plain 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def pk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    from polykernel_amd import _lib, kernels

    _lib.load()
    return kernels


def ok(got, want, bound):
    """Every value within its bound (a call of its own, so that a failure prints a number)."""
    bad = ref.far(got, want, bound)
    assert bad == 0, f"{bad} of {got.numel()} values outside their bounds"


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


# ---- rotary -----------------------------------------------------------------
ROTARY = [
    # S, H, D, rot, interleaved, magnitude, first position
    (1, 1, 2, 2, False, 1.0, 0),
    (1, 32, 128, 128, False, 1.0, 4095),
    (1, 32, 128, 128, True, 1.0, 1000003),
    (7, 3, 64, 64, False, 1.0, 131071),
    (5, 5, 80, 32, True, 1.0, 9),
    (5, 5, 80, 32, False, 1.138, 2**31 - 6),
    (33, 2, 96, 40, False, 1.0, 17),
    (4, 3, 17, 6, False, 1.0, 100),
    (4, 3, 17, 6, True, 0.5, -7),
    (259, 9, 256, 256, False, 1.0, 0),
    (3, 2, 1024, 1024, True, 1.0, 77),
    (2, 1, 1000, 8, False, 1.0, 5),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("S,H,D,rot,interleaved,magnitude,first", ROTARY)
def test_rotary(pk, S, H, D, rot, interleaved, magnitude, first, inverse):
    g = gen(S * 31 + D + rot)
    turns, _ = pk.rotary_frequencies(rot, 10000.0)
    x = normal(g, S, H, D)
    pos = (first + torch.arange(S, device="cuda")).to(torch.int32)
    pos = pos[torch.randperm(S, device="cuda", generator=g)].contiguous()
    kw = dict(interleaved=interleaved, magnitude=magnitude)
    want = ref.rotate(x.double(), pos, turns, inverse=inverse, **kw)
    bound = ref.rotate_bound(x.double(), want, turns, **kw)
    got = pk.rotary(x, pos, turns, inverse=inverse, **kw)
    assert got.is_contiguous() and ref.far(got, want, bound) == 0
    y = x.clone()
    assert pk.rotary(y, pos, turns, inverse=inverse, out=y, **kw) is y and torch.equal(y, got)  # in place


@pytest.mark.parametrize("per_sequence", [False, True])
@pytest.mark.parametrize("B,H,S,D,rot", [(1, 4, 1, 64, 64), (3, 5, 19, 128, 64), (2, 2, 70, 72, 48)])
def test_rotary_heads_first(pk, B, H, S, D, rot, per_sequence):
    g = gen(B + S)
    turns, _ = pk.rotary_frequencies(rot, 500000.0)
    x = normal(g, B, H, S, D)
    pos = torch.randint(0, 100000, (B, S) if per_sequence else (S,), generator=g, device="cuda", dtype=torch.int32)
    got = pk.rotary(x, pos, turns)
    for b in range(B):
        rows = x[b].transpose(0, 1).double()
        want = ref.rotate(rows, pos[b] if per_sequence else pos, turns)
        ok(got[b].transpose(0, 1), want, ref.rotate_bound(rows, want, turns))


@pytest.mark.parametrize("offset", [0, 8, 1, 3])  # elements from a 16-byte boundary
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_rotary_strides_and_alignment(pk, offset, pad):
    """A part of a projection's output, and an output with room around every head that stays."""
    S, H, D, rot = 13, 4, 64, 64
    g = gen(offset * 10 + pad)
    turns, _ = pk.rotary_frequencies(rot)
    flat = normal(g, S * 3 * H * (D + pad) + offset)
    x = flat[offset:].view(S, 3 * H, D + pad)[:, H:2 * H, :D]
    room = torch.full((S * H * (D + 2 * pad) + 8,), 7.0, dtype=BF, device="cuda")
    out = room[offset:offset + S * H * (D + 2 * pad)].view(S, H, D + 2 * pad)[:, :, :D]
    pos = torch.arange(50, 50 + S, device="cuda", dtype=torch.int32)
    pk.rotary(x, pos, turns, out=out)
    want = ref.rotate(x.double(), pos, turns)
    ok(out, want, ref.rotate_bound(x.double(), want, turns))
    out.fill_(7.0)
    assert bool((room == 7.0).all())


def test_rotary_copies_passed_dims_and_keeps_no_numbers_apart(pk):
    """Passed dims keep their bits (NaN payloads, infinities, -0), and a NaN stays in its pair."""
    turns, _ = pk.rotary_frequencies(16)
    x = torch.zeros(2, 3, 48, dtype=BF, device="cuda")
    bits = x.view(torch.int16)
    bits[..., 16:] = torch.arange(32, device="cuda", dtype=torch.int16) + 0x7F70
    bits[1, 1, 20] = -32768
    x[0, 0, 3] = float("nan")
    got = pk.rotary(x, torch.tensor([0, 5], device="cuda", dtype=torch.int32), turns)
    assert torch.equal(got.view(torch.int16)[..., 16:], bits[..., 16:])
    nan = torch.isnan(got[0, 0, :16])
    assert nan.nonzero().flatten().tolist() == [3, 11]
    assert bool((got[1, :, :16] == 0).all())


def test_rotary_gradient(pk):
    """The inverse is the transposed map: column by column against differences (the map is linear, so
    a difference over one unit is exact), and against the gradient of the formula in 64 bits."""
    for D, rot, interleaved in [(32, 32, False), (40, 24, True)]:
        turns, _ = pk.rotary_frequencies(rot, 100.0)
        pos = torch.full((D,), 37, device="cuda", dtype=torch.int32)
        eye = torch.eye(D, device="cuda").to(BF)[:, None].contiguous()
        fwd = pk.rotary(eye, pos, turns, interleaved=interleaved, magnitude=1.25)[:, 0]
        back = pk.rotary(eye, pos, turns, interleaved=interleaved, magnitude=1.25, inverse=True)[:, 0]
        assert torch.equal(fwd, back.T)
        g = gen(D)
        x, dy = normal(g, D, 3, D).double().requires_grad_(), normal(g, D, 3, D)
        ref.rotate(x, pos, turns, interleaved, 1.25).backward(dy.double())
        dx = pk.rotary(dy, pos, turns, interleaved=interleaved, magnitude=1.25, inverse=True)
        ok(dx, x.grad, ref.rotate_bound(dy.double(), x.grad, turns, interleaved, 1.25))


# ---- paged caches -------------------------------------------------------------
def layout(g, kvs, P, spare=2, width=0):
    """A page table of shuffled pages for kvs keys each."""
    used = [-(-k // P) for k in kvs]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((len(kvs), max(used + [width, 1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), pages


def cache(g, pages, Hkv, P, D, rows_first=False, pad=0, std=1.0):
    if rows_first:
        return normal(g, pages, P, Hkv, D + pad, std=std).transpose(1, 2)[..., :D]
    return normal(g, pages, Hkv, P, D + pad, std=std)[..., :D]


def starts(qs):
    out = [0]
    for n in qs:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


APPEND = [
    # new tokens, keys, Hq, Hkv, D, rot, P, interleaved, rows_first, pad
    ([1], [1], 1, 1, 64, 64, 16, False, False, 0),
    ([1, 1, 1], [5, 16, 17], 8, 2, 128, 128, 16, False, False, 0),
    ([1, 0, 3, 40], [100, 7, 3, 41], 4, 4, 64, 32, 32, True, True, 0),
    ([37, 2, 5], [37, 64, 300], 6, 2, 80, 80, 8, False, True, 8),
    ([9, 1], [20, 33], 3, 1, 17, 6, 5, False, False, 0),
    ([300], [1000], 2, 1, 256, 256, 64, True, False, 0),
    ([11, 4], [11, 9], 5, 1, 96, 24, 1, False, False, 3),
    ([2] * 150, [70] * 150, 2, 1, 64, 64, 48, False, False, 0),
]


@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,rot,P,interleaved,rows_first,pad", APPEND)
def test_append(pk, qs, kvs, Hq, Hkv, D, rot, P, interleaved, rows_first, pad, rotated):
    g = gen(D + P + len(qs))
    table, pages = layout(g, kvs, P)
    T = sum(qs)
    qkv = normal(g, T + 3, Hq + 2 * Hkv, D)  # three tokens behind the last sequence's
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    kc, vc = (cache(g, pages, Hkv, P, D, rows_first, pad) for _ in range(2))
    kc0, vc0 = kc.clone(), vc.clone()
    turns, _ = pk.rotary_frequencies(rot)
    q_start, kv_len = starts(qs), torch.tensor(kvs, dtype=torch.int32, device="cuda")
    qo = torch.full((T + 3, Hq, D), 3.0, dtype=BF, device="cuda")
    where = (kc, vc, table, q_start, kv_len)
    if rotated:
        kw = dict(interleaved=interleaved, magnitude=1.07)
        assert pk.paged_kv_append(k, v, *where, q=q, turns=turns, q_out=qo, **kw) is qo
    else:
        assert pk.paged_kv_append(k, v, *where) is None
    spots = ref.places(q_start, kv_len, table, P, T)
    pos = torch.tensor([p for _, _, p in spots], device="cuda")
    want_k, want_v = kc0.double(), vc0.double()
    bound = torch.zeros_like(want_k)
    if rotated:
        want = ref.rotate(q[:T].double(), pos, turns, **kw)
        ok(qo[:T], want, ref.rotate_bound(q[:T].double(), want, turns, **kw))
        new = ref.rotate(k[:T].double(), pos, turns, **kw)
        off = ref.rotate_bound(k[:T].double(), new, turns, **kw)
    else:
        new, off = k[:T].double(), torch.zeros(T, Hkv, D, dtype=torch.float64, device="cuda")
    host = table.cpu()
    for t, b, p in spots:
        page = int(host[b, p // P])
        want_k[page, :, p % P], bound[page, :, p % P] = new[t], off[t]
        want_v[page, :, p % P] = v[t].double()
    ok(kc, want_k, bound)
    assert torch.equal(vc.double(), want_v)
    assert bool((qo[T:] == 3.0).all())


def test_append_one_token_each_without_starts(pk):
    g = gen(1)
    kvs, P, Hkv, D = [1, 50, 17, 16], 16, 2, 64
    table, pages = layout(g, kvs, P)
    k, v, q = normal(g, 4, Hkv, D), normal(g, 4, Hkv, D), normal(g, 4, 6, D)
    kv_len = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    turns, _ = pk.rotary_frequencies(D)
    a, b = (torch.zeros(2, pages, Hkv, P, D, dtype=BF, device="cuda") for _ in range(2))
    qa = pk.paged_kv_append(k, v, a[0], a[1], table, starts([1] * 4), kv_len, q=q, turns=turns)
    qb = pk.paged_kv_append(k, v, b[0], b[1], table, None, kv_len, q=q, turns=turns)
    assert torch.equal(a, b) and torch.equal(qa, qb)
    assert torch.equal(pk.rotary(q, kv_len - 1, turns), qa)  # the same rotation


def test_append_leaves_what_is_not_there(pk):
    """Pages outside the cache, keys fewer than new tokens, a table too short: nothing is written for them."""
    P, Hkv, D = 16, 1, 64
    kc = torch.zeros(3, Hkv, P, D, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.tensor([[0, -1], [3, 1], [2, 2**31 - 1]], dtype=torch.int32, device="cuda")
    k = torch.ones(9, Hkv, D, dtype=BF, device="cuda")
    q_start = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device="cuda")
    # positions 15-17 (16 and 17 on page -1), 14-16 (14 and 15 on page 3 of 3), -1, 0 and 1
    kv_len = torch.tensor([18, 17, 2], dtype=torch.int32, device="cuda")
    pk.paged_kv_append(k, k, kc, vc, table, q_start, kv_len)
    want = torch.zeros_like(kc)
    want[0, :, 15] = 1
    want[1, :, 0] = 1
    want[2, :, 0:2] = 1
    assert torch.equal(kc, want) and torch.equal(vc, want)
    # lengths above the table's reach stop there: positions 30 and 31 of 32
    kc.zero_(), vc.zero_()
    pk.paged_kv_append(k[:2], k[:2], kc, vc, table[:1], q_start[:2].clamp(max=2), torch.full((1,), 10**9, dtype=torch.int32, device="cuda"))
    assert bool((kc == 0).all())
    pk.paged_kv_append(k[:2], k[:2], kc, vc, table[1:2], torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
                       torch.full((1,), 10**9, dtype=torch.int32, device="cuda"))
    want.zero_()
    want[1, :, 14:] = 1
    assert torch.equal(kc, want)


# ---- attention ------------------------------------------------------------------
def run(pk, qs, kvs, Hq, Hkv, D, P, *, window=0, causal=True, rows_first=False, pad=0, std=1.0, seed=0, scale=None,
        max_q=None, max_kv=0, spoil=None, behind=0, single=False):
    g = gen(seed + D + P)
    table, pages = layout(g, kvs, P)
    T = sum(qs)
    q = normal(g, T + behind, Hq, D, std=std)
    kc, vc = (cache(g, pages, Hkv, P, D, rows_first, pad) for _ in range(2))
    q_start = None if single else starts(qs)
    kv_len = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    if spoil:
        spoil(kc, vc, table)
    out = torch.full((T + behind, Hq, D), 5.0, dtype=BF, device="cuda")
    where = (kc, vc, table, q_start, kv_len)
    pk.paged_attention(q, *where, max_q=max_q, max_kv=max_kv, window=window, causal=causal, scale=scale, out=out)
    s = scale if scale is not None else 1.0 / math.sqrt(D)
    want, bound = ref.attend(q[:T], kc, vc, table, q_start, kv_len, s, causal, window)
    assert bool((out[T:] == 5.0).all())
    ok(out[:T], want, bound)
    return out


SHAPES = [
    # new tokens, keys, Hq, Hkv, D, P
    ([1], [1], 1, 1, 64, 16),
    ([1], [200], 32, 8, 128, 16),
    ([1], [17], 4, 4, 128, 16),
    ([1, 1, 1, 1], [1, 16, 1000, 333], 8, 2, 128, 32),
    ([1] * 70, [3 + 7 * i for i in range(70)], 4, 1, 64, 16),
    ([1, 1], [4097, 9000], 16, 2, 128, 256),
    ([1], [2500], 7, 1, 128, 16),
    ([1, 1], [600, 31], 24, 1, 128, 64),
    ([1], [700], 64, 1, 64, 16),
    ([1, 1], [300, 20], 71, 1, 64, 16),
    ([1, 1], [260, 77], 12, 4, 256, 16),
    ([1, 1], [260, 77], 6, 2, 80, 16),
    ([1, 1], [130, 5], 6, 2, 96, 48),
    ([3, 5, 1], [500, 5, 64], 8, 2, 128, 16),
    ([4] * 9, [4 + 50 * i for i in range(9)], 32, 8, 128, 32),
    ([7, 8], [900, 8], 32, 4, 64, 16),
    ([130], [130], 4, 4, 128, 16),
    ([257, 1, 64], [300, 900, 64], 8, 2, 128, 64),
    ([100, 0, 33, 1], [1000, 50, 33, 257], 6, 1, 64, 16),
    ([129], [520], 3, 1, 256, 32),
    ([513], [1100], 4, 1, 128, 128),
    ([65, 200], [65, 777], 14, 2, 96, 16),
    ([90, 3], [95, 400], 4, 4, 72, 16),
    ([1, 20], [50, 40], 4, 2, 128, 8),
    ([40, 1], [120, 77], 8, 2, 64, 1),
    ([5], [21], 2, 2, 128, 24),
    ([70, 2], [90, 300], 4, 2, 64, 40),
    ([3, 1], [40, 9], 4, 2, 17, 5),
    ([2], [30], 2, 1, 512, 16),
    ([2, 1], [70, 3], 3, 3, 1024, 7),
]


@pytest.mark.parametrize("std", [1.0, 6.0])  # flat and peaked weights
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,P", SHAPES)
def test_attention(pk, qs, kvs, Hq, Hkv, D, P, std):
    run(pk, qs, kvs, Hq, Hkv, D, P, std=std, behind=2)


@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,P", SHAPES[1:26:3])
def test_attention_rows_first_and_hints(pk, qs, kvs, Hq, Hkv, D, P):
    """The other cache layout, and a hint that is too small, too large or none: rows stay within their bounds."""
    outs = [run(pk, qs, kvs, Hq, Hkv, D, P, rows_first=True, max_q=m, std=2.0) for m in (None, 0, 1, 64, 4096)]
    assert len(outs) == 5


def plan(qs, kvs, Hq, Hkv, D, P, max_q, window=0, max_kv=0):
    from tests.test_paged_host import attention_plan

    return attention_plan(q_heads=Hq, heads=Hkv, dim=D, page_size=P, table_width=-(-max(kvs) // P), tokens=sum(qs),
                          sequences=len(qs), max_q=max_q, window=window, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", [1, 64, 1500, 10**9])
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,P", [([1] * 40, [1 + 70 * i for i in range(40)], 8, 2, 128, 16),
                                               ([60, 1, 30], [1700, 900, 30], 8, 2, 64, 16), ([20], [1500], 4, 1, 256, 8)])
def test_attention_with_wrong_numbers_of_keys(pk, qs, kvs, Hq, Hkv, D, P, max_kv):
    run(pk, qs, kvs, Hq, Hkv, D, P, std=2.0, max_kv=max_kv)


@pytest.mark.parametrize("Hq,Hkv,D,P", [(16, 2, 128, 16), (24, 2, 64, 32), (16, 2, 96, 8), (12, 1, 256, 16)])
def test_many_sequences_of_few_tokens(pk, Hq, Hkv, D, P):
    """More sequences than a wave has lanes in the chunk kernel; most waves have no rows, and short sequences are not
    cut where long ones are."""
    qs = [1 + i % 5 for i in range(90)]
    kvs = [q + 25 * i for i, q in enumerate(qs)]
    got = plan(qs, kvs, Hq, Hkv, D, P, 5)
    assert got.splits > 1 and got.workgroups == 0
    run(pk, qs, kvs, Hq, Hkv, D, P, std=2.0, max_q=5, behind=1)


@pytest.mark.parametrize("whole,kvs", [(1, [1 + 33 * i for i in range(64)]), (0, [1 + 35 * i for i in range(64)])])
@pytest.mark.parametrize("Hq,Hkv,D,P", [(8, 8, 128, 16), (16, 8, 64, 8)])
def test_items_cut_and_whole(pk, Hq, Hkv, D, P, whole, kvs):
    assert plan([1] * 64, kvs, Hq, Hkv, D, P, 1).whole == whole
    run(pk, [1] * 64, kvs, Hq, Hkv, D, P, std=2.0)


@pytest.mark.parametrize("D,P", [(128, 16), (64, 8)])
def test_two_items_for_a_short_run(pk, D, P):
    """17 to 32 rows of one short sequence are the step kernel's."""
    for q in (5, 8):
        assert plan([q], [900], 8, 2, D, P, q).splits == 0
        run(pk, [q], [900], 8, 2, D, P, std=2.0)


@pytest.mark.parametrize("window", [0, 2200])
@pytest.mark.parametrize("Hq,Hkv,D,P", [(8, 2, 128, 16), (4, 4, 64, 32), (6, 1, 80, 48), (4, 2, 256, 64), (16, 2, 96, 8),
                                        (3, 1, 192, 16)])
def test_chunks_beside_single_tokens(pk, Hq, Hkv, D, P, window):
    """Both kernels in one call: sequences of up to 16 rows by one, the others by the other."""
    few = 16 // (Hq // Hkv)
    qs = [200, 1, 3, few, 0, few + 1, 1] + [1] * 80
    kvs = [2600, 2303, 3, 1000, 7, 100, 40] + [5000] + [5 + 3 * i for i in range(79)]
    got = plan(qs, kvs, Hq, Hkv, D, P, max(qs), window)
    assert got.splits > 0 and (got.workgroups > 0 or Hkv == 1 or window)  # (few short items stay with the chunks)
    run(pk, qs, kvs, Hq, Hkv, D, P, std=2.0, max_q=max(qs), window=window, behind=1)


@pytest.mark.parametrize("Hq,Hkv,D,P", [(8, 2, 128, 16), (2, 1, 64, 8), (40, 1, 64, 16), (24, 1, 128, 16), (5, 1, 256, 16)])
def test_many_sequences_cut_between_workgroups(pk, Hq, Hkv, D, P):
    """More sequences than lanes of a wave, of very different lengths, two without new tokens."""
    qs = [0 if i in (0, 99) else 1 + (i % 7 == 0) for i in range(150)]
    kvs = [max(1, (i * 977) % 1400) + 2 for i in range(150)]
    kvs[31] = 9000
    got = plan(qs, kvs, Hq, Hkv, D, P, 1)
    assert got.workgroups > 1 and not got.whole or Hq // Hkv > 8  # (more than 16 rows of two tokens are a chunk)
    run(pk, qs, kvs, Hq, Hkv, D, P, std=2.0, max_q=1)


@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (96, 8), (256, 16)])
@pytest.mark.parametrize("q,kv", [(100, 3000), (33, 5000), (300, 1500)])
def test_chunks_cut_along_their_keys(pk, q, kv, D, P):
    got = plan([q], [kv], 4, 1, D, P, q)
    assert got.splits > 1 and got.workgroups == 0
    run(pk, [q], [kv], 4, 1, D, P, std=2.0, max_q=q)
    run(pk, [q], [kv], 4, 1, D, P, std=2.0, max_q=q, window=700)


@pytest.mark.parametrize("gone", [False, True])
@pytest.mark.parametrize("P", [1, 4, 8, 12, 20, 24, 40])
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D", [([1, 3, 1], [3000, 70, 801], 8, 2, 128), ([1, 1], [2500, 9], 4, 1, 64),
                                             ([1], [1700], 4, 2, 256), ([300, 20], [2100, 700], 6, 1, 64),
                                             ([150], [1500], 4, 2, 96)])
def test_page_sizes_that_end_inside_a_tile(pk, qs, kvs, Hq, Hkv, D, P, gone):
    """With long runs of keys, pages that are not there and no numbers on the rows behind the keys."""
    def spoil(kc, vc, table):
        for b, n in enumerate(kvs):
            if n % P:
                kc[int(table[b, n // P]), :, n % P:], vc[int(table[b, n // P]), :, n % P:] = float("nan"), float("nan")
            table[b, 1:n // P:7] = -1 - b

    run(pk, qs, kvs, Hq, Hkv, D, P, std=2.0, spoil=spoil if gone else None)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 200, 100000])
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,P", [([1, 1, 1], [1, 70, 1000], 8, 2, 128, 16),
                                               ([5, 2], [300, 40], 8, 2, 64, 32),
                                               ([300, 1], [420, 900], 4, 2, 128, 16),
                                               ([40, 9], [50, 77], 4, 1, 64, 5),
                                               ([3], [40], 4, 2, 20, 16)])
def test_attention_window(pk, qs, kvs, Hq, Hkv, D, P, window):
    run(pk, qs, kvs, Hq, Hkv, D, P, window=window, std=3.0)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("qs,kvs,Hq,Hkv,D,P", [([1, 4], [70, 100], 8, 2, 128, 16), ([200, 3], [300, 200], 4, 2, 64, 16),
                                               ([6], [9], 2, 1, 12, 4)])
def test_attention_without_causal_mask(pk, qs, kvs, Hq, Hkv, D, P, window):
    run(pk, qs, kvs, Hq, Hkv, D, P, causal=False, window=window, std=2.0)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30])
@pytest.mark.parametrize("qs,kvs", [([1, 1], [100, 33]), ([100], [260])])
def test_attention_scales(pk, qs, kvs, scale):
    run(pk, qs, kvs, 4, 2, 128, 16, scale=scale)


@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("qs,kvs", [([4, 1, 3], [2, 0, 3]), ([200, 1, 64], [130, 0, 10])])
def test_rows_that_see_nothing_are_zero(pk, qs, kvs, D):
    """More new tokens than keys: the first ones see nothing; a sequence without keys neither."""
    out = run(pk, qs, kvs, 4, 2, D, 16)
    empty = qs[0] - kvs[0]
    assert bool((out[:empty] == 0).all()) and bool((out[qs[0]:qs[0] + qs[1]] == 0).all())


@pytest.mark.parametrize("D,P", [(128, 16), (64, 48), (128, 8), (20, 16)])
@pytest.mark.parametrize("qs,kvs", [([1, 1], [100, 263]), ([3, 4], [50, 119]), ([150, 70], [301, 70])])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_rows_behind_the_keys_take_no_part(pk, qs, kvs, D, P, what):
    """Whatever unused rows and unlisted pages hold."""
    def spoil(kc, vc, table):
        used = torch.zeros(kc.shape[0], P, dtype=torch.bool, device="cuda")
        for b, kv in enumerate(kvs):
            j = torch.arange(kv, device="cuda")
            used[table[b][j // P].long(), j % P] = True
        for c in (kc, vc):
            c.transpose(1, 2)[~used] = what
    run(pk, qs, kvs, 4, 2, D, P, spoil=spoil)


@pytest.mark.parametrize("D,P", [(128, 16), (64, 8), (20, 16)])
@pytest.mark.parametrize("qs,kvs", [([1], [40]), ([5], [50]), ([40], [60]), ([150], [400])])
def test_values_that_are_no_numbers_show_only_to_tokens_that_see_them(pk, qs, kvs, D, P):
    """A NaN in the values of the last key, an infinity in those before; a NaN in keys: later tokens' alone."""
    for where in (1, 3):
        if qs[0] <= where:
            continue

        def spoil(kc, vc, table):
            kv = kvs[0]
            for j, c, what in ((kv - 1, vc, float("nan")), (kv - where, vc, float("-inf")), (kv - 1, kc, float("nan"))):
                c[int(table[0, j // P]), 0, j % P, 3] = what
        run(pk, qs, kvs, 4, 2, D, P, spoil=spoil)

    def old(kc, vc, table):  # behind the window of every token but the first
        j = kvs[0] - qs[0] - 9
        for c in (kc, vc):
            c[int(table[0, j // P]), :, j % P] = float("nan")
    run(pk, qs, kvs, 4, 2, D, P, spoil=old, window=10)


@pytest.mark.parametrize("D,P", [(128, 16), (64, 32), (128, 8), (20, 16)])
@pytest.mark.parametrize("qs,kvs", [([1, 1], [100, 263]), ([3, 4], [50, 119]), ([150, 70], [301, 70])])
def test_pages_that_are_not_there_take_no_part(pk, qs, kvs, D, P):
    def spoil(kc, vc, table):
        table[0, 0], table[0, 2] = -1, kc.shape[0]
        table[1, :] = 2**31 - 1
    run(pk, qs, kvs, 4, 2, D, P, spoil=spoil)


def test_tables_out_of_range_are_brought_into_range(pk):
    g = gen(3)
    table, pages = layout(g, [100, 100], 16)
    kc, vc, q = cache(g, pages, 2, 16, 64), cache(g, pages, 2, 16, 64), normal(g, 6, 4, 64)
    out = torch.full_like(q, 5.0)
    q_start = torch.tensor([-4, 3, 100], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([-5, 10**9], dtype=torch.int32, device="cuda")
    pk.paged_attention(q, kc, vc, table, q_start, kv_len, out=out)
    want, bound = ref.attend(q, kc, vc, table, starts([3, 3]), torch.tensor([0, table.shape[1] * 16]), 0.125)
    ok(out, want, bound)
    out.fill_(5.0)
    pk.paged_attention(q, kc, vc, table, torch.tensor([4, 2, 1], dtype=torch.int32, device="cuda"), kv_len, out=out)
    assert bool((out == 5.0).all())


@pytest.mark.parametrize("offset,pad", [(1, 0), (0, 3), (8, 8), (4, 4)])
@pytest.mark.parametrize("qs,kvs", [([1, 2], [90, 40]), ([130], [200])])
def test_attention_strides_and_alignment(pk, qs, kvs, offset, pad):
    Hq, Hkv, D, P = 4, 2, 64, 16
    g = gen(offset + pad)
    table, pages = layout(g, kvs, P)
    T = sum(qs)

    def part(*shape):
        n = math.prod(shape[:-1]) * (shape[-1] + pad)
        return normal(g, n + offset)[offset:].view(*shape[:-1], shape[-1] + pad)[..., :shape[-1]]
    q, kc, vc, out = part(T, Hq, D), part(pages, Hkv, P, D), part(pages, P, Hkv, D).transpose(1, 2), part(T, Hq, D)
    q_start, kv_len = starts(qs), torch.tensor(kvs, dtype=torch.int32, device="cuda")
    pk.paged_attention(q, kc, vc, table, q_start, kv_len, out=out)
    want, bound = ref.attend(q, kc, vc, table, q_start, kv_len, 0.125)
    ok(out, want, bound)


@pytest.mark.parametrize("D", [8, 16, 40, 136, 200, 248])
@pytest.mark.parametrize("qs,kvs", [([1, 2], [400, 33]), ([70], [300])])
def test_head_dims_that_fill_no_tile(pk, qs, kvs, D):
    run(pk, qs, kvs, 6, 2, D, 16, std=2.0, behind=1)


@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("qs,kvs", [([1] * 1000, [1 + i % 97 for i in range(1000)]),
                                    ([3] * 300, [3 + i % 211 for i in range(300)]),
                                    ([0] * 500 + [40] + [0] * 499, [9] * 500 + [200] + [0] * 499)])
def test_very_many_sequences(pk, qs, kvs, D):
    run(pk, qs, kvs, 8, 1, D, 16, max_q=max(qs))


@pytest.mark.parametrize("D", [128, 20])
@pytest.mark.parametrize("n,single", [(1, True), (5, False), (60, False)])
def test_sequences_that_share_pages(pk, n, single, D):
    """One table for all sequences (a stride of 0), and caches whose strides differ."""
    g = gen(21)
    B, Hq, Hkv, P, kv = 5, 8, 2, 16, 333
    table, pages = layout(g, [kv], P)
    table = table.expand(B, -1)
    kc, vc = cache(g, pages, Hkv, P, D, rows_first=True, pad=8), cache(g, pages, Hkv, P, D)
    q, kv_len = normal(g, B * n, Hq, D), torch.tensor([kv, 60, 200, 111, 300], dtype=torch.int32, device="cuda")
    q_start = None if single else starts([n] * B)
    out = pk.paged_attention(q, kc, vc, table, q_start, kv_len, max_q=n)
    want, bound = ref.attend(q, kc, vc, table, starts([n] * B), kv_len, 1 / math.sqrt(D))
    ok(out, want, bound)


def test_offsets_past_32_bits(pk):
    """Caches of over 2^32 elements whose far pages are used, by append and attention."""
    Hkv, P, D, Hq = 4, 64, 128, 8
    pages = (2**32) // (Hkv * P * D) + 9
    for kvs, qs in (([300, 70], [1, 1]), ([300, 200], [120, 70])):
        g = gen(7)
        kc = torch.empty(pages, Hkv, P, D, dtype=BF, device="cuda")
        vc = torch.empty(pages, Hkv, P, D, dtype=BF, device="cuda")
        table = torch.full((2, 5), -1, dtype=torch.int32)
        table[0] = torch.tensor([pages - 1, 3, pages // 2 + 1, pages - 5, 0])
        table[1, :4] = torch.tensor([pages - 2, pages - 3, pages // 2, 5])
        for p in table[table >= 0].tolist():
            kc[p], vc[p] = normal(g, Hkv, P, D), normal(g, Hkv, P, D)
        table = table.cuda()
        T = sum(qs)
        q, k, v = normal(g, T, Hq, D), normal(g, T, Hkv, D), normal(g, T, Hkv, D)
        q_start, kv_len = starts(qs), torch.tensor(kvs, dtype=torch.int32, device="cuda")
        pk.paged_kv_append(k, v, kc, vc, table, q_start, kv_len)
        host = table.cpu()
        for t, b, p in ref.places(q_start, kv_len, table, P, T):
            assert torch.equal(kc[int(host[b, p // P]), :, p % P], k[t]) and torch.equal(vc[int(host[b, p // P]), :, p % P], v[t])
        out = pk.paged_attention(q, kc, vc, table, q_start, kv_len, max_q=max(qs))
        want, bound = ref.attend(q, kc, vc, table, q_start, kv_len, 1 / math.sqrt(D))
        ok(out, want, bound)
        del kc, vc


# ---- together, as a server uses them ----------------------------------------------
@pytest.mark.parametrize("D,Hq,Hkv,P,interleaved", [(128, 8, 2, 16, False), (64, 6, 6, 8, True), (20, 2, 1, 16, False)])
def test_serving_run(pk, D, Hq, Hkv, P, interleaved):
    """A prompt in chunks and decode steps of three sequences, pages handed out as they grow; every
    step's attention against the 64-bit form over all tokens so far."""
    g = gen(D)
    B, width = 3, 64
    steps = [[40, 7, 130], [90, 0, 1], [1, 1, 1], [1, 1, 1], [3, 1, 2], [0, 0, 1]]
    pages = B * width
    free = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    kc, vc = (torch.full((pages, Hkv, P, D), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    turns, mag = pk.rotary_frequencies(D, 10000.0, "ramp", 4.0, 1.0, 32.0, 64)
    lens = [0] * B
    keys, values = [[] for _ in range(B)], [[] for _ in range(B)]
    for qs in steps:
        T = sum(qs)
        qkv = normal(g, T, Hq + 2 * Hkv, D)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        at = 0
        want = torch.empty(T, Hq, D, dtype=torch.float64, device="cuda")
        bound = torch.empty_like(want)
        for b, n in enumerate(qs):
            for p in range(-(-lens[b] // P), -(-(lens[b] + n) // P)):
                table[b, p] = free.pop()
            lens[b] += n
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            rows = slice(at, at + n)
            # what the append stores, in bf16; the attention is compared over the stored values
            keys[b].append(ref.rotate(k[rows].double(), pos, turns, interleaved, mag))
            values[b].append(v[rows].double())
            at += n
        dt, q_start = table.cuda(), starts(qs)
        kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        qr = pk.paged_kv_append(k, v, kc, vc, dt, q_start, kv_len, q=q, turns=turns, interleaved=interleaved, magnitude=mag)
        out = pk.paged_attention(qr, kc, vc, dt, q_start, kv_len, max_q=max(qs))
        for b in range(B):  # the cache holds every token so far
            j = torch.arange(lens[b], device="cuda")
            stored = kc[dt[b][j // P].long(), :, j % P]
            whole = torch.cat(keys[b])
            assert bool(((stored.double() - whole).abs() <= whole.abs() * 2.0**-8 + 2.0**-17).all())
            assert torch.equal(vc[dt[b][j // P].long(), :, j % P].double(), torch.cat(values[b]))
        want, bound = ref.attend(qr, kc, vc, dt, q_start, kv_len, 1 / math.sqrt(D))
        ok(out, want, bound)


def test_whole_prompt_equals_contiguous_attention(pk):
    """A prompt through pages and the framework's attention over a contiguous cache agree within both bounds."""
    g = gen(11)
    B, H, S, D, P = 2, 4, 150, 128, 16
    k, v, q = (normal(g, B, H, S, D) for _ in range(3))
    flat = lambda t: t.transpose(1, 2).reshape(B * S, H, D)  # noqa: E731
    table, pages = layout(g, [S] * B, P)
    kc, vc = (torch.empty(pages, H, P, D, dtype=BF, device="cuda") for _ in range(2))
    q_start, kv_len = starts([S] * B), torch.full((B,), S, dtype=torch.int32, device="cuda")
    pk.paged_kv_append(flat(k), flat(v), kc, vc, table, q_start, kv_len)
    got = pk.paged_attention(flat(q), kc, vc, table, q_start, kv_len, max_q=S)
    want, bound = ref.attend(flat(q), kc, vc, table, q_start, kv_len, 1 / math.sqrt(D))
    other = flat(pk.attention_prefill(q, k, v))
    assert bool(((got.double() - other.double()).abs() <= 2 * bound).all())


def test_steps_in_a_captured_graph(pk):
    """Append and attention captured once and replayed while lengths, tables and tokens change, with eager calls
    between; two graphs that were captured on one stream replayed on two."""
    g = gen(5)
    B, Hq, Hkv, D, P, width = 5, 8, 2, 128, 16, 40
    table = torch.randperm(B * width, generator=g, device="cuda").to(torch.int32).view(B, width)
    kc, vc = (normal(g, B * width, Hkv, P, D) for _ in range(2))
    turns, _ = pk.rotary_frequencies(D)
    state = []
    stream = torch.cuda.Stream()
    for n in (1, 40):
        q, k, v = normal(g, B * n, Hq, D), normal(g, B * n, Hkv, D), normal(g, B * n, Hkv, D)
        kcg, vcg = kc.clone(), vc.clone()
        q_start, kv_len = starts([n] * B), torch.full((B,), 100, dtype=torch.int32, device="cuda")
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            qr = pk.paged_kv_append(k, v, kcg, vcg, table, q_start, kv_len, q=q, turns=turns)
            out = pk.paged_attention(qr, kcg, vcg, table, q_start, kv_len, max_q=n)
        state.append((graph, n, q, k, v, kcg, vcg, q_start, kv_len, out))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for graph, n, q, k, v, kcg, vcg, q_start, kv_len, out in state:
            kv_len.copy_(torch.randint(n, width * P, (B,), generator=g, device="cuda", dtype=torch.int32))
            q.copy_(normal(g, B * n, Hq, D))
            k.copy_(normal(g, B * n, Hkv, D))
        torch.cuda.synchronize()
        for s, st in zip(side, state):
            with torch.cuda.stream(s):
                st[0].replay()
        torch.cuda.synchronize()
        for graph, n, q, k, v, kcg, vcg, q_start, kv_len, out in state:
            replayed, kk = out.clone(), kcg.clone()
            qr = pk.paged_kv_append(k, v, kcg, vcg, table, q_start, kv_len, q=q, turns=turns)
            eager = pk.paged_attention(qr, kcg, vcg, table, q_start, kv_len, max_q=n)
            assert torch.equal(replayed, eager) and torch.equal(kk, kcg)
            want, bound = ref.attend(qr, kcg, vcg, table, q_start, kv_len, 1 / math.sqrt(D))
            ok(eager, want, bound)


def test_calls_on_several_streams(pk):
    """Calls that overlap on two streams keep their results, and one call gives the same bits every time."""
    g = gen(9)
    kvs = [3000 + 37 * i for i in range(6)]
    table, pages = layout(g, kvs, 16)
    kc, vc = (cache(g, pages, 2, 16, 128) for _ in range(2))
    kv_len = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    qs = [normal(g, 6, 16, 128) for _ in range(4)]
    alone = [pk.paged_attention(q, kc, vc, table, None, kv_len) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        outs = []
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(pk.paged_attention(q, kc, vc, table, None, kv_len))
        torch.cuda.synchronize()
        for a, o in zip(alone, outs):
            assert torch.equal(a, o)


def test_empty_calls(pk):
    turns, _ = pk.rotary_frequencies(64)
    none = torch.empty(0, 4, 64, dtype=BF, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert pk.rotary(none, i32(), turns).shape == (0, 4, 64)
    kc = torch.zeros(2, 4, 16, 64, dtype=BF, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    pk.paged_kv_append(none, none, kc, kc, table, i32(0, 0), i32(5))
    assert pk.paged_attention(none, kc, kc, table, i32(0, 0), i32(5)).shape == (0, 4, 64)
    assert pk.paged_attention(none, kc, kc, table[:0], i32(0), i32()).shape == (0, 4, 64)
    # a table and a cache without pages: no key is there
    q = torch.ones(1, 4, 64, dtype=BF, device="cuda")
    assert bool((pk.paged_attention(q, kc[:0], kc[:0], table, i32(0, 1), i32(9)) == 0).all())
    assert bool((pk.paged_attention(q, kc, kc, table[:, :0], i32(0, 1), i32(9)) == 0).all())
    torch.cuda.synchronize()


def test_numbers_and_workspaces_refused(pk):
    q, c = (torch.zeros(*s, dtype=BF, device="cuda") for s in ((4, 2, 64), (3, 2, 16, 64)))
    where = (c, c, *(torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((1, 3), (2,), (1,))))
    for kw in (dict(window=2**32 + 5), dict(max_q=2**31), dict(max_kv=2**40), dict(window=-2**32 + 5)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            pk.paged_attention(q, *where, **kw)
    room = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="workspace"):
        pk.paged_attention(q, *where, workspace=room[::2])


def test_front_end_refusals(pk):
    """Shapes, types and strides that do not fit each other, before any launch."""
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    turns = z(32, dtype=torch.float64)
    x, k, c = z(4, 2, 64), z(4, 2, 64), z(3, 2, 16, 64)
    good = dict(k_cache=c, v_cache=c, page_table=i32(1, 3), q_start=i32(2), kv_len=i32(1))

    def bad(fn, *a, error=ValueError, match="", **kw):
        with pytest.raises(error, match=match):
            fn(*a, **kw)

    bad(pk.rotary, x, i32(5), turns, match="positions")
    bad(pk.rotary, x, i32(4).long(), turns, error=TypeError, match="positions")
    bad(pk.rotary, x, i32(4).cpu(), turns, match="positions")
    bad(pk.rotary, x, i32(8)[::2], turns, match="positions")
    bad(pk.rotary, z(2, 2, 4, 64), i32(3, 4), turns, match="positions")
    bad(pk.rotary, x, i32(4), turns.float(), error=TypeError, match="turns")
    bad(pk.rotary, x, i32(4), turns[None], match="turns")
    bad(pk.rotary, x, i32(4), None, error=TypeError, match="turns")
    bad(pk.rotary, x, i32(4), z(33, dtype=torch.float64), error=Exception, match="rotated")
    bad(pk.rotary, x.transpose(1, 2), i32(4), turns, match="contiguous")
    bad(pk.rotary, x, i32(4), turns, out=z(4, 2, 32), match="out")
    bad(pk.rotary, x, i32(4), turns, out=z(4, 2, 64, dtype=torch.float16), error=TypeError, match="out")
    for kw, match in [(dict(v_cache=z(3, 2, 8, 64)), "same shape"), (dict(page_table=i32(2, 3)), "page_table"),
                      (dict(page_table=i32(1, 6)[:, ::2]), "page_table"), (dict(q_start=i32(3)), "q_start"),
                      (dict(q_start=None), "q_start"), (dict(kv_len=i32(1, 1)), "kv_len"),
                      (dict(k_cache=z(3, 2, 64, 16).transpose(2, 3), v_cache=z(3, 2, 64, 16).transpose(2, 3)), "contiguous")]:
        bad(pk.paged_kv_append, k, k, **{**good, **kw}, match=match)
        bad(pk.paged_attention, x, **{**good, **kw}, match=match)
    bad(pk.paged_kv_append, k, z(4, 3, 64), **good, match="v: ")
    bad(pk.paged_kv_append, z(4, 2, 32), k, **good, match="k: ")
    bad(pk.paged_kv_append, k, k, q=x, **good, match="turns")
    bad(pk.paged_kv_append, k, k, q_out=x, turns=turns, **good, match="q_out")
    bad(pk.paged_kv_append, k, k, q=x, q_out=z(4, 3, 64), turns=turns, **good, match="q_out")
    bad(pk.paged_attention, z(4, 3, 64), **good, error=Exception, match="query heads")
    bad(pk.paged_attention, x, window=-1, **good, error=Exception, match="window")
    bad(pk.paged_attention, x, out=z(5, 2, 64), **good, match="out")
    bad(pk.paged_attention, x, workspace=torch.zeros(8), **good, match="workspace")
