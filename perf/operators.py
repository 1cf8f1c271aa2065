"""Serving from a paged key/value cache: the rotation of positions, the append of
new keys and values (rotated on the way) into pages, and attention of the new
tokens over the pages, as a program that serves many sequences calls them.

  rotary   rotate the heads of a tensor by their positions; `inverse` is the
           transposed rotation, which is its gradient
  append   queries rotated, keys rotated into the pages, values into the pages
  attend   attention of one new token, a few or a chunk per sequence over pages

Tokens of all sequences lie one behind the other (`q_start`); sequence b holds
kv_len[b] keys with the new ones, at page_table[b][p / page] slot p % page.
With `own` false every pass is plain torch in 32 bits (angles in 64, since a far
position times a frequency loses its fraction in 32).
"""
import math
import random

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
BASE = 500000.0


def listed():
    return [
        # the queries of one new token: 8 KiB, bound by latency
        dict(name="rotary_step", kind="rotary", B=1, S=1, H=32, D=128, rot=128, first=2040, heads_first=False,
             interleaved=False, inverse=False),
        # a turn of odd length whose heads rotate 32 of 80 dims in neighbouring
        # pairs, positions past 10^5
        dict(name="rotary_turn", kind="rotary", B=1, S=1021, H=16, D=80, rot=32, first=131000, heads_first=False,
             interleaved=True, inverse=False),
        # the gradient of a whole batch's rotation, heads before positions
        dict(name="rotary_gradient", kind="rotary", B=2, S=4096, H=32, D=128, rot=128, first=0, heads_first=True,
             interleaved=False, inverse=True),
        # one decode step of 16 sequences
        dict(name="append_step", kind="append", B=16, q=1, kv=2000, Hq=32, Hkv=8, D=128, rot=128, page=16,
             interleaved=False, rows_first=False, singles=0),
        # prompts of odd lengths into pages that keep all heads of a row together
        dict(name="append_prompts", kind="append", B=7, q=801, kv=801, Hq=16, Hkv=4, D=64, rot=64, page=32,
             interleaved=True, rows_first=True, singles=0),
        # the largest prefill of a batch
        dict(name="append_batch", kind="append", B=8, q=4096, kv=4096, Hq=32, Hkv=8, D=128, rot=128, page=64,
             interleaved=False, rows_first=False, singles=0),
        # one sequence's step on a short context, bound by latency
        dict(name="attend_step", kind="attend", B=1, q=1, kv=200, Hq=32, Hkv=8, D=128, page=16, window=0,
             rows_first=False, singles=0),
        # one step of 64 sequences of very different lengths
        dict(name="attend_batch", kind="attend", B=64, q=1, kv=8000, Hq=32, Hkv=8, D=128, page=16, window=0,
             rows_first=False, singles=0),
        # one step of two sequences of over 10^5 tokens
        dict(name="attend_long", kind="attend", B=2, q=1, kv=131071, Hq=16, Hkv=2, D=128, page=256, window=0,
             rows_first=True, singles=0),
        # five proposed tokens of each of 24 sequences checked at once
        dict(name="attend_verify", kind="attend", B=24, q=5, kv=3001, Hq=32, Hkv=8, D=128, page=32, window=0,
             rows_first=False, singles=0),
        # a chunk of 2048 tokens behind 6144 cached ones
        dict(name="attend_chunk", kind="attend", B=1, q=2048, kv=8192, Hq=32, Hkv=8, D=128, page=64, window=0,
             rows_first=False, singles=0),
        # prompts of odd lengths and 20 single steps in one batch, head dim 64,
        # each token seeing the last 1024
        dict(name="attend_mixed", kind="attend", B=24, q=1531, kv=2500, Hq=24, Hkv=4, D=64, page=16, window=1024,
             rows_first=False, singles=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8])
    return hkv * rng.choice([1, 3, 4, 7, 8, 16 if hkv <= 2 else 8]), hkv


def draw(rng):
    kind = rng.choice(["rotary", "append", "append", "attend", "attend", "attend", "attend"])
    if kind == "rotary":
        D = rng.choice([64, 80, 96, 128, 256])
        rot = D if rng.random() < 0.6 else rng.choice([D // 2, D // 4, 24])
        while True:
            B, S, H = _log(rng, 1, 8), _log(rng, 1, 8192), rng.choice([1, 8, 12, 16, 32, 40])
            if B * S * H * D <= 2 * 4096 * 32 * 128:
                break
        return dict(kind=kind, B=B, S=S, H=H, D=D, rot=rot, first=rng.choice([0, 5, 4000, 1000000]),
                    heads_first=rng.random() < 0.5, interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3)
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128, 256, 8, 48])
    rows_first = rng.random() < 0.4
    if kind == "append":
        step = rng.random() < 0.5
        while True:
            B, q = (_log(rng, 1, 256), 1) if step else (_log(rng, 1, 16), _log(rng, 2, 8192))
            if B * q * (2 * Hq + 4 * Hkv) * D <= 32768 * 96 * 128:
                break
        return dict(kind=kind, B=B, q=q, kv=q + _log(rng, 1, 4096), Hq=Hq, Hkv=Hkv, D=D,
                    rot=D if rng.random() < 0.7 else D // 2, page=page, interleaved=rng.random() < 0.4,
                    rows_first=rows_first, singles=0 if B == 1 or rng.random() < 0.7 else B // 2)
    form = rng.choice(["step", "step", "few", "chunk"])
    while True:
        if form == "step":
            B, q, kv = _log(rng, 1, 256), 1, _log(rng, 16, 65536)
        elif form == "few":
            B, q, kv = _log(rng, 1, 64), rng.randint(2, 8), _log(rng, 32, 16384)
        else:
            B, q, kv = _log(rng, 1, 16), _log(rng, 9, 2048), _log(rng, 16, 8192)
        c = dict(kind=kind, B=B, q=q, kv=q + kv, Hq=Hq, Hkv=Hkv, D=D, page=page,
                 window=0 if rng.random() < 0.75 else _log(rng, 64, 2048), rows_first=rows_first,
                 singles=0 if form != "chunk" or B == 1 or rng.random() < 0.6 else B // 2)
        # the plain form pads every sequence to the longest: what it needs stays below 6 GB of scores
        if (work(c)["flops"] <= 2.4e11 and work(c)["bytes"] <= 1.0e9 and B * Hq * q * (q + kv) <= 1.5e9
                and B * Hkv * (q + kv) * D <= 2.0e9):
            return c


def _lengths(case):
    """New tokens and keys of each sequence: of the case alone, so that every seed has the same sizes."""
    r = random.Random(case["B"] * 7919 + case["q"] * 131 + case["kv"])
    qs, kvs = [], []
    for b in range(case["B"]):
        whole = b == 0  # one sequence has the full lengths, the others less
        q = 1 if b >= case["B"] - case["singles"] else case["q"] if whole or case["q"] <= 8 else max(1, int(case["q"] * r.uniform(0.2, 1.0)))
        past = case["kv"] - case["q"]
        qs.append(q)
        kvs.append(q + (past if whole else int(past * r.uniform(0.05, 1.0))))
    return qs, kvs


def _visible(q, kv, window):
    """(keys that some new token sees, pairs of a token and a key that it sees)."""
    first, pairs = kv, 0
    for i in range(q):
        limit = kv - q + i
        low = max(0, limit - window + 1) if window else 0
        first = min(first, low)
        pairs += limit + 1 - low
    return kv - first, pairs


def work(case):
    if case["kind"] == "rotary":
        n = case["B"] * case["S"] * case["H"] * case["D"]
        return dict(bytes=4.0 * n, flops=3.0 * case["B"] * case["S"] * case["H"] * case["rot"])
    qs, kvs = _lengths(case)
    T, Hq, Hkv, D = sum(qs), case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        return dict(bytes=T * (4.0 * Hq + 8.0 * Hkv) * D, flops=3.0 * T * (Hq + Hkv) * case["rot"])
    seen = [_visible(q, kv, case["window"]) for q, kv in zip(qs, kvs)]
    return dict(bytes=4.0 * T * Hq * D + 4.0 * Hkv * D * sum(s[0] for s in seen),
                flops=4.0 * Hq * D * sum(s[1] for s in seen))


def _turns(rot):
    """Revolutions per position of each pair: base^(-2 i / rot) / (2 pi)."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    return torch.pow(torch.tensor(BASE, dtype=torch.float64, device=DEV), -2.0 * i / rot) / (2.0 * math.pi)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(BF16)

    s = dict(case=dict(case))
    if case["kind"] == "rotary":
        B, S, H, D = (case[k] for k in ("B", "S", "H", "D"))
        if case["heads_first"]:
            s["x"] = normal(B, H, S, D)
            # each sequence of the batch starts somewhere else
            start = torch.randint(0, 64, (B, 1), generator=g, device=DEV, dtype=torch.int32)
            s["positions"] = start + case["first"] + torch.arange(S, device=DEV, dtype=torch.int32)
        else:
            s["x"] = normal(B * S, H, D)
            start = torch.randint(0, 64, (1,), generator=g, device=DEV, dtype=torch.int32)
            s["positions"] = (start + case["first"] + torch.arange(S, device=DEV, dtype=torch.int32)).repeat(B)
        s["turns"] = _turns(case["rot"])
        return s

    B, Hq, Hkv, D, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    qs, kvs = _lengths(case)
    T, longest = sum(qs), max(kvs)
    width = -(-longest // page)
    used = [-(-kv // page) for kv in kvs]
    pages = sum(used) + 3
    # the pool's pages in the order in which sequences came and went
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32)
    at, host = 0, order.cpu()
    for b, n in enumerate(used):
        table[b, :n] = host[at:at + n]
        at += n
    s["page_table"] = table.to(DEV)
    starts = [0]
    for q in qs:
        starts.append(starts[-1] + q)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["kv_len"] = torch.tensor(kvs, dtype=torch.int32, device=DEV)
    for name in ("k_cache", "v_cache"):  # [pages, heads, rows of the page, D]
        s[name] = normal(pages, page, Hkv, D).transpose(1, 2) if case["rows_first"] else normal(pages, Hkv, page, D)
    s["max_q"], s["max_kv"] = max(qs), longest
    if case["kind"] == "append":
        # the three parts of one projection's output
        qkv = normal(T, Hq + 2 * Hkv, D)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        s["turns"] = _turns(case["rot"])
    else:
        s["q"] = normal(T, Hq, D)
    return s


# ---- the plain forms ---------------------------------------------------------
def _rotate(x, positions, turns, interleaved, inverse):
    """x [tokens, heads, D] in 32 bits, positions [tokens]."""
    rev = positions.double()[:, None] * turns
    angle = (rev - torch.floor(rev)) * (2.0 * math.pi)
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if inverse:
        s = -s
    rot = 2 * turns.numel()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y, z = a * c - b * s, b * c + a * s
    head = torch.stack((y, z), dim=-1).flatten(-2) if interleaved else torch.cat((y, z), dim=-1)
    return torch.cat((head, x[..., rot:]), dim=-1)


def _token_places(s):
    """Sequence and position of each new token."""
    T = s["q"].shape[0]
    t = torch.arange(T, device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["q_start"][1:].contiguous(), t, right=True)
    n = s["q_start"][1:] - s["q_start"][:-1]
    return b, (s["kv_len"] - n)[b] + t - s["q_start"][:-1][b]


def _plain_append(s):
    case = s["case"]
    b, p = _token_places(s)
    q = _rotate(s["q"].float(), p, s["turns"], case["interleaved"], False).to(BF16)
    k = _rotate(s["k"].float(), p, s["turns"], case["interleaved"], False).to(BF16)
    page, slot = s["page_table"][b, p // case["page"]].long(), (p % case["page"]).long()
    s["k_cache"][page, :, slot] = k
    s["v_cache"][page, :, slot] = s["v"]
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attend(s):
    case = s["case"]
    B, Hq, Hkv, D, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    G, mq, mk = Hq // Hkv, s["max_q"], s["max_kv"]
    n = s["q_start"][1:] - s["q_start"][:-1]
    # queries [B, heads of keys, group x tokens, D], every sequence as long as the longest
    t = (s["q_start"][:-1, None] + torch.arange(mq, device=DEV)).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"].float()[t].view(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * mq, D)
    key = torch.arange(mk, device=DEV)
    pages, slots = s["page_table"][:, key // page].long(), (key % page).expand(B, mk)
    k = s["k_cache"][pages, :, slots].float().permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).view(B, Hkv, G, mq, mk)
    del k
    limit = (s["kv_len"] - n)[:, None] + torch.arange(mq, device=DEV)
    seen = key <= limit[..., None]
    if case["window"]:
        seen &= key > limit[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(top).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    v = s["v_cache"][pages, :, slots].float().permute(0, 2, 1, 3)
    v = torch.where((key < s["kv_len"][:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(scores.view(B, Hkv, G * mq, mk), v).view(B, Hkv, G, mq, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, mq, Hq, D)
    b, p = _token_places(s)
    return o[b, p - (s["kv_len"] - n)[b]].to(BF16)


def run(s):
    case = s["case"]
    if own:
        from polykernel_amd import kernels

        if case["kind"] == "rotary":
            return kernels.rotary(s["x"], s["positions"], s["turns"], interleaved=case["interleaved"],
                                  inverse=case["inverse"])
        where = (s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_len"])
        if case["kind"] == "append":
            q = kernels.paged_kv_append(s["k"], s["v"], *where, q=s["q"], turns=s["turns"],
                                        interleaved=case["interleaved"])
            return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
        return kernels.paged_attention(s["q"], *where, max_q=s["max_q"], window=case["window"])
    if case["kind"] == "rotary":
        x = s["x"].float()
        if case["heads_first"]:
            B, H, S, D = x.shape
            flat = x.permute(0, 2, 1, 3).reshape(B * S, H, D)
            y = _rotate(flat, s["positions"].reshape(-1), s["turns"], case["interleaved"], case["inverse"])
            return y.view(B, S, H, D).permute(0, 2, 1, 3).contiguous().to(BF16)
        return _rotate(x, s["positions"], s["turns"], case["interleaved"], case["inverse"]).to(BF16)
    return _plain_append(s) if case["kind"] == "append" else _plain_attend(s)


# ---- the definitions in 64 bits ------------------------------------------------
def _spin(x, positions, turns, interleaved, sign):
    """Each pair as a complex number times e^(i sign angle); x [..., tokens, D] in 64 bits, positions of its tokens."""
    rot = 2 * turns.numel()
    head = x[..., :rot]
    z = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) if interleaved else \
        torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
    angle = torch.remainder(positions.double().unsqueeze(-1) * turns, 1.0) * (sign * 2.0 * math.pi)
    z = z * torch.polar(torch.ones_like(angle), angle)
    out = x.clone()
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        x, sign = s["x"].double(), -1.0 if case["inverse"] else 1.0
        if case["heads_first"]:
            return torch.stack([_spin(x[b], s["positions"][b], s["turns"], case["interleaved"], sign)
                                for b in range(case["B"])])
        return _spin(x.transpose(0, 1).contiguous(), s["positions"], s["turns"], case["interleaved"],
                     sign).transpose(0, 1).contiguous()
    qs, kvs = _lengths(case)
    page, Hkv = case["page"], case["Hkv"]
    outs = [s["q"].double().clone()]
    if case["kind"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
    at = 0
    for b, (n, kv) in enumerate(zip(qs, kvs)):
        places = torch.arange(kv - n, kv, device=DEV)
        if case["kind"] == "append":
            rows = slice(at, at + n)
            spin = lambda x: _spin(x[rows].double().transpose(0, 1).contiguous(), places, s["turns"],  # noqa: E731
                                   case["interleaved"], 1.0).transpose(0, 1)
            outs[0][rows] = spin(s["q"])
            k, v = spin(s["k"]), s["v"][rows].double()
            for first in range((kv - n) // page, (kv - 1) // page + 1):  # page by page
                lo, hi = max(first * page, kv - n), min((first + 1) * page, kv)
                to = int(s["page_table"][b, first])
                kc[to, :, lo - first * page:hi - first * page] = k[lo - kv + n:hi - kv + n].transpose(0, 1)
                vc[to, :, lo - first * page:hi - first * page] = v[lo - kv + n:hi - kv + n].transpose(0, 1)
        else:
            own_pages = s["page_table"][b, :-(-kv // page)].long()
            keys = s["k_cache"][own_pages].double().transpose(0, 1).flatten(1, 2)[:, :kv]
            values = s["v_cache"][own_pages].double().transpose(0, 1).flatten(1, 2)[:, :kv].contiguous()
            keys_t = keys.transpose(1, 2).contiguous()
            G = case["Hq"] // Hkv
            key = torch.arange(kv, device=DEV)
            hidden = key > places[:, None]
            if case["window"]:
                hidden = hidden | (key <= places[:, None] - case["window"])
            for h in range(case["Hq"]):
                sc = (s["q"][at:at + n, h].double() @ keys_t[h // G]) / math.sqrt(case["D"])
                p = torch.softmax(sc.masked_fill(hidden, float("-inf")), dim=-1)
                outs[0][at:at + n, h] = p @ values[h // G]
        at += n
    return dict(q=outs[0], k_cache=kc, v_cache=vc) if case["kind"] == "append" else outs[0]
