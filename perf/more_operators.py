"""Measured cases of the operators that take sequences through a softmax-attention layer with a paged cache
(`leapquant_amd.attn`).

* "rope": the norms of each head's queries and keys with the rotation by the token's position, keys and values into their
  pages (`rope_norm`);
* "attend": the attention of a ragged batch's new tokens over the pages, from one token a sequence to whole prompts
  (`attend`); pages in bf16, or in 8 bits with a scale a token and head.

Sequence n has `ctx` cached tokens in all, the last `new` of them the call's own.  The plain forms compute in fp32 with
elementary torch operations, angles in fp64, and round once; `exact` goes by the definition in fp64, a sequence and head at a
time.
"""
import math
import random

import torch

own = False
DEV = "cuda"
F64 = torch.float64
EPS = 1e-6


def _case(name, op, **kw):
    c = dict(name=name, op=op, N=1, new=1, short=1, ctx=1, HQ=32, HK=8, D=128, page=16)
    if op == "rope":
        c.update(rot=128, pairs="halves", theta=1e6, offset=0.0)
    else:
        c.update(int8=False, window=0, gate=False)
    c.update(kw)
    return c


def listed():
    """A batch's longest sequence has `new` new tokens, the others `short` at most; `ctx` is the longest context."""
    return [
        # one token of one sequence, heads of 256 of which 64 turn: latency
        _case("rope_one", "rope", ctx=8192, HQ=16, HK=2, D=256, rot=64, theta=1e7, offset=1.0),
        # a decode batch at contexts up to 8192
        _case("rope_decode_64", "rope", N=64, ctx=8192),
        # a few short prompts, heads of 64, pairs of neighbours
        _case("rope_short_64", "rope", N=5, new=300, short=300, ctx=777, HQ=16, HK=16, D=64, rot=64, pairs="neighbours", theta=1e4),
        # a full token budget of ragged prompts, some going on from a cache, far positions
        _case("rope_prefill_32k", "rope", N=13, new=5001, short=5001, ctx=65536, HQ=16, HK=2, D=256, rot=64, theta=1e7, offset=1.0, page=64),
        # one token of one sequence over 8192: latency
        _case("attend_one", "attend", ctx=8192, HQ=16, HK=2, D=256, gate=True),
        # a decode batch of 64 with contexts up to 8192
        _case("attend_decode_64", "attend", N=64, ctx=8192),
        # the same from pages in 8 bits
        _case("attend_decode_64_int8", "attend", N=64, ctx=8192, int8=True),
        # drafted tokens of a decode batch, checked in one call, large pages
        _case("attend_drafts_32", "attend", N=32, new=8, short=8, ctx=4099, HQ=16, HK=2, D=256, page=528),
        # a prompt's piece beside decode tokens
        _case("attend_mixed_16", "attend", N=16, new=449, short=1, ctx=4096),
        # short prompts under a sliding window, heads of 64, no sharing of key heads
        _case("attend_window_64", "attend", N=5, new=777, short=777, ctx=1500, HQ=16, HK=16, D=64, window=128, page=32),
        # one long prompt from nothing
        _case("attend_prompt_8k", "attend", new=8192, ctx=8192),
        # a prompt's piece of 2048 tokens over a long cache, with the layer's output gate: the largest case
        _case("attend_chunk_32k", "attend", new=2048, ctx=32768, HQ=16, HK=2, D=256, gate=True, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = ((16, 2), (32, 8), (16, 16), (24, 4), (8, 8), (20, 4), (16, 1), (6, 2), (32, 4), (40, 8))


def draw(rng):
    """One more case of the same ranges: 1 to 64 sequences, 1 to 8192 new tokens and contexts of 1 to 32768 over their
    logarithms, other head layouts and page sizes, within the cost of the largest listed case."""
    op = rng.choice(("rope", "attend", "attend", "attend"))
    while True:
        c = _case("", op)
        del c["name"]
        c["HQ"], c["HK"] = rng.choice(HEADS)
        c["D"] = rng.choice((64, 128, 128, 256))
        c["page"] = rng.choice((16, 16, 32, 64, 128, 528, 784))
        c["N"] = _log(rng, 1, 64)
        kind = rng.choice(("decode", "drafts", "prompts", "mixed"))
        c["new"] = 1 if kind == "decode" else _log(rng, 2, 24) if kind == "drafts" else _log(rng, 16, 8192)
        c["short"] = rng.choice((1, 2)) if kind == "mixed" else c["new"]
        c["ctx"] = c["new"] + rng.choice((0, 1, 1, 1)) * _log(rng, 1, 32768)
        if op == "rope":
            c["rot"] = rng.choice((c["D"], c["D"], c["D"] // 2, c["D"] // 4))
            c["pairs"], c["theta"] = rng.choice(("halves", "halves", "neighbours")), rng.choice((1e4, 1e6, 1e7))
            c["offset"] = rng.choice((0.0, 1.0))
            if c["N"] * c["new"] * (c["HQ"] + 2 * c["HK"]) * c["D"] <= 1 << 27 and c["N"] * c["ctx"] * c["HK"] * c["D"] <= 1 << 30:
                return c
        else:
            c["int8"], c["gate"] = rng.random() < 0.3, rng.random() < 0.3
            c["window"] = rng.choice((0, 0, 0, _log(rng, 1, 4096)))
            if c["N"] * c["new"] * c["HQ"] * c["ctx"] * c["D"] <= 1 << 37 and c["N"] * c["ctx"] * c["HK"] * c["D"] <= 1 << 29:
                return c


def _batch(c):
    """(new tokens, cached tokens) of each sequence: odd, and the same for every seed."""
    r = random.Random(c["N"] * 65537 + c["new"] * 31 + c["ctx"])
    new = [c["new"]] + [r.randint(1, c["short"]) for _ in range(c["N"] - 1)]
    before = c["ctx"] - c["new"]
    ctx = [c["ctx"]] + [n + (r.randint(before // 2, before) if r.random() < 0.8 else 0) for n in new[1:]]
    return new, ctx


def prepare(case, seed):
    c = dict(case)
    N, HQ, HK, D, page = (c[k] for k in ("N", "HQ", "HK", "D", "page"))
    new, ctx = _batch(c)
    T = sum(new)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g, dtype=torch.float32)     # noqa: E731
    d = {"case": c, "new": new, "ctx": ctx}
    d["loc"] = torch.tensor([sum(new[:i]) for i in range(N + 1)], dtype=torch.int32).to(DEV)
    d["lens"] = torch.tensor(ctx, dtype=torch.int32).to(DEV)
    # every sequence's pages, in no order, page 0 held by nobody
    need = torch.tensor([-(-n // page) for n in ctx])
    width, NP = int(need.max()), int(need.sum()) + 1
    order = (torch.randperm(NP - 1, device=DEV, generator=g) + 1).int()
    at = (torch.cumsum(need, 0) - need)[:, None] + torch.arange(width)
    held = torch.arange(width) < need[:, None]
    d["table"] = torch.where(held.to(DEV), order[torch.where(held, at, torch.zeros_like(at)).to(DEV)], torch.zeros((), device=DEV, dtype=torch.int32))
    if c["op"] == "rope":
        # queries, keys and values as column ranges of the input projection's output
        x = randn(T, (HQ + 2 * HK) * D).bfloat16()
        q, k, v = x.split([HQ * D, HK * D, HK * D], 1)
        d["q"], d["k"], d["v"] = q.view(T, HQ, D), k.view(T, HK, D), v.view(T, HK, D)
        d["qw"], d["kw"] = ((1 - c["offset"] + 0.2 * randn(D)).bfloat16() for _ in range(2))
        i = torch.arange(c["rot"] // 2, device=DEV, dtype=F64)
        d["inv_freq"] = (c["theta"] ** (-2 * i / c["rot"])).float()
        d["kp"], d["vp"] = (torch.zeros(NP, page, HK, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        d["out"] = torch.empty(T, HQ, D, device=DEV, dtype=torch.bfloat16)
        return d
    d["q"] = (1.5 * randn(T, HQ, D)).bfloat16()
    for x in ("k", "v"):
        p = torch.empty(NP, page, HK, D, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
        d[x + "s"] = None
        if c["int8"]:
            s = p.abs().amax(-1).float() / 127
            p = torch.round(p.float() / s[..., None]).to(torch.int8)
            d[x + "s"] = s
        d[x + "p"] = p
    # the output gate: the other half of a projection of twice the width
    d["gate"] = randn(T, HQ, 2 * D).bfloat16()[..., D:] if c["gate"] else None
    d["out"] = torch.empty(T, HQ, D, device=DEV, dtype=torch.bfloat16)
    return d


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


# ---- the framework's operators ---------------------------------------------------------------------------------------
def _own_rope(d):
    from leapquant_amd import attn
    c = d["case"]
    attn.rope_norm(d["q"], d["k"], d["v"], d["qw"], d["kw"], d["inv_freq"], attn.Pages(d["kp"], d["vp"]), d["table"], d["loc"],
                   d["lens"], d["out"], eps=EPS, offset=c["offset"], interleaved=c["pairs"] == "neighbours")
    return d["out"], d["kp"], d["vp"]


def _own_attend(d):
    from leapquant_amd import attn
    attn.attend(d["q"], attn.Pages(d["kp"], d["vp"], d["ks"], d["vs"]), d["table"], d["loc"], d["lens"], d["out"],
                window=d["case"]["window"], gate=d["gate"], longest=d["case"]["new"])
    return d["out"]


_own = {"rope": _own_rope, "attend": _own_attend}


# ---- plain forms: fp32, elementary operations ---------------------------------------------------------------------------
def _positions(d, T):
    """The sequence of each packed token, and its position there."""
    t = torch.arange(T, device=DEV)
    loc = d["loc"].long()
    n = torch.searchsorted(loc[1:].contiguous(), t, right=True)
    return n, d["lens"].long()[n] - loc[n + 1] + t


def _plain_rope(d):
    c = d["case"]
    T, half, page = d["q"].shape[0], c["rot"] // 2, c["page"]
    n, pos = _positions(d, T)
    turn = pos.double()[:, None, None] * d["inv_freq"].double()
    cos, sin = turn.cos().float(), turn.sin().float()

    def head(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (c["offset"] + w.float())
        r, rest = x[..., :2 * half], x[..., 2 * half:]
        if c["pairs"] == "halves":
            a, b = r[..., :half], r[..., half:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([r, rest], -1).bfloat16()
    at = d["table"][n, pos // page].long(), pos % page
    d["kp"][at] = head(d["k"], d["kw"])
    d["vp"][at] = d["v"]
    return head(d["q"], d["qw"]), d["kp"], d["vp"]


def _cached(d, x):
    """The cached keys or values of the batch: [N, HK, longest context, D], fp32."""
    page = d["case"]["page"]
    t = torch.arange(max(d["ctx"]), device=DEV)
    at = d["table"][:, t // page].long(), (t % page).expand(len(d["ctx"]), -1)
    y = d[x + "p"][at].float()
    if d[x + "s"] is not None:
        y = y * d[x + "s"][at][..., None]
    return y.transpose(1, 2).contiguous()


def _plain_attend(d):
    c = d["case"]
    HQ, HK, D = c["HQ"], c["HK"], c["D"]
    N, L, T = c["N"], max(d["new"]), d["q"].shape[0]
    k, v = _cached(d, "k"), _cached(d, "v")
    row = torch.arange(L, device=DEV)
    live = row < torch.tensor(d["new"], device=DEV)[:, None]
    rows = torch.where(live, d["loc"][:-1, None].long() + row, torch.zeros_like(row))
    pos = (d["lens"].long() - torch.diff(d["loc"].long()))[:, None] + row
    q = d["q"][rows].float().view(N, L, HK, HQ // HK, D).permute(0, 2, 3, 1, 4).reshape(N, HK, -1, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(N, HK, HQ // HK, L, -1)
    j = torch.arange(s.shape[-1], device=DEV)
    hidden = j > pos[..., None]
    if c["window"]:
        hidden = hidden | (j <= pos[..., None] - c["window"])
    s.masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s.view(N, HK, -1, s.shape[-1]), v).view(N, HK, HQ // HK, L, D) / s.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(N, L, HQ, D)[live]
    if d["gate"] is not None:
        o = o * torch.sigmoid(d["gate"].float())
    return o.view(T, HQ, D).bfloat16()


_plain = {"rope": _plain_rope, "attend": _plain_attend}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c = case
    HQ, HK, D, w = c["HQ"], c["HK"], c["D"], c.get("window", 0)
    new, ctx = _batch(c)
    T = sum(new)
    if c["op"] == "rope":
        n = T * (HQ + 2 * HK) * D
        return {"bytes": 4.0 * n, "flops": 8.0 * n}
    keys = pairs = 0                                     # that some row of the sequence sees; pairs of a row and such a key
    for n, m in zip(new, ctx):
        first = m - n                                    # the first new token's position
        keys += m - (max(0, first - w + 1) if w else 0)
        pairs += sum(min(w, p + 1) for p in range(first, m)) if w else n * (first + 1 + m) // 2
    row = HK * (2 * D + 8 if c["int8"] else 4 * D)
    return {"bytes": float(keys * row + T * HQ * D * (6 if c["gate"] else 4)), "flops": 4.0 * pairs * HQ * D}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------
def _slots(d, n, lo, hi):
    t = torch.arange(lo, hi, device=DEV)
    page = d["case"]["page"]
    return d["table"][n].long()[torch.div(t, page, rounding_mode="floor")], t % page


def _exact_rope(d):
    c, rot = d["case"], d["case"]["rot"]
    q, kp, vp = d["q"].to(F64), d["kp"].to(F64), d["vp"].to(F64)
    out = torch.empty_like(q)
    neighbours = c["pairs"] == "neighbours"
    a = torch.arange(rot // 2, device=DEV) * (2 if neighbours else 1)
    b = a + (1 if neighbours else rot // 2)
    for n, (m, all_) in enumerate(zip(d["new"], d["ctx"])):
        lo = sum(d["new"][:n])
        ang = torch.arange(all_ - m, all_, device=DEV, dtype=F64)[:, None, None] * d["inv_freq"].to(F64)
        done = []
        for x, w in ((q[lo:lo + m], d["qw"]), (d["k"][lo:lo + m].to(F64), d["kw"])):
            y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (w.to(F64) + c["offset"])
            z = y.clone()
            z[..., a] = y[..., a] * torch.cos(ang) - y[..., b] * torch.sin(ang)
            z[..., b] = y[..., a] * torch.sin(ang) + y[..., b] * torch.cos(ang)
            done.append(z)
        out[lo:lo + m] = done[0]
        at = _slots(d, n, all_ - m, all_)
        kp[at], vp[at] = done[1], d["v"][lo:lo + m].to(F64)
    return out, kp, vp


def _exact_attend(d):
    c = d["case"]
    G, w = c["HQ"] // c["HK"], c["window"]
    out = torch.empty(d["q"].shape, device=DEV, dtype=F64)
    for n, (m, all_) in enumerate(zip(d["new"], d["ctx"])):
        lo, at = sum(d["new"][:n]), _slots(d, n, 0, all_)
        K, V = (d[x + "p"][at].to(F64) * (1 if d[x + "s"] is None else d[x + "s"][at][..., None].to(F64)) for x in ("k", "v"))
        p = torch.arange(all_ - m, all_, device=DEV)[:, None]
        j = torch.arange(all_, device=DEV)
        seen = (j <= p) & (j > p - w) if w else j <= p
        for h in range(c["HQ"]):
            s = torch.matmul(d["q"][lo:lo + m, h].to(F64), K[:, h // G].t().contiguous()) / math.sqrt(c["D"])
            s = torch.where(seen, s, torch.full((), -math.inf, device=DEV, dtype=F64))
            e = torch.exp(s - s.max(-1, keepdim=True)[0])
            out[lo:lo + m, h] = torch.matmul(e, V[:, h // G].contiguous()) / e.sum(-1, keepdim=True)
    if d["gate"] is not None:
        out = out / (1 + torch.exp(-d["gate"].to(F64)))
    return out


def exact(case, seed):
    d = prepare(case, seed)
    return {"rope": _exact_rope, "attend": _exact_attend}[case["op"]](d)
