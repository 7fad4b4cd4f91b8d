"""The attention operators' definitions in 64 bits (torch, CPU), a token and head at a time, and seeded inputs for their tests.

Bars.  An output of rope_norm is rounded once, 2^-8 of it at most; before that the hardware's sine and cosine are off by less than
2^-19 (test_sine_and_cosine), of the pair's magnitude, and fp32 products by a few 2^-24.

An output of attend is sum_j w_j v_j / sum_j w_j.  Each weight is rounded to bf16, w_j (1 + d_j) with |d_j| <= 2^-8, above and below
alike, so that with sum_j w_j = 1 the quotient is off by sum_j w_j d_j (v_j - out), to first order: by 2^-8 (A + |out|) at most with
A = sum_j w_j |v_j|.  The rounding of the output adds 2^-8 |out|; scores in fp32 are off by D 2^-24 of |q| |k| scale at most (5e-5 at
|q| |k| scale of 3 and D = 256, where the bars are used), which moves the weights by as much: 2^-12 A is above both that and the second
order.  Roundings of weights have random signs and an rms of 2^-8 / 3^1/2 at most, so that the error's norm is in the mean at most
that of 2^-8 / 3^1/2 sqrt(sum_j w_j^2 (v_j - out)^2 + out^2), S^2 = sum_j w_j^2 v_j^2: below 2^-8 / 3^1/2 sqrt(2 S^2 + 3 out^2), as (a - b)^2 <=
2 a^2 + 2 b^2 and sum_j w_j^2 <= 1, and so below 2^-8 sqrt(S^2 + out^2)."""
import torch

BF16, F64 = torch.bfloat16, torch.float64


def page_rows(d, n, lo, hi):
    """(page, place) of the tokens lo .. hi - 1 of sequence n; entries outside the cache as they are."""
    t = torch.arange(lo, hi)
    page = d["kp"].shape[1]
    return d["table"][n].long()[t // page], t % page


def batch(d):
    """(first packed token, new tokens, cached tokens) of each sequence, held to what there is."""
    T, page = d["q"].shape[0], d["kp"].shape[1]
    loc = [min(max(x, 0), T) for x in d["loc"].tolist()]
    return [(lo, max(hi - lo, 0), min(max(m, 0), d["table"].shape[1] * page)) for lo, hi, m in zip(loc, loc[1:], d["lens"].tolist())]


def rope_head(x, w, inv_freq, pos, eps, offset, interleaved):
    """x [.., D] at positions pos [..]."""
    x = x.to(F64)
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (offset + w.to(F64))
    half = inv_freq.numel()
    a = torch.arange(half) * (2 if interleaved else 1)
    b = a + (1 if interleaved else half)
    phi = pos.to(F64)[..., None] * inv_freq.to(F64)
    y = x.clone()
    y[..., a] = x[..., a] * phi.cos() - x[..., b] * phi.sin()
    y[..., b] = x[..., a] * phi.sin() + x[..., b] * phi.cos()
    return y


def rope(d, eps=1e-6, offset=0.0, interleaved=False):
    """out [T, HQ, D]; the new tokens' keys and values [T, HK, D], and where they go: (packed token, page, place) lists."""
    out = torch.full(d["q"].shape, float("nan"), dtype=F64)
    k = torch.zeros(d["k"].shape, dtype=F64)
    where = []
    NP = d["kp"].shape[0]
    for n, (lo, m, all_) in enumerate(batch(d)):
        for j in range(m):
            pos = all_ - m + j
            if pos < 0:
                out[lo + j] = 0
                continue
            args = (d["inv_freq"], torch.tensor(pos).expand(1), eps, offset, interleaved)
            out[lo + j] = rope_head(d["q"][lo + j], d["qw"], *args)
            k[lo + j] = rope_head(d["k"][lo + j], d["kw"], *args)
            (page,), (place,) = page_rows(d, n, pos, pos + 1)
            if 0 <= int(page) < NP:
                where.append((lo + j, int(page), int(place)))
    return out, k, where


def values(d, which):
    """The cache's keys or values as numbers, 64 bits."""
    p = d[which + "p"].to(F64)
    return p if d.get(which + "s") is None else p * d[which + "s"].to(F64)[..., None]


def attend(d, scale=None, window=0):
    """out, A = sum w |v| and sqrt(sum w^2 v^2) [T, HQ, D]; NaN where no sequence holds a row."""
    T, HQ, D = d["q"].shape
    HK, NP = d["kp"].shape[2], d["kp"].shape[0]
    res = [torch.full((T, HQ, D), float("nan"), dtype=F64) for _ in range(3)]
    scale = D ** -0.5 if scale is None else scale
    kall, vall = values(d, "k"), values(d, "v")
    for n, (lo, m, all_) in enumerate(batch(d)):
        page, place = page_rows(d, n, 0, all_)
        page = torch.where((page >= 0) & (page < NP), page, torch.zeros_like(page))
        K, V = kall[page, place], vall[page, place]
        for j in range(m):
            pos = all_ - m + j
            first = max(0, pos - window + 1) if window else 0
            if pos < 0:
                for r in res:
                    r[lo + j] = 0
                continue
            k, v = (x[first:pos + 1].repeat_interleave(HQ // HK, 1).transpose(0, 1) for x in (K, V))       # [HQ, keys, D]
            s = (k @ d["q"][lo + j].to(F64)[..., None])[..., 0] * scale
            w = torch.softmax(s, -1)[:, None]
            for r, x in zip(res, (w @ v, w @ v.abs(), ((w * w) @ (v * v)).sqrt())):
                r[lo + j] = x[:, 0]
    if d.get("gate") is not None:
        for r in res:
            r *= torch.sigmoid(d["gate"].to(F64))
    return res


def near(got, want, A, S):
    got = got.detach().cpu().to(F64)
    held = ~torch.isnan(want)
    assert torch.isfinite(got[held]).all(), "not finite"
    err = (got - want)[held].abs()
    bar = 2.0 ** -8 * (2 * want.abs() + A) + 2.0 ** -12 * A + 1e-30
    off = err > bar[held]
    assert not off.any(), (int(off.sum()), float((err / bar[held]).max()))
    norm, most = float(err.norm()), float((want * want + S * S)[held].sum().sqrt())
    assert norm <= 2.0 ** -8 * most + 1e-30, (norm, most)


# ---- inputs (CPU) --------------------------------------------------------------------------------------------------------
def inputs(seed, new, ctx, HQ, HK, D, page=16, int8=False, gate=False, rot=None, freq=torch.float32, theta=1e4, wtype=BF16, extra=0,
           qscale=1.0):
    """Sequences of `new` tokens, the last of `ctx` cached ones each; `extra` packed tokens that no sequence holds."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)                    # noqa: E731
    N, T = len(new), sum(new) + extra
    need = [-(-max(m, 1) // page) for m in ctx]
    NP = sum(need) + 2
    order = (torch.randperm(NP - 1, generator=g) + 1).tolist()
    table = torch.zeros(N, max(need), dtype=torch.int32)
    for n, m in enumerate(need):
        table[n, :m] = torch.tensor([order.pop() for _ in range(m)])
    d = dict(q=(qscale * rn(T, HQ, D)).to(BF16), k=rn(T, HK, D).to(BF16), v=rn(T, HK, D).to(BF16), table=table,
             loc=torch.tensor([sum(new[:n]) for n in range(N + 1)], dtype=torch.int32), lens=torch.tensor(ctx, dtype=torch.int32),
             qw=(1 + 0.2 * rn(D)).to(wtype), kw=(1 + 0.2 * rn(D)).to(wtype), gate=rn(T, HQ, D).to(BF16) if gate else None)
    rot = D if rot is None else rot
    d["inv_freq"] = (theta ** (-2 * torch.arange(rot // 2, dtype=F64) / max(rot, 1))).to(freq)
    for x in ("k", "v"):
        p = rn(NP, page, HK, D)
        d[x + "s"] = None
        if int8:
            d[x + "s"] = p.abs().amax(-1) / 127
            p = torch.round(p / d[x + "s"][..., None]).to(torch.int8)
        d[x + "p"] = p if int8 else p.to(BF16)
    d["out"] = torch.full((T, HQ, D), 7.0, dtype=BF16)
    return d


def cuda(d):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
