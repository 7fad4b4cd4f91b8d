"""Measured cases of the operators that take whole sequences through a linear-attention layer (`leapquant_amd.seq`).

* "prefill": the gated delta rule over a ragged batch of prompts (`delta_prefill`), fp32 states in cache slots;
* "steps": the same recurrence token by token for a few tokens a sequence (`delta_steps`), GDN and KDA;
* "conv": the depthwise causal conv over a ragged batch with its taps in cache slots (`conv_prefill`);
* "gated": the norm after the block times its gate (`gated_norm`);
* "add": the residual add and the norm before the next block (`add_norm`).

A sequence starts from slot `src` (0: from nothing) and leaves its state in slot `idx`, another one here, so that a pass
can be repeated on the same inputs.  The plain forms compute in fp32 with elementary torch operations and round once;
`exact` walks the definition token by token in fp64.
"""
import math
import random

import torch

own = False
DEV = "cuda"
F64 = torch.float64
EPS = 1e-6


def _case(name, op, **kw):
    c = dict(name=name, op=op)
    if op in ("prefill", "steps"):
        c.update(K=128, V=128, HV=32, H=16, N=1, carry=0.0)
        c.update(dict(T=1) if op == "prefill" else dict(most=1, kda=False, glb=0.0))
    elif op == "conv":
        c.update(T=1, N=1, C=8192, carry=0.5, bias=False)
    elif op == "gated":
        c.update(rows=1, HV=32, D=128, act="silu")
    else:
        c.update(rows=1, D=2048, scale=1.0)
    c.update(kw)
    return c


def listed():
    return [
        # one long prompt at the benchmark's layer shape (32 value heads, 16 key heads, 128 x 128): latency along the sequence
        _case("prefill_one_8k", "prefill", T=8192),
        # a full token budget of ragged prompts, half of them going on from a state (chunked prefill): the largest case
        _case("prefill_batch_32k", "prefill", N=13, T=32768, carry=0.5),
        # a few short prompts, heads of 64, four value heads a key head
        _case("prefill_short_64", "prefill", N=5, T=777, K=64, V=64, HV=16, H=4, carry=0.5),
        # one token of one sequence: latency
        _case("steps_one", "steps", carry=1.0),
        # drafted tokens of a decode batch, checked in one call
        _case("steps_drafts_64", "steps", N=64, most=8, carry=1.0),
        # the same for Kimi Delta Attention with the bounded gate
        _case("steps_kda_32", "steps", N=32, most=4, HV=32, H=32, kda=True, glb=-5.0, carry=1.0),
        # the conv of a few short prompts
        _case("conv_short", "conv", T=333, N=3),
        # the conv of a full token budget
        _case("conv_32k", "conv", T=32768, N=13),
        # the gated norm of a decode batch
        _case("gated_decode", "gated", rows=64),
        # the gated norm of a full token budget
        _case("gated_prefill", "gated", rows=32768),
        # the residual add and norm of a decode batch (hidden size 2048)
        _case("add_decode", "add", rows=64),
        # the same of a long prompt, with a residual scale
        _case("add_prefill", "add", rows=16385, scale=0.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the same ranges: 1 to 32768 tokens and 1 to 64 sequences over their logarithms, the head
    layouts, gates and hidden sizes of the framework's shapes in other combinations, odd sizes among them."""
    op = rng.choice(("prefill", "prefill", "prefill", "steps", "steps", "conv", "gated", "add"))
    c = _case("", op)
    del c["name"]
    if op in ("prefill", "steps"):
        c["K"], c["V"] = rng.choice(((128, 128), (128, 128), (128, 128), (64, 128), (64, 64)))
        c["H"] = rng.choice((2, 4, 8, 16))
        c["HV"] = c["H"] * rng.choice((1, 2, 2, 4))
        c["carry"] = rng.choice((0.0, 0.5, 1.0))
    if op == "prefill":
        c["T"] = _log(rng, 16, 32768)
        while c["T"] * c["HV"] > 32768 * 32:
            c["T"] //= 2
        c["N"] = min(c["T"], _log(rng, 1, 64))
    elif op == "steps":
        c["N"], c["most"] = _log(rng, 1, 64), _log(rng, 1, 24)
        if rng.random() < 0.4:
            c["K"] = c["V"] = 128
            c["H"] = rng.choice((8, 16, 24, 32))
            c["HV"] = c["H"]
            c["kda"], c["glb"] = True, rng.choice((0.0, -5.0))
    elif op == "conv":
        c["T"] = _log(rng, 16, 32768)
        c["N"] = min(c["T"], _log(rng, 1, 64))
        c["C"] = 128 * rng.randint(3, 64)
        c["carry"], c["bias"] = rng.choice((0.0, 0.5, 1.0)), rng.random() < 0.3
    elif op == "gated":
        c["rows"], c["HV"], c["D"] = _log(rng, 1, 32768), rng.choice((4, 8, 15, 16, 32)), rng.choice((64, 128, 128))
        c["act"] = rng.choice(("silu", "sigmoid"))
    else:
        c["rows"], c["D"] = _log(rng, 1, 16385), rng.choice((1000, 1024, 2048, 2048, 2049, 4096))
        c["scale"] = rng.choice((1.0, 0.5, 0.22))
    return c


def _lens(c):
    """Lengths of the case's sequences: odd, and the same for every seed."""
    r = random.Random(c["N"] * 65537 + c.get("T", c.get("most", 0)))
    if c["op"] == "steps":
        return [c["most"]] + [r.randint(1, c["most"]) for _ in range(c["N"] - 1)]
    cuts = sorted(r.sample(range(1, c["T"]), c["N"] - 1)) if c["N"] > 1 else []
    return [hi - lo for lo, hi in zip([0] + cuts, cuts + [c["T"]])]


def prepare(case, seed):
    c, op = dict(case), case["op"]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)     # noqa: E731
    rand = lambda *s: torch.rand(*s, device=DEV, generator=g)       # noqa: E731
    d = {"case": c}
    if op == "gated":
        rows, HV, D = c["rows"], c["HV"], c["D"]
        d["x"], d["w"] = (0.3 * randn(rows, HV, D)).bfloat16(), (1 + 0.2 * randn(D)).bfloat16()
        # the gate is a column range of the input projection's output, as a layer has it
        d["z"] = randn(rows, 2 * HV * D).bfloat16()[:, HV * D:].view(rows, HV, D)
        d["out"] = torch.empty(rows, HV, D, device=DEV, dtype=torch.bfloat16)
        return d
    if op == "add":
        rows, D = c["rows"], c["D"]
        d["x"], d["y"] = (3 * randn(rows, D)).bfloat16(), randn(rows, D).bfloat16()
        d["w"] = (1 + 0.2 * randn(D)).bfloat16()
        d["res"], d["out"] = (torch.empty(rows, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        return d
    N, lens = c["N"], _lens(c)
    T = sum(lens)
    d["lens"] = lens
    d["loc"] = torch.tensor([sum(lens[:i]) for i in range(N + 1)], dtype=torch.int32).to(DEV)
    have = (torch.arange(N, device=DEV) + 1) * c["carry"] % 1.0 < c["carry"]       # which sequences go on from a state
    if c["carry"] in (0.0, 1.0):
        have = torch.full((N,), bool(c["carry"]), device=DEV)
    d["src"] = ((torch.randperm(N, device=DEV, generator=g) + 1) * have).int()
    d["idx"] = (torch.randperm(N, device=DEV, generator=g) + N + 1).int()
    if op == "conv":
        C = c["C"]
        d["x"] = randn(T, C).bfloat16()
        d["w"] = (0.5 * randn(C, 4)).bfloat16()
        d["bias"] = (0.1 * randn(C)).bfloat16() if c["bias"] else None
        d["taps"] = torch.zeros(2 * N + 1, C, 3, device=DEV, dtype=torch.bfloat16)
        d["taps"][1:N + 1] = randn(N, C, 3).bfloat16()
        d["out"] = torch.empty(T, C, device=DEV, dtype=torch.bfloat16)
        return d
    K, V, HV, H = (c[k] for k in ("K", "V", "HV", "H"))
    kda = c.get("kda", False)
    d["mixed"] = torch.nn.functional.silu(randn(T, 2 * H * K + HV * V)).bfloat16()       # what the conv leaves
    d["b"] = randn(T, HV).bfloat16()
    if c.get("glb", 0.0):
        d["A_log"], d["dt_bias"] = 0.5 * randn(HV), 0.5 * randn(HV * K) - 4
    else:
        # decays as trained layers have them: rates 1 to 16 a head, time steps 1e-3 to 0.1 over their logarithm
        d["A_log"] = torch.log(1 + 15 * rand(HV))
        d["dt_bias"] = torch.log(torch.expm1(torch.exp(math.log(1e-3) + math.log(100) * rand(HV * (K if kda else 1)))))
    d["a"] = (0.5 * randn(T, HV, K) if kda else 0.5 * randn(T, HV)).bfloat16()
    d["S"] = torch.zeros(2 * N + 1, HV, V, K, device=DEV)
    d["S"][1:N + 1] = 0.1 * randn(N, HV, V, K)
    d["out"] = torch.empty(T, HV, V, device=DEV, dtype=torch.bfloat16)
    return d


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


# ---- the framework's operators ---------------------------------------------------------------------------------------
def _own_prefill(d):
    from leapquant_amd import seq
    seq.delta_prefill(d["S"], d["mixed"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["idx"], d["loc"], d["out"],
                      d["case"]["H"], src=d["src"])
    return d["out"], d["S"][d["case"]["N"] + 1:]


def _own_steps(d):
    from leapquant_amd import seq
    seq.delta_steps(d["S"], d["mixed"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["idx"], d["loc"], d["out"],
                    d["case"]["H"], src=d["src"], kda=d["case"]["kda"], gate_lower_bound=d["case"]["glb"])
    return d["out"], d["S"][d["case"]["N"] + 1:]


def _own_conv(d):
    from leapquant_amd import seq
    seq.conv_prefill(d["x"], d["taps"], d["w"], d["bias"], d["idx"], d["loc"], d["out"], src=d["src"])
    return d["out"], d["taps"][d["case"]["N"] + 1:]


def _own_gated(d):
    from leapquant_amd import seq
    seq.gated_norm(d["x"], d["z"], d["w"], d["out"], eps=EPS, gate=d["case"]["act"])
    return d["out"]


def _own_add(d):
    from leapquant_amd import seq
    seq.add_norm(d["x"], d["y"], d["w"], d["res"], d["out"], eps=EPS, scale=d["case"]["scale"])
    return d["res"], d["out"]


_own = {"prefill": _own_prefill, "steps": _own_steps, "conv": _own_conv, "gated": _own_gated, "add": _own_add}


# ---- plain forms: fp32, elementary operations ---------------------------------------------------------------------------
def _where_tokens(d, length):
    """[N, length] rows of the packed tokens of each sequence, and which of them there are."""
    at = d["loc"][:-1, None].long() + torch.arange(length, device=DEV)
    live = at < d["loc"][1:, None]
    return torch.where(live, at, torch.zeros_like(at)), live


def _heads(d, x):
    """Normalised queries and keys at the value heads, values: [N, HV, tokens, K or V], fp32."""
    c = d["case"]
    K, V, HV, H = (c[k] for k in ("K", "V", "HV", "H"))
    N, L = x.shape[:2]
    q, k, v = x.split([H * K, H * K, HV * V], -1)
    q, k, v = q.view(N, L, H, K), k.view(N, L, H, K), v.view(N, L, HV, V)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) * K ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    return [y.repeat_interleave(HV // y.shape[2], 2).transpose(1, 2).contiguous() for y in (q, k, v)]


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _start(d):
    src = d["src"].long()
    return d["S"][src] * (src > 0).view(-1, 1, 1, 1)


def _finish(d, o, S):
    """o [N, HV, tokens, V] back to packed rows in bf16, states to their slots."""
    rows, live = _where_tokens(d, o.shape[2])
    out = torch.empty_like(d["out"])
    out[rows[live]] = o.transpose(1, 2)[live].bfloat16()
    d["S"][d["idx"].long()] = S
    return out, d["S"][d["case"]["N"] + 1:]


def _plain_prefill(d):
    c, Cn = d["case"], 64
    K, V, HV = c["K"], c["V"], c["HV"]
    n = -(-max(d["lens"]) // Cn)
    rows, live = _where_tokens(d, n * Cn)
    N = rows.shape[0]
    m = live[..., None]
    q, k, v = (y.view(N, HV, n, Cn, -1) for y in _heads(d, d["mixed"][rows].float() * m))
    g = -torch.exp(d["A_log"]) * _softplus(d["a"][rows].float() + d["dt_bias"]) * m
    beta = torch.sigmoid(d["b"][rows].float()) * m
    g, beta = (y.transpose(1, 2).reshape(N, HV, n, Cn) for y in (g, beta))
    G = g.cumsum(-1)
    low = torch.ones(Cn, Cn, device=DEV, dtype=torch.bool).tril()
    decay = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], torch.full((), -math.inf, device=DEV)))
    kt = k.transpose(-1, -2).contiguous()
    P = torch.matmul(q, kt) * decay
    M = -torch.matmul(k, kt) * decay.tril(-1) * beta[..., None]
    for i in range(1, Cn):                               # rows of (I + A)^-1 by substitution, all chunks at once
        M[..., i, :i] += torch.matmul(M[..., i:i + 1, :i], M[..., :i, :i])[..., 0, :]
    M = (M + torch.eye(Cn, device=DEV)) * beta[..., None, :]
    eG = G.exp()[..., None]
    kd, qd, kl = k * eG, q * eG, k * torch.exp(G[..., -1:] - G)[..., None]
    S = _start(d).transpose(-1, -2).contiguous()         # [N, HV, K, V]
    o = torch.empty_like(v)
    for i in range(n):
        U = torch.matmul(M[:, :, i], v[:, :, i] - torch.matmul(kd[:, :, i], S))
        o[:, :, i] = torch.matmul(qd[:, :, i], S) + torch.matmul(P[:, :, i], U)
        S = S * eG[:, :, i, -1:] + torch.matmul(kl[:, :, i].transpose(-1, -2).contiguous(), U)
    return _finish(d, o.view(N, HV, n * Cn, V), S.transpose(-1, -2))


def _plain_steps(d):
    c = d["case"]
    L, HV = c["most"], c["HV"]
    rows, live = _where_tokens(d, L)
    m = live[..., None]
    q, k, v = _heads(d, d["mixed"][rows].float() * m)
    N = rows.shape[0]
    x = d["a"][rows].float().view(N, L, HV, -1) + d["dt_bias"].view(HV, -1)
    ea = torch.exp(d["A_log"]).view(HV, 1)
    g = (c["glb"] * torch.sigmoid(ea * x) if c["glb"] else -ea * _softplus(x)) * m[..., None]
    alpha, beta = g.exp(), torch.sigmoid(d["b"][rows].float()) * m
    S, o = _start(d), torch.empty_like(v)
    for t in range(L):
        S = S * alpha[:, t, :, None, :]
        u = beta[:, t, :, None] * (v[:, :, t] - (S * k[:, :, t, None]).sum(-1))
        S = S + u[..., None] * k[:, :, t, None]
        o[:, :, t] = (S * q[:, :, t, None]).sum(-1)
    return _finish(d, o, S)


def _plain_conv(d):
    x, w, loc = d["x"].float(), d["w"].float(), d["loc"].long()
    taps = d["taps"][d["src"].long()].float() * (d["src"] > 0).view(-1, 1, 1)
    t = torch.arange(x.shape[0], device=DEV)
    of = torch.searchsorted(loc[1:].contiguous(), t, right=True)
    at = t - loc[of]                                     # the token's place in its sequence
    y = x * w[:, 3]
    for back in (1, 2, 3):
        here = torch.where((at >= back)[:, None], x[(t - back).clamp(min=0)], taps[of, :, (3 + at - back).clamp(0, 2)])
        y = y + here * w[:, 3 - back]
    if d["bias"] is not None:
        y = y + d["bias"].float()
    y = y * torch.sigmoid(y)
    n = loc[1:] - loc[:-1]
    last = [torch.where((n + i >= 3)[:, None], x[(loc[1:] - 3 + i).clamp(min=0)],
                        taps[torch.arange(len(n), device=DEV), :, (n + i).clamp(max=2)]) for i in range(3)]
    d["taps"][d["idx"].long()] = torch.stack(last, -1).bfloat16()
    return y.bfloat16(), d["taps"][d["case"]["N"] + 1:]


def _plain_gated(d):
    x, z = d["x"].float(), d["z"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * d["w"].float()
    s = torch.sigmoid(z)
    return (y * (s if d["case"]["act"] == "sigmoid" else z * s)).bfloat16()


def _plain_add(d):
    r = d["x"].float() + d["case"]["scale"] * d["y"].float()
    return r.bfloat16(), (r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * d["w"].float()).bfloat16()


_plain = {"prefill": _plain_prefill, "steps": _plain_steps, "conv": _plain_conv, "gated": _plain_gated, "add": _plain_add}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    if op == "gated":
        n = c["rows"] * c["HV"] * c["D"]
        return {"bytes": 6.0 * n, "flops": 10.0 * n}
    if op == "add":
        n = c["rows"] * c["D"]
        return {"bytes": 8.0 * n, "flops": 6.0 * n}
    N, T = c["N"], sum(_lens(c))
    if op == "conv":
        C = c["C"]
        return {"bytes": C * (4.0 * T + 6.0 * N * (1 + c["carry"]) + 8), "flops": 13.0 * T * C}
    K, V, HV, H = (c[k] for k in ("K", "V", "HV", "H"))
    token = 2 * (2 * H * K + HV * V) + 2 * HV * (K if c.get("kda") else 1) + 2 * HV + 2 * HV * V
    return {"bytes": float(T * token + N * HV * 4 * V * K * (1 + c["carry"])), "flops": 6.0 * T * HV * K * V}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------
def _exact_delta(d):
    """Token by token over the batch; a sequence that has ended keeps its state (decay 1, beta 0)."""
    c = d["case"]
    K, V, HV, H, N = (c[k] for k in ("K", "V", "HV", "H", "N"))
    S = torch.zeros(N, HV, V, K, device=DEV, dtype=F64)
    for n, s in enumerate(d["src"].tolist()):
        if s > 0:
            S[n] = d["S"][s].to(F64)
    lens, loc = torch.tensor(d["lens"], device=DEV), d["loc"][:-1].long()
    out = torch.zeros(sum(d["lens"]), HV, V, device=DEV, dtype=F64)
    ea, dt = d["A_log"].to(F64).exp().view(HV, 1), d["dt_bias"].to(F64).view(HV, -1)
    order = torch.argsort(lens, descending=True)         # the longest first: those still running are the first rows
    S, lens, loc = S[order], lens[order], loc[order]
    ends = sorted(d["lens"], reverse=True)
    run_n = N
    for t in range(ends[0]):
        while ends[run_n - 1] <= t:
            run_n -= 1
        r = loc[:run_n] + t
        x = d["mixed"][r].to(F64)
        q, k, v = x[:, :H * K].view(-1, H, K), x[:, H * K:2 * H * K].view(-1, H, K), x[:, 2 * H * K:].view(-1, HV, V)
        q = (q / (q.pow(2).sum(-1, keepdim=True) + EPS).sqrt() / math.sqrt(K)).repeat_interleave(HV // H, 1)
        k = (k / (k.pow(2).sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(HV // H, 1)
        z = d["a"][r].to(F64).view(run_n, HV, -1) + dt
        g = c["glb"] / (1 + torch.exp(-ea * z)) if c.get("glb") else -ea * torch.logaddexp(z, torch.zeros_like(z))
        A = S[:run_n]
        A.mul_(g.exp().unsqueeze(2))
        u = (v - torch.matmul(A, k.unsqueeze(-1)).squeeze(-1)) / (1 + torch.exp(-d["b"][r].to(F64))).unsqueeze(-1)
        A.addcmul_(u.unsqueeze(-1), k.unsqueeze(2))
        out[r] = torch.matmul(A, q.unsqueeze(-1)).squeeze(-1)
    slots = torch.zeros(N, HV, V, K, device=DEV, dtype=F64)
    slots[d["idx"].long()[order] - N - 1] = S
    return out, slots


def _exact_conv(d):
    w = d["w"].to(F64)
    ys, slots = [], torch.zeros(d["case"]["N"], w.shape[0], 3, device=DEV, dtype=F64)
    for n, (s, i) in enumerate(zip(d["src"].tolist(), d["idx"].tolist())):
        lo = sum(d["lens"][:n])
        seq = d["x"][lo:lo + d["lens"][n]].to(F64)
        seq = torch.cat([d["taps"][s].to(F64).T if s > 0 else torch.zeros(3, w.shape[0], device=DEV, dtype=F64), seq])
        y = (seq.unfold(0, 4, 1) * w).sum(-1)
        if d["bias"] is not None:
            y = y + d["bias"].to(F64)
        ys.append(y / (1 + torch.exp(-y)))
        slots[i - d["case"]["N"] - 1] = seq[-3:].T
    return torch.cat(ys), slots


def _exact_gated(d):
    x, z = d["x"].to(F64), d["z"].to(F64)
    y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * d["w"].to(F64) / (1 + torch.exp(-z))
    return y if d["case"]["act"] == "sigmoid" else y * z


def _exact_add(d):
    r = d["x"].to(F64) + d["case"]["scale"] * d["y"].to(F64)
    return r, r / (r.pow(2).sum(-1, keepdim=True) / r.shape[-1] + EPS).sqrt() * d["w"].to(F64)


def exact(case, seed):
    d = prepare(case, seed)
    return {"prefill": _exact_delta, "steps": _exact_delta, "conv": _exact_conv, "gated": _exact_gated,
            "add": _exact_add}[case["op"]](d)
