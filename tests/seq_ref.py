"""The sequence operators' definitions in 64 bits (numpy, CPU), token by token, and seeded inputs for their tests."""
import numpy as np
import torch

BF16 = torch.bfloat16


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def log_gate(a, A_log, dt_bias, glb=0.0):
    """a [.., HV, KA], A_log [HV], dt_bias [HV, KA]"""
    x, ea = a + dt_bias, np.exp(A_log)[:, None]
    return glb * sigmoid(ea * x) if glb else -ea * np.logaddexp(x, 0)


def delta(S, mixed, a, b, A_log, dt_bias, idx, loc, H, src=None, scale=None, glb=0.0):
    """out [T, HV, V] and the cache after the call; arrays in fp64, S [NS, HV, V, K], a [T, HV, KA], dt_bias [HV, KA]."""
    NS, HV, V, K = S.shape
    S, out = S.copy(), np.zeros((mixed.shape[0], HV, V))
    src = idx if src is None else src
    old = S.copy()
    scale = K ** -0.5 if scale is None else scale
    for n in range(len(idx)):
        if not 0 < idx[n] < NS:
            continue
        M = old[src[n]].copy() if 0 < src[n] < NS else np.zeros((HV, V, K))
        for t in range(loc[n], loc[n + 1]):
            q, k, v = np.split(mixed[t], [H * K, 2 * H * K])
            q, k, v = q.reshape(H, K), k.reshape(H, K), v.reshape(HV, V)
            q = np.repeat(q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6) * scale, HV // H, 0)
            k = np.repeat(k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6), HV // H, 0)
            M *= np.exp(log_gate(a[t], A_log, dt_bias, glb))[:, None, :]
            u = sigmoid(b[t])[:, None] * (v - np.einsum("hvk,hk->hv", M, k))
            M += u[:, :, None] * k[:, None, :]
            out[t] = np.einsum("hvk,hk->hv", M, q)
        S[idx[n]] = M
    return out, S


def conv(x, state, w, bias, idx, loc, src=None, silu=True):
    """x [T, C], state [NS, C, 3], w [C, 4]: out [T, C] and the state after the call."""
    NS = state.shape[0]
    old, state, out = state, state.copy(), np.zeros_like(x)
    src = idx if src is None else src
    for n in range(len(idx)):
        if not 0 < idx[n] < NS:
            continue
        taps = old[src[n]].T if 0 < src[n] < NS else np.zeros((3, x.shape[1]))
        s = np.concatenate([taps, x[loc[n]:loc[n + 1]]])
        for t in range(loc[n], loc[n + 1]):
            y = (s[t - loc[n]:t - loc[n] + 4] * w.T).sum(0) + (0 if bias is None else bias)
            out[t] = y * sigmoid(y) if silu else y
        state[idx[n]] = s[len(s) - 3:].T
    return out, state


def rms(x, w, eps, offset):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (offset + w)


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def delta_inputs(seed, lens, HV, H, K, V, kda=False, glb=0.0, gate=None, NS=None):
    """Inputs on the CPU: tokens after a conv with SiLU, decays as trained layers have them (gate None) or a raw gate of
    that value everywhere; sequences start from slots 1 .. N and end in N + 1 .. 2 N."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)                    # noqa: E731
    T, N, KA = sum(lens), len(lens), K if kda else 1
    d = dict(mixed=torch.nn.functional.silu(rn(T, 2 * H * K + HV * V)).to(BF16), b=rn(T, HV).to(BF16),
             a=(0.5 * rn(T, HV, KA) if gate is None else torch.full((T, HV, KA), float(gate))).to(BF16),
             S=0.1 * rn(NS or 2 * N + 1, HV, V, K))
    if glb:
        d["A_log"], d["dt_bias"] = 0.5 * rn(HV), 0.5 * rn(HV, KA) - 4
    else:
        d["A_log"] = torch.log(1 + 15 * torch.rand(HV, generator=g))
        dt = torch.exp(np.log(1e-3) + np.log(100) * torch.rand(HV, KA, generator=g))
        d["dt_bias"] = torch.log(torch.expm1(dt))
    if not kda:
        d["a"] = d["a"][..., 0]
    d["loc"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)
    d["src"] = torch.arange(1, N + 1, dtype=torch.int32)
    d["idx"] = torch.arange(N + 1, 2 * N + 1, dtype=torch.int32)
    return d


def delta_ref(d, H, src="src", glb=0.0, scale=None):
    HV = d["S"].shape[1]
    a, b = f64(d["a"]), f64(d["b"])
    return delta(f64(d["S"]), f64(d["mixed"]), a.reshape(a.shape[0], HV, -1), b, f64(d["A_log"]),
                 f64(d["dt_bias"]).reshape(HV, -1), d["idx"].tolist(), d["loc"].tolist(), H,
                 src=d[src].tolist() if src else None, glb=glb, scale=scale)
