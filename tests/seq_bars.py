"""Bars of the sequence operators' outputs, token by token and head by head, and the chunked form of the gated delta rule in 64 bits
with the roundings of chosen operands put in: what a bar has to let through, and what it has to catch.

bf16 has 8 bits: a rounding moves a value by 2^-8 of it at most, 1.7e-3 in the root mean square.  Where fp32 arithmetic is
rounded once, what comes before moves it further by 2^-24 of its terms, a few times and more from token to token: 1e-5 of the
terms' root sum of squares over K, sqrt(sum_k S_vk^2 q_k^2).  The output itself is no measure of that: a query nearly orthogonal
to the only key that a strong decay has left makes it as small as one likes.  (Where outputs do not cancel, its rms over V is.)

The chunked form carries the state (as it is read) and W, the weights of a chunk's values in its outputs, in two bf16 parts:
2.8e-6 of an element short in the mean, 2^-16 at most.  An output sums such errors of random sign over K channels and the
chunk's 32 tokens, whose terms may be a few times those: about 1e-5 of them, five deviations, and twice that: 2^-13.  With one
part, 1.7e-3 in the mean, it would be 14 times over the bar.

Its states: three parts (5e-9) in what is appended, two in the state that is read for it, so that what a chunk appends is off by
2.8e-6 of it in the mean, of random signs from chunk to chunk; with the fp32 sums' 2e-7 within 4e-6 of the norm."""
import numpy as np

from tests import seq_ref as R

ONCE, CHUNKS, STATE = 1e-5, 2.0 ** -13, 4e-6


def off(got, want, more, scale=None):
    """How many elements of got [T, HV, V] are further off than a rounding and `more` of `scale`, their terms (None: the rms of
    their token and head)."""
    scale = np.sqrt((want ** 2).mean(-1, keepdims=True)) if scale is None else scale
    return int((~(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + more * scale)).sum())


def near(out, want, more, scale=None):
    got = R.f64(out)
    bad = off(got, want, more, scale)
    assert not bad, (bad, float(np.abs(got - want).max()))


def states_near(S, want, bar=STATE):
    """Every head's state by its own norm."""
    got = R.f64(S)
    err, norm = (np.sqrt((x ** 2).sum((-1, -2))) for x in (got - want, want))
    assert (err <= bar * norm).all(), float((err / np.maximum(norm, 1e-300)).max())


def terms(d, H, glb=0.0, scale=None):
    """sqrt(sum_k S_vk^2 q_k^2) of every output [T, HV, V]: the states by the definition, one token's at a time."""
    NS, HV, V, K = d["S"].shape
    mixed, S, loc, src, idx = R.f64(d["mixed"]), R.f64(d["S"]), d["loc"].tolist(), d["src"].tolist(), d["idx"].tolist()
    T = mixed.shape[0]
    g = R.log_gate(R.f64(d["a"]).reshape(T, HV, -1), R.f64(d["A_log"]), R.f64(d["dt_bias"]).reshape(HV, -1), glb)
    beta, out = R.sigmoid(R.f64(d["b"])), np.zeros((T, HV, V))
    unit = lambda x: np.repeat(x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6), HV // H, 0)       # noqa: E731
    for n in range(len(idx)):
        if not 0 < idx[n] < NS:
            continue
        M = S[src[n]].copy() if 0 < src[n] < NS else np.zeros((HV, V, K))
        for t in range(loc[n], loc[n + 1]):
            q, k, v = np.split(mixed[t], [H * K, 2 * H * K])
            q, k, v = unit(q.reshape(H, K)) * (K ** -0.5 if scale is None else scale), unit(k.reshape(H, K)), v.reshape(HV, V)
            M *= np.exp(g[t])[:, None, :]
            M += (beta[t][:, None] * (v - (M @ k[..., None])[..., 0]))[..., None] * k[:, None, :]
            out[t] = np.sqrt((M * M) @ (q * q)[..., None])[..., 0]
    return out


def bf16(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).double().numpy()


def parts(x, n):
    """x in n bf16 parts."""
    y = np.zeros_like(x)
    for _ in range(n):
        y = y + bf16(x - y)
    return y


def chunked(mixed, a, b, A_log, dt_bias, H, HV, K, V, C=32, w_parts=None, s_parts=None):
    """The rule of one sequence from zero in chunks, W and the state as it is read in so many bf16 parts: out [T, HV, V]."""
    T = mixed.shape[0]
    out, S = np.zeros((T, HV, V)), np.zeros((HV, V, K))
    cut = lambda x, n: x if n is None else parts(x, n)                   # noqa: E731
    for lo in range(0, T, C):
        m, n = mixed[lo:lo + C], min(C, T - lo)
        q, k, v = np.split(m, [H * K, 2 * H * K], 1)
        q, k, v = q.reshape(n, H, K), k.reshape(n, H, K), v.reshape(n, HV, V)
        q = np.repeat(q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6) * K ** -0.5, HV // H, 1).transpose(1, 0, 2)
        k = np.repeat(k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6), HV // H, 1).transpose(1, 0, 2)
        v = v.transpose(1, 0, 2)
        G = np.cumsum(R.log_gate(a[lo:lo + n, :, None], A_log, dt_bias[:, None])[..., 0], 0).T
        beta = R.sigmoid(b[lo:lo + n]).T
        dec = np.exp(np.minimum(G[:, :, None] - G[:, None, :], 0))
        A = np.tril(beta[:, :, None] * dec * (k @ k.transpose(0, 2, 1)), -1)
        Tm = np.linalg.inv(np.eye(n) + A) * beta[:, None, :]
        W = cut(np.tril(dec * (q @ k.transpose(0, 2, 1))) @ Tm, w_parts)
        Sr = cut(S, s_parts)
        eG = np.exp(G)[:, :, None]
        Rv = v - eG * (k @ Sr.transpose(0, 2, 1))
        out[lo:lo + n] = (eG * (q @ Sr.transpose(0, 2, 1)) + W @ Rv).transpose(1, 0, 2)
        S = eG[:, -1:] * S + (Tm @ Rv).transpose(0, 2, 1) @ (np.exp(G[:, -1:] - G)[:, :, None] * k)
    return out
