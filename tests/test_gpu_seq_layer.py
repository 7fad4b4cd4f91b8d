"""The operators for whole sequences as a layer uses them (MI355X): prompts through `LeapQuantState.prefill` into 8-bit
checkpoints and decode from there, and the block of examples/gdn_block.py, against the recurrence in 64 bits.

Bars.  The recurrence of a prefill: the operators' own (tests/test_gpu_seq.py).  After a checkpoint: 3e-2 of the outputs' norm,
as for the 8-bit decode.  The block: every stage rounds to bf16 (2^-9 of an element at most, about 1.1e-3 of a norm): input
projection, conv, rule, gated norm, output projection, sum: sqrt(6) 1.1e-3 = 2.7e-3 of the block's contribution if no stage
amplified; the norms of q, k and of the heads may by small factors: 1e-2.
"""
import numpy as np
import pytest
import torch

from tests import seq_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def rel(got, want):
    return float(np.linalg.norm(R.f64(got) - want) / np.linalg.norm(want))


def _args(d, lo=0, hi=None):
    return [d[k][lo:hi].to(DEV) for k in ("mixed", "a", "b")] + [d["A_log"].to(DEV), d["dt_bias"].to(DEV)]


@pytest.mark.parametrize("kda,H", [(False, 2), (True, 4)])
@pytest.mark.parametrize("lens", [[5, 16, 1], [70, 0, 33], [300, 20, 64]], ids=str)
def test_prefill_then_decode(kda, H, lens):
    """Prompts from zero, their next pieces from the checkpoints, and tokens by `decode` after them."""
    from leapquant_amd.state import LeapQuantState
    HV, more, steps, glb = 4, [20, 3, 40], 3, -5.0 if kda else 0.0
    N = len(lens)
    spans = [list(x) for x in zip(lens, more, [steps] * N)]
    d = R.delta_inputs(31, [sum(x) for x in spans], HV, H, 128, 128, kda=kda, glb=glb, NS=N + 1)
    if kda:
        d["a"], d["dt_bias"] = d["a"], d["dt_bias"].reshape(-1)
    d["idx"] = d["src"] = torch.arange(1, N + 1, dtype=torch.int32)
    ref = dict(d, S=torch.zeros_like(d["S"]))
    want, _ = R.delta_ref(ref, H, glb=glb)
    ssm = torch.full((N + 1, HV, 128, 128), float("nan"), device=DEV)
    st = LeapQuantState(ssm, H, kda=kda, gate_lower_bound=glb)
    idx, starts = d["idx"].to(DEV), d["loc"].numpy()
    for piece in range(2):
        rows = [np.arange(starts[n] + sum(spans[n][:piece]), starts[n] + sum(spans[n][:piece + 1])) for n in range(N)]
        loc = torch.tensor(np.concatenate([[0], np.cumsum([len(r) for r in rows])]), dtype=torch.int32, device=DEV)
        rows = np.concatenate(rows)
        p = dict(d, **{k: d[k][rows] for k in ("mixed", "a", "b")})
        out = torch.full((len(rows), HV, 128), 7.0, dtype=torch.bfloat16, device=DEV)
        st.prefill(ssm, *_args(p), idx, loc, out, has_state=torch.full((N,), bool(piece), device=DEV))
        assert rel(out, want[rows]) <= (3e-2 if piece else 4e-3), piece
        assert int(st.hcnt[1:].abs().sum()) == 0
    for t in range(steps):
        rows = np.array([starts[n] + lens[n] + more[n] + t for n in range(N)])
        p = dict(d, **{k: d[k][rows] for k in ("mixed", "a", "b")})
        out = torch.empty(N, HV, 128, dtype=torch.bfloat16, device=DEV)
        st.decode(ssm, *_args(p), idx, out)
        assert rel(out, want[rows]) <= 3e-2, t


def test_prefill_leaves_other_slots(lens=(40, 9)):
    """Padding sequences and slots that a call does not name keep their checkpoints; has_state is per sequence."""
    from leapquant_amd.state import LeapQuantState
    d = R.delta_inputs(32, [40, 9, 50], 4, 2, 128, 128, NS=5)
    ssm = torch.randn(5, 4, 128, 128, device=DEV) * 0.05
    st = LeapQuantState(ssm, 2)
    st.quantize(ssm, torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=DEV))
    before = ssm.clone()
    fp = ssm.clone()
    LeapQuantState(fp, 2).dequantize(fp, torch.tensor([2], dtype=torch.int32, device=DEV))
    out = torch.full((99, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    idx = torch.tensor([2, 0, 4], dtype=torch.int32, device=DEV)
    st.prefill(ssm, *_args(d), idx, d["loc"].to(DEV), out, has_state=torch.tensor([True, True, False], device=DEV))
    ref = dict(d, S=fp.cpu(), idx=torch.tensor([2, 0, 4]), src=torch.tensor([2, 0, 0]))
    want, _ = R.delta_ref(ref, 2)
    assert rel(out[:40], want[:40]) <= 4e-3 and rel(out[49:], want[49:]) <= 4e-3 and not out[40:49].any()
    for s in (0, 1, 3):
        assert torch.equal(ssm[s].view(torch.int32), before[s].view(torch.int32)), s


def test_block():
    """The block's prefill and its decode against the same block in 64 bits."""
    from examples.gdn_block import GDNBlock
    lens, steps, hidden, H, HV, D = [75, 1, 40], 3, 256, 2, 4, 128
    N, T = len(lens), sum(lens)
    block = GDNBlock(hidden, H, HV, D, N)
    g = torch.Generator().manual_seed(33)
    x = torch.randn(T + steps * N, hidden, generator=g).to(R.BF16)
    loc = np.concatenate([[0], np.cumsum(lens)])
    rows = [np.concatenate([np.arange(loc[n], loc[n + 1]), T + n + N * np.arange(steps)]) for n in range(N)]   # of each sequence
    idx = torch.arange(1, N + 1, dtype=torch.int32, device=DEV)
    got = [block.prefill(x[:T].to(DEV), x[:T].to(DEV), idx, torch.tensor(loc, dtype=torch.int32, device=DEV))]
    for t in range(steps):
        xt = x[T + t * N:T + (t + 1) * N].to(DEV)
        got.append(block.decode(xt, xt, idx))
    y, h = (torch.cat([p[i] for p in got]) for i in range(2))

    order = np.concatenate(rows)
    at = np.concatenate([[0], np.cumsum([len(r) for r in rows])])
    xs = R.f64(x)[order]
    mixed, z, b, a = np.split(xs @ R.f64(block.w_in), np.cumsum([block.C, HV * D, HV]), 1)
    m, _ = R.conv(mixed, np.zeros((N + 1, block.C, 3)), R.f64(block.w_conv), None, range(1, N + 1), at)
    o, _ = R.delta(np.zeros((N + 1, HV, D, D)), m, a[..., None], b, R.f64(block.A_log), R.f64(block.dt_bias)[:, None],
                   range(1, N + 1), at, H)
    z = z.reshape(-1, HV, D)
    o = R.rms(o, np.ones(D), 1e-6, 0.0) * z * R.sigmoid(z)
    add = np.empty((len(order), hidden))
    add[order] = o.reshape(len(order), -1) @ R.f64(block.w_out)
    r = R.f64(x) + add
    part = slice(0, T)
    assert np.linalg.norm(R.f64(y)[part] - r[part]) <= 1e-2 * np.linalg.norm(add[part])
    assert rel(h[part], R.rms(r[part], np.ones(hidden), 1e-6, 0.0)) <= 1e-2
    part = slice(T, None)                                 # on the 8-bit state
    assert np.linalg.norm(R.f64(y)[part] - r[part]) <= 3e-2 * np.linalg.norm(add[part])
