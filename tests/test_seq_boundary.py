"""CPU tests of liblq_seq's boundary: it exports what include/lq_seq.h declares, its entry points refuse bad arguments before
any launch, and the Python operators refuse what the kernels do not take.  No kernel is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from tests import seq_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from leapquant_amd import _lib
    if not os.path.exists(_lib.SEQ_LIB_PATH):
        from leapquant_amd import build
        build.build()
    return _lib.seq_lib()


def test_header_binding_and_library_agree(lib):
    from leapquant_amd import _lib
    src = open(os.path.join(ROOT, "include", "lq_seq.h")).read()
    names = set(re.findall(r"^(?:int|long long)\s+(lq_\w+)\s*\(", src, flags=re.M))
    assert names == set(_lib.SEQ_SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.SEQ_LIB_PATH], capture_output=True, text=True, check=True)
    assert names <= {ln.split()[-1] for ln in out.stdout.splitlines() if ln.strip()}


def test_importable_under_the_reference_name():
    import leapquant.seq
    import leapquant_amd.seq
    assert leapquant.seq is leapquant_amd.seq


def _delta(**kw):
    from leapquant_amd import _lib
    d = dict(S=16, slot_stride=4 * 128 * 128, NS=3, HV=4, H=2, K=128, V=128, mixed=16, a=16, b=16, A_log=16, dt_bias=16,
             out=16, mixed_ld=1024, a_ld=4, b_ld=4, scale=0.1, gate_bf16=0, kda=0, glb=0.0)
    d.update(kw)
    return _lib.LqDelta(**d)


def _seqs(**kw):
    from leapquant_amd import _lib
    return _lib.LqSeqs(**{**dict(loc=16, idx=16, src=None, N=0, T=0), **kw})


BAD_DELTA = [dict(K=96), dict(V=64), dict(K=64, V=96), dict(H=3), dict(H=0), dict(HV=0), dict(NS=0), dict(S=None), dict(S=8),
             dict(slot_stride=100), dict(slot_stride=4 * 128 * 128 + 2), dict(mixed_ld=1016), dict(mixed_ld=1028),
             dict(a_ld=3), dict(b_ld=3), dict(mixed=8), dict(out=8), dict(A_log=None), dict(dt_bias=None), dict(gate_bf16=4),
             dict(kda=2), dict(glb=-5.0), dict(kda=1), dict(kda=1, a_ld=514), dict(kda=1, a_ld=512, a=12)]


@pytest.mark.parametrize("bad", BAD_DELTA, ids=str)
def test_delta_refuses(lib, bad):
    d, s = _delta(**bad), _seqs()
    assert lib.lq_delta_steps(ctypes.byref(d), ctypes.byref(s), None) == -1
    assert lib.lq_delta_prefill(ctypes.byref(d), ctypes.byref(s), None, 0, None) == -1


def test_delta_takes_and_refuses_batches(lib):
    ok = _delta()
    for s, rc in ((_seqs(), 0), (_seqs(N=-1), -1), (_seqs(T=-1), -1), (_seqs(N=1, loc=None), -1), (_seqs(N=1, idx=None), -1)):
        assert lib.lq_delta_steps(ctypes.byref(ok), ctypes.byref(s), None) == rc
        assert lib.lq_delta_prefill(ctypes.byref(ok), ctypes.byref(s), None, 0, None) == rc
    assert lib.lq_delta_steps(None, ctypes.byref(_seqs()), None) == -1
    assert lib.lq_delta_steps(ctypes.byref(ok), None, None) == -1
    kda = _delta(kda=1, a_ld=512, glb=-5.0)
    assert lib.lq_delta_steps(ctypes.byref(kda), ctypes.byref(_seqs()), None) == 0
    assert lib.lq_delta_prefill(ctypes.byref(kda), ctypes.byref(_seqs()), None, 0, None) == -1       # GDN only
    s = _seqs(N=2, T=100)
    need = lib.lq_delta_workspace(ctypes.byref(ok), ctypes.byref(s))
    if need > 0:
        for work, n in ((None, need), (16, need - 1), (8, need)):
            assert lib.lq_delta_prefill(ctypes.byref(ok), ctypes.byref(s), work, n, None) == -1


def _norm(**kw):
    from leapquant_amd import _lib
    d = dict(x=16, z=16, weight=16, res=16, out=16, x_ld=64, x_hd=64, z_ld=64, z_hd=64, o_ld=64, o_hd=64, rows=0, heads=1,
             D=64, eps=1e-6, scale=1.0, offset=0.0, act=0, weight_bf16=0)
    d.update(kw)
    return _lib.LqNorm(**d)


@pytest.mark.parametrize("bad", [dict(D=0), dict(D=16385), dict(rows=-1), dict(heads=0), dict(act=2), dict(weight_bf16=2),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(rows=1, x=None), dict(rows=1, out=None)], ids=str)
def test_norms_refuse(lib, bad):
    n = _norm(**bad)
    assert lib.lq_gated_norm(ctypes.byref(n), None) == -1
    assert lib.lq_add_norm(ctypes.byref(n), None) == -1
    assert lib.lq_gated_norm(ctypes.byref(_norm()), None) == 0
    assert lib.lq_add_norm(ctypes.byref(_norm(rows=1, res=None)), None) == -1


@pytest.mark.parametrize("bad", [dict(W=3), dict(silu=2), dict(NS=0), dict(weight=12), dict(state=None), dict(slot_stride=100),
                                 dict(ch_stride=0), dict(tap_stride=0)], ids=str)
def test_conv_refuses(lib, bad):
    from leapquant_amd import _lib
    f = dict(state=16, weight=16, bias=None, slot_stride=192, ch_stride=3, tap_stride=1, W=4, silu=1, NS=2)
    cv = _lib.LqConv(**{**f, **bad})
    s = ctypes.byref(_seqs())
    assert lib.lq_conv_seq(ctypes.byref(cv), s, 16, 64, 16, 64, None) == -1
    ok = ctypes.byref(_lib.LqConv(**f))
    assert lib.lq_conv_seq(ok, s, 16, 64, 16, 64, None) == 0
    assert lib.lq_conv_seq(ok, s, 16, 63, 16, 64, None) == -1
    assert lib.lq_conv_seq(ok, s, 16, 64, 16, 0, None) == -1


# ---- the Python operators -----------------------------------------------------------------------------------------------
def _args(**kw):
    d = R.delta_inputs(1, [5, 3], 4, 2, 128, 128)
    d["out"] = torch.empty(8, 4, 128, dtype=torch.bfloat16)
    d["H"] = 2
    d.update(kw)
    return [d[k] for k in ("S", "mixed", "a", "b", "A_log", "dt_bias", "idx", "loc", "out", "H")], dict(src=d["src"])


BAD_ARGS = [("S", lambda t: t.double(), TypeError), ("S", lambda t: t[0], TypeError), ("S", lambda t: t[..., :96], ValueError),
            ("S", lambda t: t.transpose(2, 3), ValueError), ("mixed", lambda t: t.float(), TypeError),
            ("mixed", lambda t: t[:, :-8], ValueError), ("mixed", lambda t: t[None], ValueError),
            ("mixed", lambda t: t.t().contiguous().t(), ValueError), ("mixed", lambda t: torch.cat([t, t[:, :4]], 1)[:, 4:], ValueError),
            ("a", lambda t: t.float(), TypeError), ("a", lambda t: t[:4], ValueError), ("b", lambda t: t[:, :3], ValueError),
            ("A_log", lambda t: t[:3], ValueError), ("dt_bias", lambda t: t.repeat(2, 1), ValueError),
            ("idx", lambda t: t.float(), TypeError), ("idx", lambda t: t[:1], ValueError), ("loc", lambda t: t[:2], ValueError),
            ("loc", lambda t: t[:, None], ValueError), ("src", lambda t: t[:1], ValueError), ("out", lambda t: t.float(), ValueError),
            ("out", lambda t: t[:4], ValueError), ("H", lambda t: 3, ValueError), ("H", lambda t: 0, ValueError)]


@pytest.mark.parametrize("name,change,error", BAD_ARGS, ids=lambda v: v if isinstance(v, str) else "")
def test_delta_arguments(name, change, error):
    from leapquant_amd import seq
    args, kw = _args()
    names = ["S", "mixed", "a", "b", "A_log", "dt_bias", "idx", "loc", "out", "H"]
    if name == "src":
        kw["src"] = change(kw["src"])
    else:
        args[names.index(name)] = change(args[names.index(name)])
    for fn in (seq.delta_prefill, seq.delta_steps):
        with pytest.raises(error):
            fn(*args, **kw)


def test_operators_take_gpu_tensors_only():
    from leapquant_amd import seq
    args, kw = _args()
    with pytest.raises(ValueError, match="GPU tensors only"):
        seq.delta_prefill(*args, **kw)
    with pytest.raises(ValueError, match="KDA only"):
        seq.delta_steps(*args, gate_lower_bound=-5.0, **kw)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64)
    for call in (lambda: seq.gated_norm(x, x, w, x), lambda: seq.add_norm(x, x, w, x, x),
                 lambda: seq.conv_prefill(x, torch.zeros(2, 64, 3, dtype=torch.bfloat16), torch.zeros(64, 4, dtype=torch.bfloat16),
                                          None, args[6], args[7], x)):
        with pytest.raises(ValueError, match="GPU tensors only"):
            call()


def test_norm_and_conv_arguments():
    from leapquant_amd import seq
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64)
    i, l = torch.ones(1, dtype=torch.int32), torch.tensor([0, 4])
    st, cw = torch.zeros(2, 64, 3, dtype=torch.bfloat16), torch.zeros(64, 4, dtype=torch.bfloat16)
    for call in (lambda: seq.gated_norm(x, x, w, x, gate="tanh"), lambda: seq.gated_norm(x.float(), x, w, x),
                 lambda: seq.gated_norm(x, x[:2], w, x), lambda: seq.gated_norm(x, x, w[:32], x),
                 lambda: seq.gated_norm(x, x, w.half(), x), lambda: seq.add_norm(x, x.float(), w, x, x),
                 lambda: seq.gated_norm(x, x.t().contiguous().t(), w, x),
                 lambda: seq.add_norm(x, x, w, torch.zeros(4, 72, dtype=torch.bfloat16)[:, :64], x),
                 lambda: seq.conv_prefill(x, st[:, :32], cw, None, i, l, x), lambda: seq.conv_prefill(x, st, cw[:, :3], None, i, l, x),
                 lambda: seq.conv_prefill(x, st, cw[:32], None, i, l, x), lambda: seq.conv_prefill(x, st.float(), cw, None, i, l, x),
                 lambda: seq.conv_prefill(x, st, cw, w, i, l, x), lambda: seq.conv_prefill(x, st, cw, None, i, l, x[:2]),
                 lambda: seq.conv_prefill(x, st, cw, None, i, l[:1], x)):
        with pytest.raises(ValueError):
            call()


def test_direct_calls_leave_all_else_to_the_operators():
    """What the extension in front of the library does not take as it is, it hands back without a launch or an error."""
    from leapquant_amd import _lib
    c = _lib.seq_call()
    t, n = torch.zeros(2, 8, dtype=torch.bfloat16), c.NOT_PLAIN
    idx = torch.zeros(2, dtype=torch.int32)
    for bad in (t, None, 3, "x"):
        assert c.norm(bad, t, t[0], t, None, 1e-6, 0.0, 0.0, 0, False) == n
        assert c.norm(t, t, t[0], t, bad, 1e-6, 0.0, 0.0, 0, True) == n
        assert c.conv(bad, t, t, None, idx, idx, t, None, True) == n
        assert c.delta(bad, t, t, t, t, t, idx, idx, t, None, 2, None, False, 0.0, True) == n
    assert c.norm() == c.conv() == c.delta() == n
    from leapquant_amd import seq
    with pytest.raises(ValueError):
        seq.gated_norm(t, t, torch.ones(8), t)


def test_state_prefill_refuses():
    from leapquant_amd.state import LeapQuantState
    ssm = torch.zeros(3, 4, 128, 128)
    st = LeapQuantState(ssm, 2)
    mixed, a = torch.zeros(5, 1024, dtype=torch.bfloat16), torch.zeros(5, 4, dtype=torch.bfloat16)
    out, p = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(4)
    idx, loc = torch.tensor([1, 2], dtype=torch.int32), torch.tensor([0, 2, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="idx"):
        st.prefill(ssm, mixed, a, a, p, p, idx[None], loc, out)
    with pytest.raises(ValueError, match="has_state"):
        st.prefill(ssm, mixed, a, a, p, p, idx, loc, out, has_state=torch.ones(3, dtype=torch.bool))
    with pytest.raises(ValueError, match="GPU"):
        st.prefill(ssm, mixed, a, a, p, p, idx, loc, out)
    with pytest.raises(ValueError, match="mixed"):
        st.prefill(ssm, mixed[:, 1:], a, a, p, p, idx, loc, out)
