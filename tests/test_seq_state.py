"""`LeapQuantState.prefill` around the sequence operators (CPU): what it does before a call that is refused, and which form of the
rule it picks.  No kernel is launched."""
import pytest
import torch

from leapquant_amd import seq
from leapquant_amd.state import LeapQuantState


def call(N=2, T=5, HV=4, H=2, kda=False, **kw):
    """Arguments of a prefill on the CPU, and its state."""
    ssm = torch.zeros(N + 1, HV, 128, 128)
    lens = [T - N + 1] + [1] * (N - 1)
    d = dict(ssm=ssm, mixed=torch.zeros(T, 2 * H * 128 + HV * 128, dtype=torch.bfloat16),
             a=torch.zeros(T, HV, 128, dtype=torch.bfloat16) if kda else torch.zeros(T, HV, dtype=torch.bfloat16),
             b=torch.zeros(T, HV, dtype=torch.bfloat16), A_log=torch.zeros(HV), dt_bias=torch.zeros(HV * 128 if kda else HV),
             idx=torch.arange(1, N + 1, dtype=torch.int32),
             loc=torch.tensor([sum(lens[:n]) for n in range(N + 1)], dtype=torch.int32),
             out=torch.zeros(T, HV, 128, dtype=torch.bfloat16), has_state=torch.ones(N, dtype=torch.bool))
    d.update(kw)
    return LeapQuantState(ssm, H, kda=kda), d


BAD = [dict(), dict(mixed=torch.zeros(5, 1032, dtype=torch.bfloat16)[:, 1:1025]), dict(a=torch.zeros(5, 4)), dict(b=torch.zeros(4, 4)),
       dict(A_log=torch.zeros(3)), dict(dt_bias=torch.zeros(5)), dict(loc=torch.zeros(2, dtype=torch.int32)),
       dict(out=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), dict(ssm=torch.zeros(3, 2, 128, 128)),
       dict(idx=torch.ones(2)), dict(has_state=torch.ones(3, dtype=torch.bool))]


@pytest.mark.parametrize("kda", [False, True])
@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(b) or "host tensors")
def test_a_refused_prefill_leaves_the_checkpoints(monkeypatch, kda, bad):
    """The checkpoints of has_state slots are turned into fp32 states only when nothing refuses the call any more."""
    st, d = call(kda=kda)
    d.update(bad)
    for name in ("dequantize", "quantize", "flush"):
        monkeypatch.setattr(st, name, lambda *a, name=name: pytest.fail("%s before the arguments were checked" % name))
    with pytest.raises((ValueError, TypeError)):
        st.prefill(**d)


def test_a_failed_workspace_leaves_the_checkpoints(monkeypatch):
    """The chunked form's workspace is taken before the checkpoints are touched."""
    st, d = call(T=40)
    monkeypatch.setattr(st, "dequantize", lambda *a: pytest.fail("dequantize before the workspace"))
    monkeypatch.setattr(seq, "_on", lambda *a, **k: None)            # as if all were on the GPU

    def empty(*a, **k):
        raise MemoryError
    monkeypatch.setattr(seq.torch, "empty", empty)
    monkeypatch.setattr(seq._lib.seq_lib(), "lq_delta_workspace", lambda *a: 1 << 20)
    with pytest.raises(MemoryError):
        st.prefill(**d)


@pytest.mark.parametrize("N,T,longest,chunks", [
    (64, 512, None, True), (64, 512, 449, True), (64, 512, 8, False), (64, 512, 9, True), (1, 8, None, False), (1, 9, None, True),
    (3, 8, None, False), (256, 256, None, True), (256, 256, 1, False), (0, 0, None, False)])
def test_prefill_goes_by_the_longest_sequence(monkeypatch, N, T, longest, chunks):
    """Token by token takes as long as the longest sequence: 63 single tokens beside a prompt of 449 go in chunks."""
    st, d = call(N=N, T=T, HV=2, H=1, loc=torch.zeros(N + 1, dtype=torch.int32)) if N else call(N=1, T=0)
    if not N:
        d.update(idx=d["idx"][:0], loc=d["loc"][:1], has_state=d["has_state"][:0])
    took = []
    monkeypatch.setattr(seq, "_rule", lambda *a: took.append(a[14]))
    for name in ("dequantize", "quantize"):
        monkeypatch.setattr(st, name, lambda *a: None)
    st.prefill(**d, longest=longest)
    assert took == [chunks]
    st.kda = True
    st.prefill(**d, longest=longest)
    assert took == [chunks, False]
    with pytest.raises(TypeError, match="longest"):
        st.prefill(**d, longest=torch.tensor(3))


def test_check_entry_answers_as_the_calls():
    """lq_delta_check without a launch: the grids' limits and the forms that each call takes."""
    import ctypes
    from tests.test_seq_boundary import _delta, _seqs
    from leapquant_amd import _lib
    check = _lib.seq_lib().lq_delta_check
    ask = lambda d, s, chunks: check(ctypes.byref(d), ctypes.byref(s), chunks)          # noqa: E731
    ok, s = _delta(), _seqs(N=2, T=100)
    assert ask(ok, s, 0) == ask(ok, s, 1) == 0 and ask(ok, s, 2) == -1
    kda = _delta(kda=1, a_ld=512, glb=-5.0)
    assert ask(kda, s, 0) == 0 and ask(kda, s, 1) == -1
    assert ask(_delta(mixed_ld=(1 << 24) + 8), s, 1) == -1 and ask(_delta(mixed_ld=(1 << 24) + 8), s, 0) == 0
    many = _seqs(N=1 << 30, T=100)
    assert ask(ok, many, 0) == ask(ok, many, 1) == -1
    assert check(None, ctypes.byref(s), 0) == check(ctypes.byref(ok), None, 1) == -1
