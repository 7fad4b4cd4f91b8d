"""`LeapQuantState.prefill` on the GPU around the sequence operators: calls that are refused leave every slot's bits."""
import pytest
import torch

from tests import seq_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def layer(lens, HV=4, H=2, kda=False, seed=50):
    """A state whose slots 1 .. N hold checkpoints, and the arguments of a prefill that goes on from all of them."""
    from leapquant_amd.state import LeapQuantState
    N = len(lens)
    d = R.delta_inputs(seed, lens, HV, H, 128, 128, kda=kda, NS=N + 1)
    ssm = d["S"].to(DEV)
    st = LeapQuantState(ssm, H, kda=kda)
    idx = torch.arange(1, N + 1, dtype=torch.int32, device=DEV)
    st.quantize(ssm, idx)
    args = {k: d[k].to(DEV) for k in ("mixed", "a", "b", "A_log", "loc")}
    args.update(ssm=ssm, idx=idx, dt_bias=d["dt_bias"].reshape(-1).to(DEV), has_state=torch.ones(N, dtype=torch.bool, device=DEV),
                out=torch.zeros(sum(lens), HV, 128, dtype=torch.bfloat16, device=DEV))
    return st, args


@pytest.mark.parametrize("kda", [False, True])
@pytest.mark.parametrize("lens", [[3, 2], [70, 33]], ids=str)
def test_refused_calls_leave_every_slot(kda, lens):
    T, H = sum(lens), 4 if kda else 2
    st, args = layer(lens, H=H, kda=kda)
    bits, counts = args["ssm"].clone(), st.hcnt.clone()
    wide = torch.zeros(T, args["mixed"].shape[1] + 8, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(mixed=wide[:, 1:-7]), dict(out=args["out"][:, :, :64]), dict(A_log=args["A_log"][:3]), dict(loc=args["loc"][:2]),
                dict(a=args["a"].float()), dict(b=args["b"][:1]), dict(dt_bias=args["dt_bias"].cpu()), dict(idx=args["idx"].float())):
        with pytest.raises((ValueError, TypeError)):
            st.prefill(**{**args, **bad})
        torch.cuda.synchronize()
        assert torch.equal(args["ssm"].view(torch.int32), bits.view(torch.int32)) and torch.equal(st.hcnt, counts), list(bad)
    st.prefill(**args)                                               # and the call itself still runs
    torch.cuda.synchronize()
    assert torch.isfinite(args["out"].float()).all() and not torch.equal(args["ssm"].view(torch.int32), bits.view(torch.int32))


def test_no_memory_for_the_workspace_leaves_every_slot():
    """The allocator is held to what it has, in segments without room: the workspace of 4096 tokens (33 MB) cannot be had."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    st, args = layer([4000, 96], HV=32, H=16)
    bits = args["ssm"].clone()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / torch.cuda.get_device_properties(0).total_memory)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            st.prefill(**args)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    torch.cuda.synchronize()
    assert torch.equal(args["ssm"].view(torch.int32), bits.view(torch.int32))
