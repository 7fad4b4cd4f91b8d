"""The delta rule's kernels as calls of real batches pick them (MI355X): all rows of a head in a lane group, states past the shared
cache, more sequences than a search step and the length sort take; and the bars of tests/seq_bars.py, by token and head."""
import numpy as np
import pytest
import torch

from tests import seq_bars as Bars, seq_ref as R
from tests.test_gpu_seq import DEV, DIMS, gpu, run_delta

pytestmark = pytest.mark.gpu
CUS = 256


@pytest.fixture(scope="module")
def seq():
    from leapquant_amd import seq
    return seq


def check(d, H, out, S, more, bar, glb=0.0, scale=None, by_terms=True):
    """Outputs and states against the definition, a padding sequence's, and the slots that no sequence ends in."""
    want, ref = R.delta_ref(d, H, glb=glb, scale=scale)
    terms = Bars.terms(d, H, glb, scale) if by_terms else None
    NS, at = d["S"].shape[0], d["loc"].tolist()
    for n, slot in enumerate(d["idx"].tolist()):
        rows = slice(at[n], at[n + 1])
        if 0 < slot < NS:
            Bars.near(out[rows], want[rows], more, terms[rows] if by_terms else None)
            Bars.states_near(S[slot], ref[slot], bar)
        else:
            assert not out[rows].any(), n
    ended = set(d["idx"].tolist())
    for s in range(NS):
        if s not in ended or s == 0:
            assert torch.equal(S[s].cpu(), d["S"][s]), s


# ---- token by token: V / 32 rows a lane where T > N and N HV V / 32 > 2 CUs ----------------------------------------------------
FORMS = pytest.mark.parametrize("kda,glb,K,V,HV,H", [
    (False, 0.0, 128, 128, 8, 4), (False, 0.0, 64, 128, 8, 2), (False, 0.0, 64, 64, 16, 16), (True, 0.0, 128, 128, 8, 8),
    (True, -5.0, 128, 128, 8, 4)])


def batch(kda, glb, K, V, HV, H, gate=None):
    """Ragged, a sequence of nothing, single tokens, a padding sequence; every fourth from zero."""
    lens = [9, 0, 1, 5, 2, 17, 3, 1, 8, 4] * 4
    N = len(lens)
    assert sum(lens) > N and N * HV * (V // 32) > 2 * CUS
    d = R.delta_inputs(61, lens, HV, H, K, V, kda=kda, glb=glb, gate=gate)
    d["src"][::4] = 0
    d["idx"][7] = 0
    return d, dict(kda=True, gate_lower_bound=glb) if kda else {}


@FORMS
def test_steps_of_a_batch(seq, kda, glb, K, V, HV, H):
    d, kw = batch(kda, glb, K, V, HV, H)
    g = gpu(d)
    out = run_delta(seq.delta_steps, g, H, **kw)
    check(d, H, out, g["S"], Bars.ONCE, 1e-5, glb=glb, by_terms=False)


@FORMS
@pytest.mark.parametrize("gate", [None, 6.0], ids=["trained", "strong decay"])
def test_steps_of_a_batch_equal_its_sequences(seq, kda, glb, K, V, HV, H, gate):
    """Each sequence in a call of its own has one row a lane: the same sums in the same order, the same bits.  The strong decay
    takes GDN's factor through its rescaling."""
    d, kw = batch(kda, glb, K, V, HV, H, gate)
    g = gpu(d)
    S, at = g["S"].clone(), d["loc"].tolist()
    out = run_delta(seq.delta_steps, g, H, **kw)
    for n in range(len(at) - 1):
        t, m = slice(at[n], at[n + 1]), slice(n, n + 1)
        own = torch.empty_like(out[t])
        seq.delta_steps(S, g["mixed"][t], g["a"][t], g["b"][t], g["A_log"], g["dt_bias"], g["idx"][m], g["loc"][n:n + 2] - at[n], own,
                        H, src=g["src"][m], **kw)
        assert torch.equal(own, out[t]), n
    assert torch.equal(S, g["S"])


@pytest.mark.parametrize("kda,K,V,HV", [(False, 128, 128, 32), (True, 128, 128, 32), (False, 64, 64, 64)])
@pytest.mark.parametrize("lens,parts", [([1], 4), ([3, 1, 2], 4)], ids=["one row a lane", "all rows"])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_past_the_shared_cache(seq, kda, K, V, HV, lens, parts, in_place):
    """More than 256 MiB of states in a call against the same sequences in smaller calls of the same form: the same bits."""
    H, size = HV, 4 * HV * V * K
    N = -(-(300 << 20) // size)
    N += -N % (3 * parts)
    assert N * size > 256 << 20 and N // parts * size <= 256 << 20 and N // parts * HV * (V // 32) > 2 * CUS
    lens = lens * (N // len(lens))
    at = np.concatenate([[0], np.cumsum(lens)])
    T, KA = int(at[-1]), K if kda else 1
    g = torch.Generator(device=DEV).manual_seed(62)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)             # noqa: E731
    mixed, b, a = rn(T, 2 * H * K + HV * V).bfloat16(), rn(T, HV).bfloat16(), rn(T, HV, KA).bfloat16()
    a = a if kda else a[..., 0]
    A_log, dt = 0.5 * rn(HV), rn(HV * KA) - 4
    S1 = 0.1 * rn((1 if in_place else 2) * N + 1, HV, V, K)
    S2 = S1.clone()
    loc = torch.tensor(at, dtype=torch.int32, device=DEV)
    src = torch.arange(1, N + 1, dtype=torch.int32, device=DEV)
    idx = src if in_place else src + N
    o1, o2 = (torch.zeros(T, HV, V, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def run(S, out, lo, hi):
        t = slice(int(at[lo]), int(at[hi]))
        seq.delta_steps(S, mixed[t], a[t], b[t], A_log, dt, idx[lo:hi], loc[lo:hi + 1] - loc[lo], out[t], H,
                        src=None if in_place else src[lo:hi], kda=kda)

    run(S1, o1, 0, N)
    for i in range(parts):
        run(S2, o2, i * N // parts, (i + 1) * N // parts)
    torch.cuda.synchronize()
    assert torch.equal(o1, o2) and torch.equal(S1, S2)
    assert bool(o1.any())


EDGES = {"no decay": dict(gate=-40.0), "strong": dict(gate=4.0), "nothing left": dict(gate=60.0), "past any exponent": dict(gate=3e4),
         "trained": {}, "equal keys": dict(gate=-40.0), "zero and large": {}, "a scale": {}}


def edge(name, lens, HV, H, K=128, V=128, seed=63):
    d = R.delta_inputs(seed, lens, HV, H, K, V, **EDGES[name])
    if name == "equal keys":
        d["mixed"][:, H * K:2 * H * K] = d["mixed"][0, H * K:2 * H * K]
        d["b"][:] = 9.0
    if name == "zero and large":
        d["mixed"][3:9] = 0
        d["mixed"][30:34] *= 1e4
    return d


@pytest.mark.parametrize("case", EDGES)
@pytest.mark.parametrize("N", [2, 40], ids=["one row a lane", "all rows"])
def test_steps_at_the_edges(seq, case, N):
    """The steps at their own accuracy, one rounding of fp32 arithmetic, where other tests hold them to the chunks' looser bar."""
    lens = [40, 20] if N == 2 else [40, 20] + [2] * 38
    d = edge(case, lens, 8, 4)
    g = gpu(d)
    scale = 0.2 if case == "a scale" else None
    check(d, 4, run_delta(seq.delta_steps, g, 4, scale=scale), g["S"], Bars.ONCE, 1e-5, scale=scale)


# ---- chunks -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("N", [3, 24], ids=["eight waves", "one wave"])
@pytest.mark.parametrize("K,V", DIMS)
@pytest.mark.parametrize("case", ["trained", "no decay", "strong", "nothing left", "past any exponent"])
def test_prefill_by_token_and_head(seq, case, K, V, N):
    """Every token and head by the two-part bar, heads of small outputs beside heads of large ones."""
    HV, H = 8, 4
    lens = [70, 33, 129] if N == 3 else [70, 33, 64, 5] * 6
    assert (N * HV * (V // 16) <= 2 * CUS) == (N == 3)
    d = edge(case, lens, HV, H, K, V, seed=64)
    v = d["mixed"][:, 2 * H * K:].unflatten(1, (HV, V))
    v *= torch.tensor([1.0, 2.0 ** -10, 1.0, 2.0 ** 7] * 2)[:, None]     # values by head: states and outputs scale with them
    d["src"][:] = 0
    g = gpu(d)
    check(d, H, run_delta(seq.delta_prefill, g, H), g["S"], Bars.CHUNKS, Bars.STATE)


@pytest.mark.parametrize("N,HV,H,K,V", [(64, 1, 1, 64, 64), (65, 1, 1, 64, 64), (100, 1, 1, 64, 64), (128, 1, 1, 64, 64),
                                        (64, 2, 1, 128, 128), (65, 2, 1, 64, 128), (256, 2, 1, 64, 64), (257, 2, 2, 64, 64), (300, 2, 1, 128, 128)])
def test_prefill_of_more_sequences_than_a_step_of_the_search(seq, N, HV, H, K, V):
    """Up to 128 sequences of one head in the walk of eight waves, more in the other; past 256 they are not sorted by length."""
    rng = np.random.default_rng(N)
    lens = rng.choice([0, 1, 2, 5, 17, 31, 32, 33, 40], N).tolist()
    lens[N // 2], lens[-1] = 100, 0
    d = R.delta_inputs(65, lens, HV, H, K, V)
    d["src"][::3] = -1
    d["idx"] = torch.tensor(rng.permutation(N) + N + 1, dtype=torch.int32)
    d["idx"][5] = 2 * N + 1                                              # past the cache: a padding sequence
    g = gpu(d)
    check(d, H, run_delta(seq.delta_prefill, g, H), g["S"], Bars.CHUNKS, Bars.STATE)
