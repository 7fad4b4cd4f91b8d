"""The sequence operators (leapquant_amd/seq.py) on the GPU against their definitions in 64 bits (tests/seq_ref.py).

Bars, from what is rounded where:
  * a bf16 output of fp32 arithmetic (conv, norms, delta_steps): half a unit in the last place is 2^-9 of the value; 2^-8 lets
    an fp32 error move a value over a rounding edge.  Plus 1e-5 of the row's scale where terms cancel.
  * fp32 states of delta_steps: a few roundings of 2^-24 a token, 24 tokens: 1e-5 of the norm.
  * delta_prefill's states: operands of the matrix cores carried in two or three bf16 parts, 2^-17 of each element at most, four
    products in a chain, errors of random sign: 1e-5 of the norm.  Its outputs besides their own rounding take the
    attention weights in bf16 (2^-9 each, random signs): 4e-3 of the norm, and 2^-6 of the larger of value and rms."""
import numpy as np
import pytest
import torch

from tests import seq_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DIMS = [(128, 128), (64, 128), (64, 64)]


@pytest.fixture(scope="module")
def seq():
    from leapquant_amd import seq
    return seq


def gpu(d):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def close_bf16(got, want, scale=None):
    got = R.f64(got)
    scale = np.sqrt((want ** 2).mean(-1, keepdims=True)) if scale is None else scale
    bad = np.abs(got - want) > 2.0 ** -8 * np.abs(want) + 1e-5 * scale
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()))


def rel(got, want):
    n = np.linalg.norm(want)
    return float(np.linalg.norm(R.f64(got) - want) / n) if n else float(np.abs(R.f64(got)).max(initial=0))


def near_prefill(out, want):
    got = R.f64(out)
    assert rel(out, want) <= 4e-3, rel(out, want)
    rms = np.sqrt((want ** 2).mean())
    assert (np.abs(got - want) <= 2.0 ** -6 * np.maximum(rms, np.abs(want))).all()


def run_delta(fn, d, H, out=None, src="src", **kw):
    T, HV, V = d["mixed"].shape[0], d["S"].shape[1], d["S"].shape[2]
    out = torch.full((T, HV, V), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
    fn(d["S"], d["mixed"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["idx"], d["loc"], out, H,
       src=d[src] if src else None, **kw)
    torch.cuda.synchronize()
    return out


# ---- the gated delta rule -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", [[1], [3, 0, 1], [24, 7, 13]], ids=str)
@pytest.mark.parametrize("K,V", DIMS)
@pytest.mark.parametrize("HV,H", [(2, 2), (4, 2), (8, 2), (6, 2)])
def test_steps(seq, lens, K, V, HV, H):
    d = R.delta_inputs(1, lens, HV, H, K, V)
    want, S = R.delta_ref(d, H)
    g = gpu(d)
    out = run_delta(seq.delta_steps, g, H)
    close_bf16(out, want)
    assert rel(g["S"], S) <= 1e-5
    assert torch.equal(g["S"][:len(lens) + 1].cpu(), d["S"][:len(lens) + 1])      # the slots that were only read


@pytest.mark.parametrize("glb", [0.0, -5.0])
@pytest.mark.parametrize("lens", [[1, 1], [17, 0, 5]], ids=str)
@pytest.mark.parametrize("HV,H", [(2, 2), (4, 2)])
def test_steps_kda(seq, glb, lens, HV, H):
    d = R.delta_inputs(2, lens, HV, H, 128, 128, kda=True, glb=glb)
    want, S = R.delta_ref(d, H, glb=glb)
    g = gpu(d)
    out = run_delta(seq.delta_steps, g, H, kda=True, gate_lower_bound=glb)
    close_bf16(out, want)
    assert rel(g["S"], S) <= 1e-5


LENS = [[1], [31], [32], [33], [64], [200], [1, 2, 0, 63, 65, 17], [128, 31]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("K,V", DIMS)
def test_prefill(seq, lens, K, V):
    d = R.delta_inputs(3, lens, 4, 2, K, V)
    d["src"][::2] = 0                                     # every other sequence starts from zero
    want, S = R.delta_ref(d, 2)
    g = gpu(d)
    out = run_delta(seq.delta_prefill, g, 2)
    near_prefill(out, want)
    for n in range(len(lens)):
        assert rel(g["S"][d["idx"][n]], S[d["idx"][n]]) <= 1e-5, n
    assert torch.equal(g["S"][:len(lens) + 1].cpu(), d["S"][:len(lens) + 1])


@pytest.mark.parametrize("HV,H", [(1, 1), (3, 1), (8, 2), (32, 16)])
def test_prefill_head_layouts(seq, HV, H):
    d = R.delta_inputs(4, [70, 45], HV, H, 128, 128)
    want, S = R.delta_ref(d, H)
    g = gpu(d)
    near_prefill(run_delta(seq.delta_prefill, g, H), want)
    assert rel(g["S"][3:], S[3:]) <= 1e-5


MANY = [0, 70, 31, 1, 96, 64, 33, 2, 45, 32, 5, 130, 20, 17, 63, 65, 3, 40]


@pytest.mark.parametrize("case", ["trained", "equal keys", "no decay", "strong decay", "zero and large"])
@pytest.mark.parametrize("K,V", DIMS)
def test_prefill_of_many_sequences(seq, K, V, case):
    """More heads and sequences than the compute units take 16 rows a time of (the walk with a wave alone for them), at the
    values and gates where the other one is tested too; a padding sequence among them, every third from zero."""
    HV, H, N = 8, 2, len(MANY)
    d = R.delta_inputs(17, MANY, HV, H, K, V, gate={"equal keys": -40.0, "no decay": -40.0, "strong decay": 60.0}.get(case))
    if case == "equal keys":
        d["mixed"][:, H * K:2 * H * K] = d["mixed"][0, H * K:2 * H * K]
        d["b"][:] = 9.0
    if case == "zero and large":
        d["mixed"][100:110] = 0
        d["mixed"][200:204] *= 1e4
    d["src"][::3] = 0
    d["idx"][4] = 0
    want, S = R.delta_ref(d, H)
    g = gpu(d)
    out = run_delta(seq.delta_prefill, g, H)
    at = d["loc"].tolist()
    for n in range(N):
        if n == 4:
            assert not out[at[n]:at[n + 1]].any()
        elif MANY[n]:
            near_prefill(out[at[n]:at[n + 1]], want[at[n]:at[n + 1]])
        if n != 4:
            assert rel(g["S"][N + 1 + n], S[N + 1 + n]) <= 1e-5, n
    assert torch.equal(g["S"][:N + 1].cpu(), d["S"][:N + 1])
    assert torch.equal(g["S"][N + 5].cpu(), d["S"][N + 5])            # the padding sequence's


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
@pytest.mark.parametrize("gate", [-40.0, 4.0, 60.0, 3e4])
def test_gates_at_their_ends(seq, fn, gate):
    """No decay at all, decays that leave nothing after a token, and gates whose sum over a chunk passes any exponent."""
    d = R.delta_inputs(5, [40, 20], 4, 2, 128, 128, gate=gate)
    want, S = R.delta_ref(d, 2)
    g = gpu(d)
    near_prefill(run_delta(getattr(seq, fn), g, 2), want)
    for n in (3, 4):
        assert rel(g["S"][n], S[n]) <= 1e-5


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_equal_keys(seq, fn):
    """One key for all tokens, beta near 1 and no decay: (I + A) is all ones below its diagonal, whose powers grow like
    binomials."""
    d = R.delta_inputs(6, [130], 2, 1, 128, 128, gate=-40.0)
    d["mixed"][:, 128:256] = d["mixed"][0, 128:256]
    d["b"][:] = 9.0
    want, S = R.delta_ref(d, 1)
    g = gpu(d)
    near_prefill(run_delta(getattr(seq, fn), g, 1), want)
    assert rel(g["S"][2], S[2]) <= 1e-5


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_zero_and_large_tokens(seq, fn):
    """Rows of zeros (the norms' epsilon) and of large values."""
    d = R.delta_inputs(7, [50, 50], 4, 2, 128, 128)
    d["mixed"][3:9] = 0
    d["mixed"][60:64] *= 1e4
    want, S = R.delta_ref(d, 2)
    g = gpu(d)
    out = run_delta(getattr(seq, fn), g, 2)
    for lo, hi in ((0, 50), (50, 100)):
        near_prefill(out[lo:hi], want[lo:hi])
    for n in (3, 4):
        assert rel(g["S"][n], S[n]) <= 1e-5


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_in_place_padding_and_foreign_rows(seq, fn):
    """In place (no src), a padding sequence and one past the cache between others, rows no sequence holds, NaN in rows that
    are not a sequence's own and in the states that nothing reads."""
    lens = [37, 5, 40, 3]
    d = R.delta_inputs(8, lens, 4, 2, 128, 128, NS=6)
    d["idx"] = torch.tensor([2, 0, 1, 6], dtype=torch.int32)
    d["mixed"] = torch.cat([d["mixed"], torch.full((9, d["mixed"].shape[1]), float("nan")).to(R.BF16)])
    d["a"], d["b"] = (torch.cat([d[k], torch.full((9, 4), float("nan")).to(R.BF16)]) for k in ("a", "b"))
    d["mixed"][37:42] = float("nan")                      # the padding sequence's tokens
    d["S"][3:] = float("nan")
    want, S = R.delta_ref({**d, "mixed": torch.nan_to_num(d["mixed"]), "S": torch.nan_to_num(d["S"])}, 2, src=None)
    g = gpu(d)
    out = run_delta(getattr(seq, fn), g, 2, src=None)
    assert not out[37:42].any() and not out[82:85].any()  # padding
    assert bool((out[85:] == 7).all())                    # not written
    for lo, hi in ((0, 37), (42, 82)):
        near_prefill(out[lo:hi], want[lo:hi])
    for n in (1, 2):
        assert rel(g["S"][n], S[n]) <= 1e-5
    assert torch.isnan(g["S"][3:]).all() and torch.equal(g["S"][0].cpu(), d["S"][0])


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_nan_stays_in_its_sequence(seq, fn):
    d = R.delta_inputs(9, [20, 44, 9], 4, 2, 128, 128)
    want, S = R.delta_ref(d, 2)
    d["mixed"][30] = float("nan")
    d["a"][31] = float("nan")
    g = gpu(d)
    out = run_delta(getattr(seq, fn), g, 2)
    near_prefill(out[:20], want[:20])
    near_prefill(out[64:], want[64:])
    assert torch.isnan(out[32:64]).all() and torch.isnan(g["S"][5]).any()
    for n in (4, 6):
        assert rel(g["S"][n], S[n]) <= 1e-5


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_strided_inputs_and_parameter_types(seq, fn):
    """Column ranges of one wide projection, a cache of strided slots, int64 indexes, bf16 gate parameters, a scale."""
    HV, H, K, V = 4, 2, 128, 128
    d = R.delta_inputs(10, [33, 50], HV, H, K, V)
    T, C = d["mixed"].shape
    wide = torch.randn(T, C + 64 + 2 * HV).to(R.BF16)
    wide[:, 32:32 + C], wide[:, C + 64:C + 64 + HV], wide[:, C + 64 + HV:] = d["mixed"], d["b"], d["a"]
    d["A_log"], d["dt_bias"] = d["A_log"].to(R.BF16), d["dt_bias"].to(R.BF16)
    want, S = R.delta_ref(d, H, scale=0.2)
    g = gpu(d)
    w = wide.to(DEV)
    pad = torch.zeros(5, HV * V * K + 12, device=DEV)
    cache = pad[:, :HV * V * K].unflatten(1, (HV, V, K))
    cache.copy_(g["S"])
    g.update(S=cache, mixed=w[:, 32:32 + C], b=w[:, C + 64:C + 64 + HV], a=w[:, C + 64 + HV:], idx=g["idx"].long(),
             loc=g["loc"].long())
    near_prefill(run_delta(getattr(seq, fn), g, H, scale=0.2), want)
    assert rel(g["S"][3:], S[3:]) <= 1e-5
    assert not pad[:, HV * V * K:].any()


def test_prefill_continues_a_prefill(seq):
    """A prompt in two calls equals the prompt in one, and its tokens one by one."""
    d = R.delta_inputs(11, [150], 4, 2, 128, 128)
    want, S = R.delta_ref(d, 2)
    g = gpu(d)
    out = torch.empty(150, 4, 128, dtype=torch.bfloat16, device=DEV)
    lo = 0
    for n, fn in ((45, seq.delta_prefill), (1, seq.delta_steps), (64, seq.delta_prefill), (3, seq.delta_steps),
                  (37, seq.delta_prefill)):
        loc = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        fn(g["S"], g["mixed"][lo:lo + n], g["a"][lo:lo + n], g["b"][lo:lo + n], g["A_log"], g["dt_bias"], g["idx"], loc,
           out[lo:lo + n], 2, src=g["src"] if lo == 0 else None)
        lo += n
    near_prefill(out, want)
    assert rel(g["S"][2], S[2]) <= 1e-5


def test_long_prefill(seq):
    d = R.delta_inputs(12, [1500, 700], 2, 1, 128, 128)
    want, S = R.delta_ref(d, 1)
    g = gpu(d)
    near_prefill(run_delta(seq.delta_prefill, g, 1), want)
    assert rel(g["S"][3:], S[3:]) <= 1e-5


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_graph_and_streams(seq, fn):
    """Replays of a captured call equal the eager result, with other work between; a call on a side stream too."""
    d = R.delta_inputs(13, [70, 9, 33], 4, 2, 128, 128)
    g = gpu(d)
    eager = run_delta(getattr(seq, fn), g, 2)
    S = g["S"].clone()
    args = (g["S"], g["mixed"], g["a"], g["b"], g["A_log"], g["dt_bias"], g["idx"], g["loc"])
    out = torch.zeros_like(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        getattr(seq, fn)(*args, out, 2, src=g["src"])
    for _ in range(4):
        g["S"][4:].zero_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(g["S"], S)
        assert torch.equal(run_delta(getattr(seq, fn), g, 2), eager)
    side = torch.cuda.Stream()
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        getattr(seq, fn)(*args, out, 2, src=g["src"])
    side.synchronize()
    assert torch.equal(out, eager)


def test_empty_calls(seq):
    d = gpu(R.delta_inputs(14, [0, 0], 4, 2, 128, 128))
    S = d["S"].clone()
    for fn in (seq.delta_prefill, seq.delta_steps):
        run_delta(fn, d, 2)
        assert torch.equal(d["S"][3:], S[1:3])            # a sequence of no tokens hands its state on
        none = dict(d, idx=d["idx"][:0], src=d["src"][:0], loc=d["loc"][:1])
        run_delta(fn, none, 2)


@pytest.mark.parametrize("fn,first", [("delta_prefill", 1), ("delta_prefill", 100), ("delta_steps", 5)])
def test_rows_before_the_first_sequence(seq, fn, first):
    """Packed rows before loc[0] belong to nobody: not read, not written."""
    d = R.delta_inputs(16, [first, 40, 0, 33], 4, 2, 64, 64)
    for k in ("loc", "src", "idx"):
        d[k] = d[k][1:]
    for k in ("mixed", "a", "b"):
        d[k][:first] = float("nan")
    want, S = R.delta_ref(d, 2)
    g = gpu(d)
    out = torch.full((first + 73, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    getattr(seq, fn)(g["S"], g["mixed"], g["a"], g["b"], g["A_log"], g["dt_bias"], g["idx"], g["loc"], out, 2, src=g["src"])
    torch.cuda.synchronize()
    assert bool((out[:first] == 7).all())
    near_prefill(out[first:], want[first:])
    assert rel(g["S"], S) <= 1e-5


# ---- the conv ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C,bias,silu", [(256, True, True), (1000, False, True), (70, True, False), (33, False, True)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 3, 1], [16, 17, 50, 4]], ids=str)
def test_conv(seq, C, bias, silu, lens):
    g = torch.Generator().manual_seed(20)
    rn = lambda *s: torch.randn(*s, generator=g)                    # noqa: E731
    T, N = sum(lens), len(lens)
    x, w, st = rn(T, C).to(R.BF16), (0.5 * rn(C, 4)).to(R.BF16), rn(2 * N + 2, C, 3).to(R.BF16)
    b = rn(C).to(R.BF16) if bias else None
    loc = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)
    src, idx = torch.arange(1, N + 1, dtype=torch.int32), torch.arange(N + 1, 2 * N + 1, dtype=torch.int32)
    src[0] = -1
    want, state = R.conv(R.f64(x), R.f64(st), R.f64(w), None if b is None else R.f64(b), idx.tolist(), loc.tolist(),
                         src.tolist(), silu)
    s, out = st.to(DEV), torch.empty(T, C, dtype=torch.bfloat16, device=DEV)
    seq.conv_prefill(x.to(DEV), s, w.to(DEV), None if b is None else b.to(DEV), idx.to(DEV), loc.to(DEV), out,
                     src=src.to(DEV), silu=silu)
    torch.cuda.synchronize()
    close_bf16(out, want, scale=1.0)
    assert np.array_equal(R.f64(s), state)


def test_conv_in_place_strided_and_padding(seq):
    """In place, a state whose taps come first, a column range of wider rows, a padding sequence, rows nobody holds."""
    C, lens = 128, [5, 2, 20, 1]
    g = torch.Generator().manual_seed(21)
    wide = torch.randn(40, C + 24, generator=g).to(R.BF16)
    st = torch.randn(4, 3, C, generator=g).to(R.BF16)
    w = torch.randn(C, 4, generator=g).to(R.BF16)
    loc = torch.tensor(np.concatenate([[0], np.cumsum(lens)]))
    idx = torch.tensor([3, 0, 1, 2])
    want, state = R.conv(R.f64(wide[:, 8:8 + C]), R.f64(st).transpose(0, 2, 1), R.f64(w), None, idx.tolist(), loc.tolist())
    s, out = st.to(DEV), torch.full((40, C), 7.0, dtype=torch.bfloat16, device=DEV)
    seq.conv_prefill(wide.to(DEV)[:, 8:8 + C], s.transpose(1, 2), w.to(DEV), None, idx.to(DEV), loc.to(DEV), out)
    torch.cuda.synchronize()
    close_bf16(out[:28], want[:28], scale=1.0)
    assert not out[5:7].any() and bool((out[28:] == 7).all())
    assert np.array_equal(R.f64(s.transpose(1, 2)), state)


def test_conv_of_one_token_equals_the_decode_update(seq):
    from leapquant_amd import kernels as KN
    g = torch.Generator(device=DEV).manual_seed(22)
    N, C = 5, 384
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)      # noqa: E731
    x, w, b, st = rn(N, C), rn(C, 4), rn(C), rn(N + 1, C, 3)
    idx = torch.arange(1, N + 1, dtype=torch.int32, device=DEV)
    s1, s2, o1, o2 = st.clone(), st.clone(), torch.empty_like(x), torch.empty_like(x)
    KN.conv_update(x, s1, w, b, idx, o1)
    seq.conv_prefill(x, s2, w, b, idx, torch.arange(N + 1, dtype=torch.int32, device=DEV), o2)
    torch.cuda.synchronize()
    assert torch.equal(s1, s2)
    a, b = R.f64(o1), R.f64(o2)                           # both round the same sum: at most a unit apart
    assert (np.abs(a - b) <= 2.0 ** -7 * np.abs(a) + 1e-5).all()


@pytest.mark.parametrize("first", [1, 8, 21, 40])
def test_conv_rows_before_the_first_sequence(seq, first):
    """Packed rows before loc[0] belong to nobody: not read, not written."""
    C, lens = 64, [9, 0, 30]
    g = torch.Generator().manual_seed(23)
    T = first + sum(lens)
    x, st, w = (torch.randn(*s, generator=g).to(R.BF16) for s in ((T, C), (7, C, 3), (C, 4)))
    x[:first] = float("nan")
    loc = torch.tensor(first + np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)
    src, idx = torch.tensor([1, 2, 3], dtype=torch.int32), torch.tensor([4, 5, 6], dtype=torch.int32)
    want, state = R.conv(R.f64(x), R.f64(st), R.f64(w), None, idx.tolist(), loc.tolist(), src.tolist())
    s, out = st.to(DEV), torch.full((T, C), 7.0, dtype=torch.bfloat16, device=DEV)
    seq.conv_prefill(x.to(DEV), s, w.to(DEV), None, idx.to(DEV), loc.to(DEV), out, src=src.to(DEV))
    torch.cuda.synchronize()
    assert bool((out[:first] == 7).all())
    close_bf16(out[first:], want[first:], scale=1.0)
    assert np.array_equal(R.f64(s), state)


@pytest.mark.parametrize("N", [64, 65, 300, 4500])
def test_conv_of_many_sequences(seq, N):
    """The search for a run's sequence, in one step, two and three."""
    C, rng = 2, np.random.default_rng(N)
    lens = rng.integers(0, 4, N)
    lens[N // 2] = 100
    g = torch.Generator().manual_seed(24)
    T = int(lens.sum())
    x, st, w = (torch.randn(*s, generator=g).to(R.BF16) for s in ((T, C), (N + 1, C, 3), (C, 4)))
    loc = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)
    idx = torch.tensor(rng.permutation(N) + 1, dtype=torch.int32)
    want, state = R.conv(R.f64(x), R.f64(st), R.f64(w), None, idx.tolist(), loc.tolist())
    s, out = st.to(DEV), torch.empty(T, C, dtype=torch.bfloat16, device=DEV)
    seq.conv_prefill(x.to(DEV), s, w.to(DEV), None, idx.to(DEV), loc.to(DEV), out)
    torch.cuda.synchronize()
    close_bf16(out, want, scale=1.0)
    assert np.array_equal(R.f64(s), state)


def test_conv_large_call_equals_its_sequences(seq):
    """A call of 2^27 elements against each of its sequences in a call of its own (narrower accesses): the same bits."""
    C, lens = 8192, [9000, 1, 0, 5, 7411]
    N, T = len(lens), sum(lens)
    g = torch.Generator(device=DEV).manual_seed(25)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)      # noqa: E731
    assert T * C >= 1 << 27
    x, w, b, st = rn(T, C), rn(C, 4), rn(C), rn(2 * N + 1, C, 3)
    at = np.concatenate([[0], np.cumsum(lens)])
    loc = torch.tensor(at, dtype=torch.int32, device=DEV)
    src = torch.arange(1, N + 1, dtype=torch.int32, device=DEV)
    s1, s2, o1, o2 = st.clone(), st.clone(), torch.empty_like(x), torch.empty_like(x)
    seq.conv_prefill(x, s1, w, b, src + N, loc, o1, src=src)
    for n in range(N):
        own = slice(int(at[n]), int(at[n + 1]))
        seq.conv_prefill(x[own], s2, w, b, src[n:n + 1] + N, loc[n:n + 2] - loc[n], o2[own], src=src[n:n + 1])
    torch.cuda.synchronize()
    assert torch.equal(o1, o2) and torch.equal(s1, s2)


# ---- the norms --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [1, 7, 64, 72, 128, 200, 256, 512, 1000])
@pytest.mark.parametrize("gate,wdt,offset", [("silu", torch.bfloat16, 0.0), ("sigmoid", torch.float32, 1.0)])
def test_gated_norm(seq, D, gate, wdt, offset):
    g = torch.Generator().manual_seed(30)
    rows, HV = 5, 3
    x, z = torch.randn(rows, HV, D, generator=g).to(R.BF16), (3 * torch.randn(rows, 2 * HV * D + 8, generator=g)).to(R.BF16)
    w = torch.randn(D, generator=g).to(wdt)
    x[1, 1] = 0                                           # a row of nothing: the epsilon
    zv = z[:, HV * D:2 * HV * D].unflatten(1, (HV, D))
    s = R.sigmoid(R.f64(zv))
    want = R.rms(R.f64(x), R.f64(w), 1e-5, offset) * (s if gate == "sigmoid" else s * R.f64(zv))
    out = torch.empty(rows, HV, D, dtype=torch.bfloat16, device=DEV)
    zd = z.to(DEV)[:, HV * D:2 * HV * D].unflatten(1, (HV, D))
    seq.gated_norm(x.to(DEV), zd, w.to(DEV), out, eps=1e-5, gate=gate, offset=offset)
    torch.cuda.synchronize()
    close_bf16(out, want, scale=0.1)


@pytest.mark.parametrize("D", [1, 96, 1000, 2048, 2049, 4096, 5000, 8192, 16384, 16383])
@pytest.mark.parametrize("wdt", [torch.bfloat16, torch.float32])
def test_add_norm(seq, D, wdt):
    g = torch.Generator().manual_seed(31)
    x, y = torch.randn(3, D, generator=g).to(R.BF16), torch.randn(3, D, generator=g).to(R.BF16)
    w = torch.randn(D, generator=g).to(wdt)
    r = R.f64(x) + 0.25 * R.f64(y)
    want = R.rms(r, R.f64(w), 1e-6, 1.0)
    xd, out = x.to(DEV), torch.empty(3, D, dtype=torch.bfloat16, device=DEV)
    seq.add_norm(xd, y.to(DEV), w.to(DEV), xd, out, scale=0.25, offset=1.0)         # in place
    torch.cuda.synchronize()
    close_bf16(xd, r, scale=0.1)
    close_bf16(out, want, scale=0.1)


def test_norms_extremes(seq):
    """Gates and values at the ends of their range: no overflow on the way, NaN and infinity only where they belong."""
    x = torch.tensor([[1e18, -1e18] * 32, [1e-20] * 64, [float("nan")] + [1.0] * 63], dtype=R.BF16)
    z = torch.tensor([[-300.0, 300.0] * 32] * 3, dtype=R.BF16)
    w = torch.ones(64)
    out = torch.empty_like(x, device=DEV)
    seq.gated_norm(x.to(DEV), z.to(DEV), w.to(DEV), out)
    torch.cuda.synchronize()
    got = R.f64(out)
    assert np.array_equal(got[0, ::2], np.zeros(32)) and np.allclose(got[0, 1::2], -300.0, rtol=2 ** -8)
    assert np.isfinite(got[1]).all() and np.isnan(got[2]).all()


def test_norm_graph(seq):
    x, y = (torch.randn(37, 2048, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(2048, device=DEV)
    r, o, r2, o2 = (torch.empty_like(x) for _ in range(4))
    seq.add_norm(x, y, w, r, o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seq.add_norm(x, y, w, r2, o2)
        seq.gated_norm(o2, y, w, o2)
    seq.gated_norm(o, y, w, o)
    for _ in range(3):
        r2.zero_(), o2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r, r2) and torch.equal(o, o2)


@pytest.mark.parametrize("op", ["gated", "add"])
def test_norm_large_call_equals_its_parts(seq, op):
    """A call of more bytes than the caches hold against the same rows in smaller calls: the same bits."""
    rows, D = 23000, 2048
    g = torch.Generator(device=DEV).manual_seed(39)
    x, y = (torch.randn(rows, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(D, generator=g, device=DEV)
    assert 3 * x.numel() * 2 > 256 << 20
    a, b = ([torch.empty_like(x) for _ in range(2)] for _ in range(2))

    def run(to, part):
        if op == "gated":
            seq.gated_norm(x[part], y[part], w, to[0][part])
        else:
            seq.add_norm(x[part], y[part], w, to[0][part], to[1][part], scale=0.5)

    run(a, slice(None))
    for lo in range(0, rows, 6000):
        run(b, slice(lo, lo + 6000))
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and (op == "gated" or torch.equal(a[1], b[1]))


def test_direct_and_checked_calls_agree(seq, monkeypatch):
    """Arguments as the kernels read them go straight to the library; the same call through the Python checks (64-bit indexes,
    half-precision gates' copies) leaves the same bits."""
    d = R.delta_inputs(43, [40, 3], 4, 2, 128, 128)
    d["A_log"] = d["A_log"].half().float()
    g = gpu(d)
    x, w = g["mixed"], torch.randn(g["mixed"].shape[1], 4, device=DEV).to(torch.bfloat16)
    taps = torch.randn(5, x.shape[1], 3, device=DEV).to(torch.bfloat16)
    nw = torch.nn.Parameter(torch.randn(x.shape[1], device=DEV))

    def run(**kw):
        e = dict(g, **kw)
        out = [run_delta(fn, e, 2) for fn in (seq.delta_prefill, seq.delta_steps)] + [e["S"].clone()]
        y, t = torch.empty_like(x), taps.clone()
        seq.conv_prefill(x, t, w, None, e["idx"], e["loc"], y, src=e["src"])
        n, r, o = (torch.empty_like(x) for _ in range(3))
        seq.gated_norm(y, x, nw, n)
        seq.add_norm(x, n, nw, r, o, scale=0.5)
        torch.cuda.synchronize()
        return out + [y, t, n, r, o]

    checked = run(idx=g["idx"].long(), loc=g["loc"].long(), A_log=g["A_log"].half())
    with monkeypatch.context() as m:
        for name in ("_delta", "_norm", "_batch"):
            m.setattr(seq, name, None)                    # not to be reached
        direct = run()
    assert all(torch.equal(a, b) for a, b in zip(checked, direct))


# ---- together -----------------------------------------------------------------------------------------------------------
def test_graph_of_conv_and_norms(seq):
    """Replays of the conv and both norms equal the eager results, with other work between."""
    g = torch.Generator(device=DEV).manual_seed(40)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)      # noqa: E731
    x, st, w, nw = rn(77, 256), rn(7, 256, 3), rn(256, 4), rn(256)
    loc = torch.tensor([0, 40, 41, 77], dtype=torch.int32, device=DEV)
    src = torch.arange(1, 4, dtype=torch.int32, device=DEV)
    y, n, r, o = (torch.zeros_like(x) for _ in range(4))

    def run():
        seq.conv_prefill(x, st, w, None, src + 3, loc, y, src=src)
        seq.gated_norm(y, x, nw, n)
        seq.add_norm(x, n, nw, r, o, scale=0.5)

    run()
    torch.cuda.synchronize()
    want = [t.clone() for t in (st, y, n, r, o)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(4):
        for t in (y, n, r, o, st[4:]):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((st, y, n, r, o), want))
        torch.matmul(x, w)
        torch.cuda.synchronize()


def _far(rows, cols, ld):
    """bf16 [rows, cols] whose last rows lie past 2^32 elements."""
    return torch.empty((rows - 1) * ld + cols, dtype=torch.bfloat16, device=DEV).as_strided((rows, cols), (ld, 1))


@pytest.mark.parametrize("fn", ["delta_prefill", "delta_steps"])
def test_delta_offsets_past_32_bits(seq, fn):
    """Slots past 2^31 floats of the state cache and tokens past 2^32 elements: the bits of the same call on small tensors."""
    d = R.delta_inputs(41, [40, 30], 2, 1, 128, 128)
    g = gpu(d)
    want = run_delta(getattr(seq, fn), g, 1)
    NS = (1 << 31) // (2 * 128 * 128) + 8
    S = torch.empty(NS, 2, 128, 128, device=DEV)
    far = [NS - 4, NS - 3, NS - 2, NS - 1]
    S[far[0]], S[far[1]] = d["S"][1].to(DEV), d["S"][2].to(DEV)
    mixed = _far(70, d["mixed"].shape[1], 1 << 24 if fn == "delta_prefill" else 1 << 26)
    mixed.copy_(g["mixed"])
    out = torch.zeros_like(want)
    getattr(seq, fn)(S, mixed, g["a"], g["b"], g["A_log"], g["dt_bias"], torch.tensor(far[2:], device=DEV), g["loc"], out, 1,
                     src=torch.tensor(far[:2], device=DEV))
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(S[far[2]], g["S"][3]) and torch.equal(S[far[3]], g["S"][4])


def test_conv_and_norm_offsets_past_32_bits(seq):
    g = torch.Generator(device=DEV).manual_seed(42)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)      # noqa: E731
    T, C, ld = 70, 64, 1 << 26
    x, w, st, nw = rn(T, C), rn(C, 4), rn(3, C, 3), rn(C)
    far = _far(T, C, ld)
    far.copy_(x)
    loc = torch.tensor([0, 60, T], dtype=torch.int32, device=DEV)
    idx = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    s1, s2, a, b = st.clone(), st.clone(), torch.empty_like(x), torch.empty_like(x)
    seq.conv_prefill(x, s1, w, None, idx, loc, a)
    seq.conv_prefill(far, s2, w, None, idx, loc, b)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(s1, s2)
    seq.gated_norm(x, x, nw, a)
    seq.gated_norm(far, x, nw, far)                       # in place
    torch.cuda.synchronize()
    assert torch.equal(far, a)
