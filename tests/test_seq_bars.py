"""The bars of tests/seq_bars.py against planted roundings (CPU): what the kernels leave out passes, a part less does not."""
import pytest

from tests import seq_bars as Bars, seq_ref as R


@pytest.mark.parametrize("K,V", [(128, 128), (64, 64)])
def test_bars(K, V):
    HV, H = 4, 2
    d = R.delta_inputs(60, [150], HV, H, K, V)
    d["src"][:] = 0
    want, _ = R.delta_ref(d, H)
    args = [R.f64(d[k]) for k in ("mixed", "a", "b", "A_log")] + [R.f64(d["dt_bias"])[:, 0], H, HV, K, V]
    terms = Bars.terms(d, H)
    run = lambda **kw: Bars.bf16(Bars.chunked(*args, **kw))              # noqa: E731
    assert Bars.off(run(), want, Bars.ONCE, terms) == 0                         # the chunked form is the definition
    assert Bars.off(run(w_parts=2, s_parts=2), want, Bars.CHUNKS, terms) == 0
    for lost in (dict(w_parts=1, s_parts=2), dict(w_parts=2, s_parts=1)):
        assert Bars.off(run(**lost), want, Bars.CHUNKS, terms) > 100, lost
