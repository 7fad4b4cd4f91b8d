"""CPU tests of liblq_attn's boundary: it exports what include/lq_attn.h declares, its entry points refuse bad arguments before any
launch, and the Python operators refuse what the kernels do not take.  No kernel is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from tests import attn_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from leapquant_amd import _lib
    if not os.path.exists(_lib.ATTN_LIB_PATH):
        from leapquant_amd import build
        build.build()
    return _lib.attn_lib()


def test_header_binding_and_library_agree(lib):
    from leapquant_amd import _lib
    src = open(os.path.join(ROOT, "include", "lq_attn.h")).read()
    names = set(re.findall(r"^(?:int|long long)\s+(lq_\w+)\s*\(", src, flags=re.M))
    assert names == set(_lib.ATTN_SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.ATTN_LIB_PATH], capture_output=True, text=True, check=True)
    assert names <= {ln.split()[-1] for ln in out.stdout.splitlines() if ln.strip()}


def test_structures_as_the_header_has_them(tmp_path):
    """Sizes and the last fields' places, from a C compiler."""
    from leapquant_amd import _lib
    structs = dict(lq_pages=(_lib.LqPages, "int8"), lq_batch=(_lib.LqBatch, "T"), lq_rows=(_lib.LqRows, "hd"), lq_rope=(_lib.LqRope, "offset"),
                   lq_attention=(_lib.LqAttention, "scale"))
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s/include/lq_attn.h"\nint main(void) {\n' % ROOT + "".join(
        '  printf("%%zu %%zu\\n", sizeof(%s), offsetof(%s, %s));\n' % (n, n, f) for n, (_, f) in structs.items()) + "  return 0;\n}\n")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    want = [v for t, f in structs.values() for v in (ctypes.sizeof(t), getattr(t, f).offset)]
    assert [int(v) for v in out] == want


def test_importable_under_the_reference_name():
    import leapquant.attn
    import leapquant_amd.attn
    assert leapquant.attn is leapquant_amd.attn


def test_files_of_another_version_are_refused(monkeypatch):
    from leapquant_amd import _lib
    _lib.attn_call()
    for name, value in (("_ATTN_LIB", [None]), ("_ATTN_CALL", [None]), ("ATTN_ABI_VERSION", 10 ** 6)):
        monkeypatch.setattr(_lib, name, value)
    with pytest.raises(RuntimeError, match="rebuild"):
        _lib.attn_lib()
    monkeypatch.setattr(_lib, "attn_lib", lambda: None)
    with pytest.raises(RuntimeError, match="rebuild"):
        _lib.attn_call()


# ---- the C entries ---------------------------------------------------------------------------------------------------------
def _pages(**kw):
    from leapquant_amd import _lib
    d = dict(k=16, v=16, k_scale=None, v_scale=None, page_ld=16 * 2 * 128, row_ld=2 * 128, head_ld=128, s_page_ld=0, s_row_ld=0,
             s_head_ld=0, NP=3, page=16, HK=2, D=128, int8=0)
    d.update(kw)
    return _lib.LqPages(**d)


def _batch(**kw):
    from leapquant_amd import _lib
    return _lib.LqBatch(**{**dict(loc=16, lens=16, table=16, table_ld=4, width=4, N=0, T=0), **kw})


def _rows(p=16, ld=512, hd=128):
    from leapquant_amd import _lib
    return _lib.LqRows(p, ld, hd)


def _attention(**kw):
    from leapquant_amd import _lib
    return _lib.LqAttention(**{**dict(q=_rows(), gate=_rows(None, 0, 0), out=_rows(), HQ=4, window=0, scale=0.1), **kw})


def _rope(**kw):
    from leapquant_amd import _lib
    d = dict(q=_rows(), k=_rows(ld=256), v=_rows(ld=256), out=_rows(), q_weight=16, k_weight=16, inv_freq=16, HQ=4, rot=128, weight_bf16=0,
             freq64=0, interleaved=0, eps=1e-6, offset=0.0)
    d.update(kw)
    return _lib.LqRope(**d)


def _call(lib, a=None, r=None, p=None, b=None, longest=0):
    ref = lambda x: ctypes.byref(x) if x is not None else None      # noqa: E731
    p, b = p if p is not None else _pages(), b if b is not None else _batch()
    if r is not None:
        return lib.lq_rope_norm(ref(r), ref(p), ref(b), None)
    rc = lib.lq_attend(ref(a), ref(p), ref(b), longest, None, 0, None)
    assert min(lib.lq_attend_workspace(ref(a), ref(p), ref(b), longest), 0) == rc
    return rc


def test_entries_take_empty_batches(lib):
    assert _call(lib, a=_attention()) == 0 and _call(lib, r=_rope()) == 0
    assert _call(lib, a=_attention(q=_rows(None)), b=_batch(N=2)) == 0 and _call(lib, r=_rope(q=_rows(None)), b=_batch(N=2)) == 0
    int8 = _pages(int8=1, k_scale=16, v_scale=16, s_page_ld=32, s_row_ld=2, s_head_ld=1)
    assert _call(lib, a=_attention(), p=int8) == 0 and _call(lib, r=_rope(), p=int8) == 0


BAD_PAGES = [dict(k=None), dict(v=None), dict(k=8), dict(v=24), dict(NP=0), dict(page=0), dict(page=8), dict(page=17), dict(HK=0), dict(D=96),
             dict(D=32), dict(D=512), dict(int8=2), dict(row_ld=260), dict(head_ld=12), dict(page_ld=-16), dict(row_ld=-16), dict(head_ld=-8),
             dict(page_ld=4), dict(row_ld=1 << 26, page=32), dict(row_ld=1 << 40), dict(head_ld=1 << 29), dict(int8=1), dict(int8=1, k_scale=16),
             dict(int8=1, k_scale=16, v_scale=16, row_ld=264), dict(int8=1, k_scale=16, v_scale=16, s_row_ld=-1),
             dict(int8=1, k_scale=16, v_scale=16, s_row_ld=1 << 30)]
BAD_BATCH = [dict(N=-1), dict(T=-1), dict(width=-1), dict(N=1, loc=None), dict(N=1, lens=None), dict(N=1, table=None),
             dict(N=2, table_ld=-1), dict(width=1 << 27)]


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_BATCH, ids=str)
def test_entries_refuse_caches_and_batches(lib, bad):
    batch = bad in BAD_BATCH
    p, b = _pages(**({} if batch else bad)), _batch(**(bad if batch else {}))
    assert _call(lib, a=_attention(), p=p, b=b) == -1
    assert _call(lib, r=_rope(), p=p, b=b) == -1


def test_entries_refuse_nothing_at_all(lib):
    a, r, p, b = (ctypes.byref(x) for x in (_attention(), _rope(), _pages(), _batch()))
    for args in ((None, p, b), (a, None, b), (a, p, None)):
        assert lib.lq_attend(*args, 0, None, 0, None) == -1 and lib.lq_attend_workspace(*args, 0) == -1
    for args in ((None, p, b), (r, None, b), (r, p, None)):
        assert lib.lq_rope_norm(*args, None) == -1
    # pages so large that a place does not divide exactly
    assert _call(lib, a=_attention(), p=_pages(page=1 << 20, page_ld=1 << 28), b=_batch(width=2)) == -1


FULL = dict(N=1, T=5)
BAD_ATTENTION = [dict(HQ=0), dict(HQ=3), dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                 dict(q=_rows), dict(out=_rows), dict(q=(8,)), dict(q=(16, 516)), dict(q=(16, 512, 132)), dict(out=(24,)),
                 dict(out=(16, 500, 128)), dict(out=(16, 64, 128)), dict(out=(16, 0, 128)), dict(out=(16, 128, 128)), dict(out=(16, 512, 64)),
                 dict(gate=(8,)), dict(gate=(16, 4, 128))]


@pytest.mark.parametrize("bad", BAD_ATTENTION, ids=str)
def test_attend_refuses(lib, bad):
    kw = {k: _rows(None) if v is _rows else _rows(*v) if isinstance(v, tuple) else v for k, v in bad.items()}
    assert _call(lib, a=_attention(**kw), b=_batch(**FULL)) == -1


def test_attend_refuses_work_and_sizes(lib):
    a, p, b = _attention(), _pages(NP=1000), _batch(N=1, T=1, width=1000, table_ld=1000)
    ref = [ctypes.byref(x) for x in (a, p, b)]
    assert _call(lib, a=a, p=p, b=b, longest=-1) == -1
    need = lib.lq_attend_workspace(*ref, 1)
    assert need > 0                                             # one token over 16000: pieces
    for work, n in ((None, need), (16, need - 1), (8, need)):
        assert lib.lq_attend(*ref, 1, work, n, None) == -1
    far = _batch(N=1, T=1, width=(1 << 27) - 1)                 # 2^31 - 16 places: a tile past the last would leave 32 bits
    assert _call(lib, a=a, b=far) == -1 and lib.lq_attend_workspace(ref[0], ref[1], ctypes.byref(far), 1) == -1
    big = _batch(N=1, T=1 << 30, width=4)
    assert _call(lib, a=a, b=big) == -1                         # rows in 32 bits


BAD_ROPE = [dict(HQ=0), dict(HQ=1 << 21), dict(rot=-16), dict(rot=24), dict(rot=144), dict(weight_bf16=4), dict(freq64=2), dict(interleaved=2),
            dict(eps=-1.0), dict(eps=float("nan")), dict(q=_rows), dict(k=_rows), dict(v=_rows), dict(out=_rows), dict(q_weight=None),
            dict(k_weight=None), dict(inv_freq=None), dict(q_weight=8), dict(k_weight=24), dict(inv_freq=18), dict(inv_freq=20, freq64=1),
            dict(k=(8,)), dict(v=(16, 260, 128)), dict(q=(16, 512, 4)), dict(out=(16, 64, 128)), dict(out=(16, 512, 0))]


@pytest.mark.parametrize("bad", BAD_ROPE, ids=str)
def test_rope_norm_refuses(lib, bad):
    kw = {k: _rows(None) if v is _rows else _rows(*v) if isinstance(v, tuple) else v for k, v in bad.items()}
    assert _call(lib, r=_rope(**kw), b=_batch(**FULL)) == -1


# ---- the Python operators -----------------------------------------------------------------------------------------------------
def _args(int8=False, **kw):
    d = R.inputs(1, [5, 3], [9, 40], 4, 2, 128, int8=int8, gate=True)
    d.update(kw)
    return d


def _both(d):
    from leapquant_amd import attn
    p = d.get("pages", attn.Pages(d["kp"], d["vp"], d["ks"], d["vs"]))
    return (lambda: attn.rope_norm(d["q"], d["k"], d["v"], d["qw"], d["kw"], d["inv_freq"], p, d["table"], d["loc"], d["lens"], d["out"],
                                   **d.get("rope", {})),
            lambda: attn.attend(d["q"], p, d["table"], d["loc"], d["lens"], d["out"], gate=d["gate"], **d.get("attend", {})))


@pytest.mark.parametrize("int8", [False, True])
def test_operators_take_gpu_tensors_only(int8):
    for call in _both(_args(int8)):
        with pytest.raises(ValueError, match="GPU tensors only"):
            call()


BOTH = [("q", lambda t: t.float(), TypeError), ("q", lambda t: t[:, :, :64], ValueError), ("q", lambda t: t.flatten(1), ValueError),
        ("q", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), ValueError), ("q", lambda t: t[:, :0], ValueError), ("q", lambda t: None, TypeError),
        ("q", lambda t: torch.cat([t, t], -1).flatten()[4:].as_strided(t.shape, (1024, 256, 1)), ValueError),
        ("out", lambda t: t.float(), TypeError), ("out", lambda t: t[:4], ValueError), ("out", lambda t: t[:1].expand(8, 4, 128), ValueError),
        ("out", lambda t: t[:, :1].expand(8, 4, 128), ValueError), ("out", lambda t: torch.zeros(9000, dtype=BF16).as_strided(t.shape, (128, 128, 1)), ValueError),
        ("kp", lambda t: t.float(), TypeError), ("kp", lambda t: t[0], ValueError), ("kp", lambda t: t[..., :96], ValueError),
        ("kp", lambda t: t[:, :8], ValueError), ("kp", lambda t: t[:0], ValueError), ("vp", lambda t: t[:2], ValueError), ("vp", lambda t: t.float(), TypeError),
        ("vp", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), ValueError), ("ks", lambda t: torch.zeros(1), ValueError),
        ("pages", lambda t: (1, 2), TypeError), ("pages", lambda t: (None, None, None, None), TypeError),
        ("table", lambda t: t[0], ValueError), ("table", lambda t: t.float(), TypeError), ("table", lambda t: t[:1], ValueError),
        ("table", lambda t: t[:, :1].expand(2, 1 << 27), ValueError),
        ("loc", lambda t: t[:2], ValueError), ("loc", lambda t: t[:, None], ValueError), ("loc", lambda t: t.float(), TypeError),
        ("lens", lambda t: t[:1], ValueError), ("lens", lambda t: t.double(), TypeError), ("lens", lambda t: [1, 2], TypeError)]


@pytest.mark.parametrize("name,change,error", BOTH, ids=lambda v: v if isinstance(v, str) else "")
def test_arguments_of_both(name, change, error):
    d = _args()
    d[name] = change(d.get(name))
    for call in _both(d):
        with pytest.raises(error):
            call()


ROPE = [("k", lambda t: t[:, :1], ValueError), ("k", lambda t: t.half(), TypeError), ("v", lambda t: t[:4], ValueError),
        ("qw", lambda t: t[:64], ValueError), ("qw", lambda t: t.half(), ValueError), ("kw", lambda t: t[None], ValueError),
        ("inv_freq", lambda t: t[:7], ValueError), ("inv_freq", lambda t: torch.cat([t, t]), ValueError), ("inv_freq", lambda t: t.half(), ValueError),
        ("inv_freq", lambda t: t[::2], ValueError), ("rope", lambda t: dict(eps=-1.0), ValueError), ("rope", lambda t: dict(eps="x"), TypeError),
        ("rope", lambda t: dict(offset=None), TypeError)]


@pytest.mark.parametrize("name,change,error", ROPE, ids=lambda v: v if isinstance(v, str) else "")
def test_arguments_of_rope_norm(name, change, error):
    d = _args()
    d[name] = change(d.get(name))
    with pytest.raises(error):
        _both(d)[0]()


ATTEND = [("attend", lambda t: dict(scale=0.0), ValueError), ("attend", lambda t: dict(scale=-1), ValueError), ("attend", lambda t: dict(scale=float("nan")), ValueError),
          ("attend", lambda t: dict(window=-1), ValueError), ("attend", lambda t: dict(window=2.5), TypeError), ("attend", lambda t: dict(longest=-1), ValueError),
          ("attend", lambda t: dict(longest=torch.tensor(3)), TypeError), ("gate", lambda t: t[:4], ValueError), ("gate", lambda t: t.float(), TypeError),
          ("q", lambda t: t[:, :3], ValueError)]


@pytest.mark.parametrize("name,change,error", ATTEND, ids=lambda v: v if isinstance(v, str) else "")
def test_arguments_of_attend(name, change, error):
    d = _args()
    d[name] = change(d.get(name))
    with pytest.raises(error):
        _both(d)[1]()


def test_scales_of_8_bits():
    for name, change in (("ks", lambda t: None), ("vs", lambda t: t.half()), ("vs", lambda t: t[:, :8]), ("ks", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))):
        d = _args(True)
        d[name] = change(d[name])
        for call in _both(d):
            with pytest.raises((ValueError, TypeError)):
                call()


def test_a_call_with_other_arguments_does_not_reach_the_tensors():
    from leapquant_amd import _lib
    c = _lib.attn_call()
    for f in (c.rope_norm, c.attend):
        for args in ((), (1,), (None,) * 14, (None,) * 10):
            with pytest.raises(TypeError):
                f(*args)


@pytest.mark.parametrize("scale", [2.0 ** 127, 3e38])
def test_attend_refuses_scales_that_leave_32_bits(lib, scale):
    """The kernels take scale times log2(e) in fp32; just below the border it is finite."""
    assert _call(lib, a=_attention(scale=scale), b=_batch(**FULL)) == -1
    assert lib.lq_attend_workspace(*(ctypes.byref(x) for x in (_attention(scale=1.7e38), _pages(), _batch(**FULL))), 0) >= 0
    d = _args()
    d["attend"] = dict(scale=scale)
    with pytest.raises(ValueError, match="2\\^127"):
        _both(d)[1]()
    d["attend"] = dict(scale=1.7e38)
    with pytest.raises(ValueError, match="GPU tensors only"):
        _both(d)[1]()
