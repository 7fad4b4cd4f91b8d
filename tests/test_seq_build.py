"""What is built and shipped of the sequence operators (CPU): stale files are refused before a call."""
import pytest

from leapquant_amd import _lib


def test_a_library_of_another_version_is_refused(monkeypatch):
    """Structures go to the library as bytes: a file of another layout, or one without a version, must not get them."""
    assert _lib.seq_lib().lq_seq_abi_version() == _lib.SEQ_ABI_VERSION
    monkeypatch.setattr(_lib, "_SEQ_LIB", [None])
    with monkeypatch.context() as m:
        m.setattr(_lib, "SEQ_ABI_VERSION", 10 ** 6)
        with pytest.raises(RuntimeError, match="rebuild"):
            _lib.seq_lib()
    monkeypatch.setattr(_lib, "SEQ_LIB_PATH", _lib.LIB_PATH)         # a library that has no such version
    with pytest.raises(RuntimeError, match="rebuild"):
        _lib.seq_lib()


def test_an_extension_of_another_build_is_refused(monkeypatch):
    """The extension reads torch's tensors and fills the library's structures: both as they were when it was built."""
    import torch
    monkeypatch.setattr(_lib, "_SEQ_CALL", [None])
    c = _lib.seq_call()
    assert (c.ABI, c.TORCH) == (_lib.SEQ_ABI_VERSION, torch.__version__)
    for where, name, value in ((torch, "__version__", "1.0"), (_lib, "SEQ_ABI_VERSION", 10 ** 6)):
        monkeypatch.setattr(_lib, "_SEQ_CALL", [None])
        with monkeypatch.context() as m:
            m.setattr(where, name, value)
            with pytest.raises(RuntimeError, match="rebuild"):
                _lib.seq_call()
