"""What is built and shipped of the sequence operators (CPU): stale files are refused before a call."""
import fnmatch
import os

import pytest

from leapquant_amd import _lib, build as B

ROOT = os.path.dirname(B.HERE)


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


def test_the_package_ships_what_it_loads():
    """An installed package holds the libraries that its modules load, and the sources of each."""
    tomli = pytest.importorskip("tomli")
    with open(os.path.join(ROOT, "pyproject.toml"), "rb") as f:
        globs = tomli.load(f)["tool"]["setuptools"]["package-data"]["leapquant_amd"]
    files = [_lib.LIB_PATH, _lib.SEQ_LIB_PATH, _lib.SEQ_CALL_PATH] + [os.path.join(B.CSRC, f) for f in os.listdir(B.CSRC)]
    for f in files:
        assert any(fnmatch.fnmatch(os.path.relpath(f, B.HERE), g) for g in globs), f
