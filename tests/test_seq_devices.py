"""The sequence operators in a process with several GPUs (CPU): what is asked of the runtime once a device, and which device is
current at a launch.  The library runs against stand-ins for the HIP runtime's entry points (tests/hip_stub.cpp)."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

from leapquant_amd import _lib, seq
from tests.test_seq_state import call

HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = """
import ctypes, importlib.util, sys
stub, root, path = sys.argv[1:]
hip = ctypes.CDLL(stub, mode=ctypes.RTLD_GLOBAL)            # before the library, which then finds these first
spec = importlib.util.spec_from_file_location("_lib", root + "/leapquant_amd/_lib.py")
M = importlib.util.module_from_spec(spec); spec.loader.exec_module(M)
L = M.seq_lib()
d = M.LqDelta(S=16, slot_stride=4 * 128 * 128, NS=3, HV=4, H=2, K=128, V=128, mixed=16, a=16, b=16, A_log=16, dt_bias=16, out=16,
              mixed_ld=1024, a_ld=4, b_ld=4, scale=0.1, gate_bf16=0, kda=0, glb=0.0)
s = M.LqSeqs(loc=16, idx=16, src=None, N=1, T=100)
n = L.lq_delta_workspace(ctypes.byref(d), ctypes.byref(s))
def prefill(device):
    hip.stub_device(device)
    return L.lq_delta_prefill(ctypes.byref(d), ctypes.byref(s), 16, n, None)
assert prefill(0) == 0 and prefill(0) == 0 and hip.stub_launches() == 4
assert prefill(1) == 0 and prefill(3) == 0 and prefill(0) == 0 and prefill(3) == 0
assert [hip.stub_asked(i) for i in range(4)] == [1, 1, 0, 1], [hip.stub_asked(i) for i in range(4)]
hip.stub_fail(1)
before = hip.stub_launches()
assert prefill(2) == -2 and hip.stub_launches() == before   # no launch without it
assert prefill(2) == 0 and hip.stub_asked(2) == 1           # and asked for again
print("ok")
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="needs g++")
def test_lds_is_asked_for_on_every_device(tmp_path):
    stub = str(tmp_path / "libhipstub.so")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", os.path.join(HERE, "hip_stub.cpp"), "-o", stub], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, stub, os.path.dirname(HERE), _lib.SEQ_LIB_PATH], capture_output=True, text=True,
                       env=dict(os.environ, HIP_VISIBLE_DEVICES="-1"))
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr


@pytest.mark.parametrize("T", [5, 40])
def test_the_tensors_device_is_current_at_the_launch(monkeypatch, T):
    """A default stream is the current device's: with another one current, the launch would go there."""
    now, at = [], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            now.append(self.dev)

        def __exit__(self, *e):
            now.pop()

    class Lib:
        lq_delta_check = staticmethod(lambda *a: 0)
        lq_delta_workspace = staticmethod(lambda *a: 0)
        lq_delta_steps = lq_delta_prefill = staticmethod(lambda *a: at.append(list(now)) or 0)
    st, d = call(T=T)
    monkeypatch.setattr(seq, "_on", lambda *a, **k: None)
    monkeypatch.setattr(seq, "_raw_stream", lambda t: 0)
    monkeypatch.setattr(_lib, "seq_lib", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    for name in ("dequantize", "quantize"):
        monkeypatch.setattr(st, name, lambda *a: at.append(list(now)))
    st.prefill(**d)
    assert at == [[-1]] * 3                      # the host's index: the checkpoints' way there, the rule, the way back
