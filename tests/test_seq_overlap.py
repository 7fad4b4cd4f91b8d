"""Outputs whose rows overlap each other are refused (CPU, before any launch): rows would be written over one another in no order."""
import ctypes

import pytest
import torch

from leapquant_amd import _lib, seq
from tests.test_seq_boundary import _norm


@pytest.mark.parametrize("bad", [dict(rows=2, o_ld=0), dict(rows=2, o_ld=63), dict(rows=1, heads=2, o_hd=0), dict(rows=3, heads=2, o_hd=32)],
                         ids=str)
def test_entries_refuse(bad):
    n = _norm(**bad)
    assert _lib.seq_lib().lq_gated_norm(ctypes.byref(n), None) == -1
    assert _lib.seq_lib().lq_add_norm(ctypes.byref(n), None) == -1


def test_operators_refuse():
    x, w = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.ones(64)
    for out in (x[:1].expand(4, 2, 64), x[:, :1].expand(4, 2, 64), torch.zeros(4000, dtype=torch.bfloat16).as_strided(x.shape, (100, 36, 1))):
        for fn in (lambda: seq.gated_norm(x, x, w, out), lambda: seq.add_norm(x, x, w, out, out)):
            with pytest.raises(ValueError, match="overlap"):
                fn()
    for out in (x, x.transpose(0, 1).contiguous().transpose(0, 1), torch.zeros(4, 2, 72, dtype=torch.bfloat16)[..., :64]):
        with pytest.raises(ValueError, match="GPU tensors only"):    # all but the device is as it should be
            seq.gated_norm(x[:1].expand(4, 2, 64), x, w, out)
