"""The kernels of the built liblq_seq.so against their compiled metadata (CPU): no register is spilled to scratch memory, the
registers allow the waves on a SIMD that each launch is drawn for, and the LDS fits a compute unit."""
import os
import shutil

import pytest

from leapquant_amd import build as B
from tests import lq_codeobj as C

pytestmark = pytest.mark.skipif(not os.path.exists(B.SEQ_LIB) or not os.path.exists(C.READELF) or not shutil.which("c++filt"),
                                reason="needs the built liblq_seq.so, llvm-readelf and c++filt")

# (kernel, threads, waves on a SIMD at least)
KERNELS = [("walk_kernel", 512, 2), ("lone_kernel", 256, 3), ("chunk_kernel", 256, 4), ("steps_kernel", 256, 2),
           ("conv_seq_kernel", 256, 4), ("norm_kernel", 256, 2)]


@pytest.fixture(scope="module")
def kernels():
    return C.kernels(B.SEQ_LIB)


def test_every_kernel_is_listed(kernels):
    assert kernels and all(any(name in k["name"] for name, _, _ in KERNELS) for k in kernels)


@pytest.mark.parametrize("name,threads,waves", KERNELS)
def test_registers_and_scratch(kernels, name, threads, waves):
    hit = [k for k in kernels if name in k["name"]]
    assert hit, name
    for k in hit:
        regs = -(-(k["vgpr"] + k["agpr"]) // 8) * 8
        assert k["block"] == threads and k["scratch"] == 0 and k["lds"] <= 64 * 1024, k
        assert C.VGPRS_PER_SIMD_LANE // regs >= waves, k
