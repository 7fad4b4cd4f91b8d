"""The kernels of the built liblq_attn.so against their compiled metadata (CPU): no register is spilled to scratch memory, the
registers allow the waves on a SIMD that each launch is drawn for."""
import os
import shutil

import pytest

from leapquant_amd import build as B
from tests import lq_codeobj as C

pytestmark = pytest.mark.skipif(not os.path.exists(B.ATTN_LIB) or not os.path.exists(C.READELF) or not shutil.which("c++filt"),
                                reason="needs the built liblq_attn.so, llvm-readelf and c++filt")

# (kernel, waves on a SIMD at least; heads of 256: one)
KERNELS = [("rope_norm_kernel", 4), ("few_kernel", 2), ("many_kernel", 2), ("both_kernel", 2), ("join_kernel", 4)]


@pytest.fixture(scope="module")
def kernels():
    return C.kernels(B.ATTN_LIB)


def test_every_kernel_is_listed(kernels):
    assert kernels and all(any(name in k["name"] for name, _ in KERNELS) for k in kernels)


@pytest.mark.parametrize("name,waves", KERNELS)
def test_registers_and_scratch(kernels, name, waves):
    hit = [k for k in kernels if name in k["name"]]
    assert hit, name
    for k in hit:
        # .vgpr_count holds the accumulation registers of a kernel that has them
        regs = -(-k["vgpr"] // 8) * 8
        assert k["block"] == 256 and k["scratch"] == 0, k
        assert C.VGPRS_PER_SIMD_LANE // regs >= (1 if waves == 2 and "<256" in k["name"] else waves), k
