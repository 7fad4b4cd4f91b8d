"""The order of barriers and LDS writes in the built kernels that take many rows (CPU, from the assembly of the library built here).

A workgroup's waves share tiles of keys in LDS.  Before their loop they load the first tiles, meet at a barrier and each read the
first tile's keys, their neighbours' part among them, for the first scores.  The loop then fills those places again.  Between such
reads and the next writes into LDS every wave has to meet the others once more: a wave that is ahead, above all one without rows,
would write over keys that a slower one still reads.  When that happens depends on timing, which no run shows for certain: so
here no path from that first barrier may lead to a write into LDS without another barrier between."""
import os
import re
import subprocess
import tempfile

import pytest

from leapquant_amd import build as B
from tests import lq_codeobj as C

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
pytestmark = pytest.mark.skipif(not os.path.exists(B.ATTN_LIB) or not os.path.exists(OBJDUMP), reason="needs the built liblq_attn.so and llvm-objdump")
WRITES = re.compile(r"global_load_lds_|buffer_load_\w+ .*\blds\b|ds_write|ds_store")
PRODUCT = "v_mfma_f32_32x32x16_bf16"            # of many rows alone


def functions():
    """{mangled name: [(address, instruction, address that it may branch to or None)]}"""
    out = {}
    for co in C._code_objects(B.ATTN_LIB):
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(co)
            f.flush()
            text = subprocess.run([OBJDUMP, "-d", f.name], capture_output=True, text=True, check=True).stdout
        code = None
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if head:
                code = out.setdefault(head.group(1), [])
            ins = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+): ([0-9A-F]{8})", line)
            if ins and code is not None:
                at, to = int(ins.group(2), 16), None
                if re.match(r"s_c?branch", ins.group(1)):
                    step = int(ins.group(3), 16) & 0xffff
                    to = at + 4 + 4 * (step - 0x10000 if step & 0x8000 else step)
                code.append((at, ins.group(1), to))
    return out


def reached(code, index, start):
    """Instructions that may run after code[start] (start -1: from the entry) up to and with the next barrier on each way."""
    seen, todo = set(), [start + 1]
    while todo:
        i = todo.pop()
        if i in seen or i >= len(code):
            continue
        seen.add(i)
        _, ins, to = code[i]
        assert not re.match(r"s_(setpc|swappc|call)", ins), ins
        if re.match(r"s_barrier|s_endpgm", ins):
            continue
        if to is not None:
            todo.append(index[to])
        if not ins.startswith("s_branch"):
            todo.append(i + 1)
    return seen


@pytest.fixture(scope="module")
def code():
    return functions()


@pytest.mark.parametrize("kernel,count", [("many_kernel", 6), ("both_kernel", 6)])
def test_tiles_are_not_written_over_while_the_first_scores_read_them(code, kernel, count):
    hit = [name for name in code if kernel in name and not name.endswith(".kd")]
    assert len(hit) == count                                    # heads of 64, 128 and 256, in bf16 and from codes
    for name in hit:
        ins = code[name]
        index = {at: i for i, (at, _, _) in enumerate(ins)}
        starts = 0
        for i in sorted(reached(ins, index, -1)):
            if not ins[i][1].startswith("s_barrier"):
                continue
            after = reached(ins, index, i)
            if any(ins[j][1].startswith(PRODUCT) for j in after):           # the first tiles are there; the first scores follow
                starts += 1
                early = [ins[j][1] for j in after if WRITES.match(ins[j][1])]
                assert not early, (name, early[:4])
        assert starts >= 1, name
