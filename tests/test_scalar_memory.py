"""The build's scan for scalar-memory instructions that are not reads
(tools/scalar_store_check.py): on the built library and on lines by hand."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LLVM = "/opt/rocm/lib/llvm/bin"


@pytest.fixture(scope="module")
def gate():
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import scalar_store_check
    return scalar_store_check


HEAD = "0000000000001900 <kernel>:\n"


def test_lines(gate):
    reads = HEAD + ("\ts_load_dwordx4 s[0:3], s[4:5], 0x0    // 000000001900: C00A0002 00000000\n"
                    "\ts_memrealtime s[0:1]                  // 000000001908: C0940000 00000000\n"
                    "\tv_mov_b32_e32 v0, s0                  // 000000001910: 7E000200\n"
                    "\ts_endpgm                              // 000000001914: BF810000\n")
    assert gate.scan(reads) == (2, [])
    for name in ("s_other_dword", ".long"):  # another of that encoding, or one it cannot name
        other = "\t%s s0, s[4:5], 0x0                 // 000000001918: C0400002 00000000\n" % name
        seen, problems = gate.scan(reads + other)
        assert seen == 3 and len(problems) == 1
        assert all(w in problems[0] for w in ("kernel", "1918", name))


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-objdump")),
                    reason="ROCm llvm tools absent")
def test_the_library(gate):
    assert gate.check() == []
    import isa_check
    insns = [m for k in isa_check.disassemble_all(isa_check.DEFAULT_SO).values() for _, m, _, _ in k]
    listed = sum(m.startswith(gate.READS) for m in insns)
    seen = sum(gate.scan(isa_check._run("llvm-objdump", co, "-d", "--mcpu=gfx950"))[0]
               for co in isa_check.code_objects(isa_check.DEFAULT_SO))
    assert listed > 1000 and seen == listed
