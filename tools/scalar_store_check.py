"""Build-time gate: no kernel of the library writes through the scalar data cache.
Runs of such code were followed by whole-machine resets, so
__graft_entry__.build() refuses a library that contains any.

Stated from the other side: every instruction of the scalar-memory encoding (the
first dword's top six bits are 110000) is a load or a clock read.  Host only: it
disassembles the built .so (tools/isa_check.py) and runs nothing on a GPU."""
import os
import re
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import isa_check  # noqa: E402

READS = ("s_load_", "s_buffer_load_", "s_memtime", "s_memrealtime")
SCALAR_MEMORY = 0b110000

# "\ts_load_dword s0, s[4:5], 0x0   // 000000001900: C0020002 00000000"
_LINE = re.compile(r"^\s+([.a-z_0-9]+).*//\s*([0-9A-Fa-f]+):\s*([0-9A-Fa-f]{8})\b")
_HEAD = re.compile(r"^[0-9a-f]+ <([^>]+)>:")


def scan(listing):
    """(scalar-memory instructions seen, [what is not a read]) of a disassembly."""
    seen, problems, kernel = 0, [], "?"
    for line in listing.splitlines():
        h = _HEAD.match(line)
        if h:
            kernel = h.group(1)
        m = _LINE.match(line)
        if m and int(m.group(3), 16) >> 26 == SCALAR_MEMORY:
            seen += 1
            if not m.group(1).startswith(READS):
                problems.append("%s 0x%s: %s" % (kernel, m.group(2), m.group(1)))
    return seen, problems


def check(so_path=isa_check.DEFAULT_SO):
    problems = []
    for co in isa_check.code_objects(so_path):
        seen, bad = scan(isa_check._run("llvm-objdump", co, "-d", "--mcpu=gfx950"))
        problems += bad
        if not seen:  # a kernel loads its arguments this way
            problems.append("no scalar-memory instruction found: the listing's form is not known")
    return problems


if __name__ == "__main__":
    probs = check(sys.argv[1] if len(sys.argv) > 1 else isa_check.DEFAULT_SO)
    for p in probs:
        print(p)
    print("scalar_store_check: %s" % ("FAIL" if probs else "ok"))
    sys.exit(1 if probs else 0)
