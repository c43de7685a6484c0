"""tools/build_variant.sh builds what the Makefile builds: every source, the same
code-generation flags (no compiler is run)."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "distributed_ddpg_amd", "csrc")


def command():
    text = open(os.path.join(ROOT, "tools", "build_variant.sh")).read()
    return text[text.index("hipcc"):].replace("\\\n", " ").split("\n")[0].split()


def test_every_source_is_in_it():
    named = [w for w in command() if w.endswith((".hip", ".cpp"))]
    found = {os.path.basename(f) for w in named for f in glob.glob(os.path.join(CSRC, w))}
    assert found == {f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp"))}


def test_its_flags_are_the_makefiles():
    make = open(os.path.join(CSRC, "Makefile")).read().replace("\\\n", " ")
    flags = re.search(r"^CXXFLAGS := (.*)$", make, re.M).group(1).replace("$(ARCH)", "gfx950")
    kept = [w for w in flags.split() if not w.startswith(("-I", "-W"))]
    got = command()
    assert "-packed-fp32-ops" in kept and [w for w in got if w in kept] == kept, (kept, got)
