"""Wait states behind wide stores in inline assembly.  A store of more than 64 bits reads its data registers a little later than
it is issued; on gfx950 a vector instruction may overwrite them two wait states behind it at the earliest.  The compiler sees to that
for its own stores but does not look into inline assembly, where the registers count as free behind the block.  So the device assembly of
every source is read here: inside the block, such a store has to be followed by two wait states."""
import os
import re
import shutil
import subprocess

import pytest

from test_build_resources import CSRC, HIPCC

SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
WIDE_STORE = re.compile(r"^(global|flat|buffer|scratch)_store_(dwordx[34]|b96|b128)\b")


def violations(assembly):
    """(number of wide stores in inline assembly, those with fewer than two wait states behind them in the block)"""
    stores, bad = 0, []
    for block in re.findall(r";;#ASMSTART\n(.*?);;#ASMEND", assembly, re.S):
        lines = [x.split(";")[0].split("//")[0].strip() for x in block.splitlines()]
        lines = [x for x in lines if x]
        for i, text in enumerate(lines):
            if WIDE_STORE.match(text):
                stores += 1
                passed = 0
                for x in lines[i + 1:]:
                    nop = re.match(r"s_nop (\d+)", x)
                    if not nop and not x.startswith("s_"):
                        break
                    passed += int(nop.group(1)) + 1 if nop else 1
                if passed < 2:
                    bad.append(text)
    return stores, bad


def test_the_check_itself():
    block = "\t;;#ASMSTART\n\tglobal_store_dwordx4 v[0:1], v[2:5], off sc1\n%s\t;;#ASMEND\n\tv_mov_b32 v2, 0\n"
    assert violations(block % "") == violations(block % "\ts_nop 0\n") == (1, ["global_store_dwordx4 v[0:1], v[2:5], off sc1"])
    assert violations(block % "\ts_nop 1\n") == violations(block % "\ts_nop 0\n\ts_waitcnt vmcnt(0)\n") == (1, [])
    assert violations((block % "").replace("dwordx4", "dwordx2")) == (0, [])
    assert violations("\tglobal_store_dwordx4 v[0:1], v[2:5], off\n\tv_mov_b32 v2, 0\n") == (0, [])


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="hipcc not found")
@pytest.mark.parametrize("source", SOURCES)
def test_wide_stores_in_inline_assembly_wait(source, tmp_path):
    text = open(os.path.join(CSRC, source)).read() + "".join(
        open(os.path.join(CSRC, h)).read() for h in re.findall(r'#include "(\w+\.hpp)"', open(os.path.join(CSRC, source)).read()))
    if not re.search(r"asm[^;]*_store_", text):
        return  # nothing to compile for
    out = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature",
                          "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", source, "-o", str(tmp_path / "out.s")],
                         cwd=CSRC, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    stores, bad = violations(open(tmp_path / "out.s").read())
    assert not bad, "%d of %d stores: %s" % (len(bad), stores, bad[0])
