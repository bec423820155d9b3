"""Compiled order of the paged decode's merge (CPU: hipcc cross-compiles gfx950): the first slots of a row are loaded
in the first block that loads anything but arguments, before a branch that needs the row's position. (An early return of
idle rows moves them behind it, and costs every row a memory latency.)"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_decode_issue_order import _build_module

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(),
                                reason="hipcc not installed")


def test_the_first_slots_are_loaded_ahead_of_the_position(tmp_path):
    b = _build_module()
    src, out = b.CSRC / "attn_paged.hip", tmp_path / "attn_paged.s"
    cmd = [b.HIPCC, *b.HIP_FLAGS, *b.SOURCE_FLAGS.get(src.name, []), "--offload-device-only", "-S", str(src), "-o",
           str(out)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout[-2000:]
    asm, seen = out.read_text(), set()
    for m in re.finditer(r"^(_Z\S*attn_paged_combine_kernelILi(\d+)ELi(\d+)E\S*):", asm, re.M):
        body = asm[m.end():asm.index(".Lfunc_end", m.end())]
        blocks = re.split(r"^\.LBB\d+_\d+:.*$|^\s*s_c?branch\S*.*$", body, flags=re.M)
        first = next(x for x in blocks if "global_load" in x)
        # a slot is a 16-byte and an 8-byte load (the compiler may issue them in any order)
        assert len(re.findall(r"global_load_dwordx4", first)) == int(m.group(3)), m.group(1)
        assert "vmcnt" not in first, m.group(1)
        seen.add(m.group(2))
    assert seen == {"1", "4", "16"}
