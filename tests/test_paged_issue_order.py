"""Compiled order of the paged decode's tile loads, and its registers (CPU: hipcc cross-compiles gfx950).

A tile's K rows go to LDS by LDS-DMA loads, its V rows to registers, and K is read after an explicit wait for
all but 16 loads: right only if the tile's 16 V loads were issued after the last of its K loads. In a basic block,
between waits, no LDS-DMA load may therefore follow one of V, and K loads come as whole tiles. A wait for
everything inside the loop would end the look-ahead (no fault, but a memory latency for every tile), as would
spilled addresses."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_decode_issue_order import _build_module

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(),
                                reason="hipcc not installed")
NAME = re.compile(r"attn_paged_partials_kernelILi(\d)ELb(\d)ELb(\d)ELb(\d)E")  # NT, KV8, P16, BATCH


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    b = _build_module()
    src, out = b.CSRC / "attn_paged.hip", tmp_path_factory.mktemp("asm") / "attn_paged.s"
    cmd = [b.HIPCC, *b.HIP_FLAGS, *b.SOURCE_FLAGS.get(src.name, []), "--offload-device-only", "-S",
           "-Rpass-analysis=kernel-resource-usage", str(src), "-o", str(out)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout[-2000:]
    usage = {}
    for line in r.stdout.splitlines():
        if m := re.search(r"Function Name: (\S+)", line):
            usage[m.group(1)] = cur = {}
        elif m := re.search(r"remark: .*?(ScratchSize \[bytes/lane\]|Occupancy \[waves/SIMD\]): (\d+)", line):
            cur[m.group(1)] = int(m.group(2))
    asm = out.read_text()
    bodies = {}
    for m in re.finditer(r"^(_Z\S*attn_paged_partials_kernel\S*):", asm, re.M):
        bodies[m.group(1)] = asm[m.end():asm.index(".Lfunc_end", m.end())]
    return bodies, usage


def runs(body):
    """Runs of buffer loads: 'L' to LDS, 'R' to registers, '|' a wait for loads, '0' one for all of them."""
    out = []
    for block in re.split(r"^(?:\.LBB\d+_\d+:|; %bb).*$", body, flags=re.M):
        s = ""
        for line in block.split("\n"):
            t = line.strip()
            if t.startswith("s_waitcnt") and (m := re.search(r"vmcnt\((\d+)\)", t)):
                s += "0" if m.group(1) == "0" else "|"
            elif t.startswith("buffer_load"):
                s += "L" if t.endswith(" lds") else "R"
        out.append(s)
    return out


def test_tile_loads_keep_their_order(compiled):
    bodies, _ = compiled
    assert len(bodies) == 16
    for name, body in bodies.items():
        m = NAME.search(name)
        tile = 8 if m.group(2) == "1" else 16
        got = [r for block in runs(body) if (r := re.sub("[|0]", "", block))]
        assert set(got) <= {"L" * tile + "R" * 16, "L" * tile, "R" * 16}, (name, got)
        assert "L" * tile + "R" * 16 in got, name  # an item's first tile


def test_the_loop_does_not_wait_for_all_loads(compiled):
    """In a block that issues a tile's K and later the next V, no wait in between is one for everything."""
    for name, body in compiled[0].items():
        for block in runs(body):
            if m := re.search(r"L+([|0]*)R", block):
                assert "0" not in m.group(1), name


def test_registers(compiled):
    """No kernel spills to memory (some keep registers in the other half of the file), and two workgroups of the
    fp8 kernel with one column tile fit on a compute unit."""
    usage = {k: v for k, v in compiled[1].items() if NAME.search(k)}
    assert len(usage) == 16
    for name, u in usage.items():
        assert u["ScratchSize [bytes/lane]"] == 0, (name, u)
        if NAME.search(name).groups()[:2] == ("1", "1"):
            assert u["Occupancy [waves/SIMD]"] >= 2, (name, u)
