"""Rotary positions and windowed attention where a call can go wrong, without a device: the built code's waits, sizes of workspaces and grids, what a plan holds, options of the
text tower."""
import os
import re
import subprocess

import pytest

from ct_clip_amd import build

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def windowed_kernels(tmp_path_factory):
    """{symbol: instructions (and None where a block begins)} of the built library's windowed attention kernels."""
    if not os.path.exists(OBJDUMP) or not os.path.exists(build.LIB):
        pytest.skip("needs the built library and llvm-objdump")
    where = tmp_path_factory.mktemp("isa")
    os.symlink(build.LIB, where / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=where, check=True, capture_output=True)
    kernels = {}
    for f in sorted(where.glob("*gfx950")):
        if b"3win" not in f.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", str(f)], check=True, capture_output=True, text=True).stdout
        at = None
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
            if m and re.fullmatch(r"L\d+", m[1]):
                if at is not None:
                    at.append(None)
            elif m:
                at = kernels.setdefault(m[1], []) if "3win" in m[1] else None
            elif at is not None and line.startswith("\t"):
                at.append(line.split("//")[0].strip())
    return kernels


def test_a_tile_is_refilled_behind_the_reads_of_it(windowed_kernels):
    """Loads into LDS are not ordered with a wave's LDS reads: in the block that starts a refill, a wait for them stands in front."""
    seen = set()
    for name, code in windowed_kernels.items():
        for i, ins in enumerate(code):
            if not (ins and ins.startswith("buffer_load") and ins.endswith("lds")):
                continue
            seen.add(re.search(r"(fwd_kernel|rows_kernel|dq_kernel|dkv_kernel)", name)[1])
            back = i - 1
            while code[back] and not code[back].startswith(("ds_read", "s_branch", "s_cbranch")) and "lgkmcnt(0)" not in code[back]:
                back -= 1
            assert code[back] and "lgkmcnt(0)" in code[back], f"{name}: {code[back]} ... {ins}"
    assert seen == {"fwd_kernel", "rows_kernel", "dq_kernel", "dkv_kernel"}
