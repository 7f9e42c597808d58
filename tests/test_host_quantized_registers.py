"""Registers of the built narrow kernels over a quantised cache, from the library's own
metadata: the bounds that they are compiled for hold what they keep."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from qattention_amd import build

LLVM = "/opt/rocm/llvm/bin"
NAME = re.compile(r"quant_attn_kernelINS_\d+(B?F16)E" + "".join(rf"Li(?P<{n}>\d+)E" for n in
                                                                ("D", "bits", "tiles", "waves", "heads", "sets")))


@pytest.fixture(scope="module")
def spills(tmp_path_factory):
    """(D, bits, tiles, heads) -> the most registers of a lane that any such kernel spills."""
    tools = [os.path.join(LLVM, t) for t in ("llvm-objdump", "llvm-readelf")]
    if not all(os.path.exists(t) for t in tools):
        pytest.skip("no LLVM tools")
    at = tmp_path_factory.mktemp("code")
    lib = shutil.copy(build.LIB_PATH, at)
    subprocess.run([tools[0], "--offloading", lib], cwd=at, check=True, capture_output=True)
    found = {}
    for f in sorted(at.iterdir()):
        if not f.name.endswith("gfx950"):
            continue
        notes = subprocess.run([tools[1], "--notes", str(f)], check=True, capture_output=True, text=True).stdout
        for name, spill in re.findall(r"\.name: +(\S+)\n.*?\.vgpr_spill_count: (\d+)\n", notes, re.S):
            m = NAME.search(name)
            if m:
                key = tuple(int(m[k]) for k in ("D", "bits", "tiles", "heads"))
                found[key] = max(found.get(key, 0), int(spill))
    return found


def test_kernels_are_found(spills):
    assert len(spills) == 6 * 2 + 5 * 2 + 3  # one head, one or two tiles; two heads, also with a tile each; four


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tiles", [1, 2])
def test_one_head_spills_nothing(spills, D, bits, tiles):
    assert spills[D, bits, tiles, 1] == 0


def test_several_heads(spills):
    """Two heads of 128 with a tile each fill a lane's 256 registers; no other form spills more
    than a few."""
    for (D, bits, tiles, heads), n in spills.items():
        assert n <= (24 if (D, tiles, heads) == (128, 2, 2) else 8), (D, bits, tiles, heads, n)
