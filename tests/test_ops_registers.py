"""What the tile products of the gated block take of a compute unit, read from the built library: their plan counts on
three blocks of 64 x 128 (168 registers), and the 256 x 256 gradient of the gate, which spills, was measured with so many
spilled registers. (Twelve more of the former and 13 more spilled made the gradients of 131,072 rows of 1600-240-240 and
8,192 of 2048-8192-2048 1 % slower.)"""
import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin/"


@pytest.fixture(scope="module")
def kernels(dp, tmp_path_factory):
    """{(element kind, layout, layout, epilogue, tile): (registers, spilled)} of the products."""
    if not (os.path.exists(LLVM + "llvm-objdump") and os.path.exists(LLVM + "llvm-readelf") and os.path.exists(dp.LIB_PATH)):
        pytest.skip("no tools, or the library is not built")
    at = tmp_path_factory.mktemp("kernels")
    subprocess.run([LLVM + "llvm-objdump", "--offloading", shutil.copy(dp.LIB_PATH, at)], check=True, cwd=at, capture_output=True)
    found = {}
    for name in os.listdir(at):
        if "gfx950" in name:
            text = subprocess.run([LLVM + "llvm-readelf", "--notes", name], check=True, cwd=at, capture_output=True, text=True).stdout
            for m in re.finditer(r"\.name:\s+\S*k_productILi(\d)ELi(\d)ELi(\d)ELi(\d)ENS_5ShapeILi(\d+)ELi(\d+)E.*?"
                                 r"\.vgpr_count:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", text, re.S):
                found[tuple(int(v) for v in m.groups()[:4]) + (m[5] + " x " + m[6],)] = int(m[7]), int(m[8])
    assert len(found) > 60
    return found


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_blocks_of_64_by_128(kernels, kind):
    for product in ((0, 1, 1), (0, 1, 0), (0, 0, 2), (0, 0, 0), (1, 1, 0)):
        assert kernels[(kind,) + product + ("64 x 128",)][0] <= 168, product


@pytest.mark.parametrize("kind", [0, 1])
def test_blocks_of_256_by_256(kernels, kind):
    for product, spilled in (((0, 1, 1), 0), ((0, 1, 0), 0), ((0, 0, 2), 17), ((0, 0, 0), 0), ((1, 1, 0), 16)):
        assert kernels[(kind,) + product + ("256 x 256",)][1] <= spilled, product
