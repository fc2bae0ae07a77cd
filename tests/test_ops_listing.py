"""What the compiler does not check of the instructions that product.h writes itself, read from the
built library: the loads straight into LDS take their address from scalar registers, and
where a vector instruction (a lane read) wrote one of these, five wait states have to lie between. The
compiler inserts them for its own instructions, not for written ones; here their addresses come from
scalar instructions, which need none."""
import os
import re
import shutil
import subprocess

import pytest

DUMP = "/opt/rocm/llvm/bin/llvm-objdump"
STATES = 5


def scalars(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", operand)
    return {int(m[1])} if m else set()


def too_early(lines):
    """(loads seen, those whose address a vector instruction wrote fewer than five states before)."""
    before, seen, bad = [], 0, []
    for line in lines:
        m = re.match(r"\s+([a-z]\w+)\s*(.*?)\s*(//.*|;.*)?$", line)
        if not m:
            continue
        op, args = m[1], [a.strip() for a in m[2].split(",")]
        if op.startswith("global_load_lds"):
            seen += 1
            address, states = scalars(args[1].split()[0]), 0
            for o, a in reversed(before):
                if states >= STATES:
                    break
                written = a[:2] if "_co_" in o or "div_scale" in o else a[:1]  # (the former two write a mask too)
                if o.startswith("v_") and address & set().union(*map(scalars, written)):
                    bad.append(line.strip())
                    break
                states += int(a[0], 0) + 1 if o == "s_nop" else 1
        before = (before + [(op, args)])[-8:]
    return seen, bad


def test_reader():
    head = "\tv_readfirstlane_b32 s5, v3  // 0000\n"
    load = "\tglobal_load_lds_dwordx4 v1, s[4:5]  // 0000\n"
    assert too_early((head + "\ts_mov_b32 m0, s9\n\ts_nop 0\n" + load).split("\n")) == (1, [load.strip().split("\n")[0]])
    assert too_early((head + "\ts_mov_b32 m0, s9\n\ts_nop 3\n" + load).split("\n")) == (1, [])
    assert too_early(("\ts_add_u32 s4, s6, s7\n\ts_mov_b32 m0, s9\n\ts_nop 0\n" + load).split("\n")) == (1, [])
    assert too_early(("\tv_add_u32_e32 v1, s4, v1\n" + load).split("\n")) == (1, [])
    assert too_early((head.replace("s5", "s6") + load).split("\n")) == (1, [])


def test_addresses_of_the_loads_into_lds(dp, tmp_path):
    if not (os.path.exists(DUMP) and os.path.exists(dp.LIB_PATH)):
        pytest.skip("no disassembler, or the library is not built")
    lib = shutil.copy(dp.LIB_PATH, tmp_path)
    subprocess.run([DUMP, "--offloading", lib], check=True, cwd=tmp_path, capture_output=True)
    seen = 0
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name:
            continue
        text = subprocess.run([DUMP, "-d", name], check=True, cwd=tmp_path, capture_output=True, text=True).stdout
        if "k_product" not in text:
            continue
        n, bad = too_early(text.split("\n"))
        seen += n
        assert not bad, (name, bad[:3])
    assert seen > 1000
