"""Stores written as inline asm bring the wait that the compiler adds to its own.

A store of more than 64 bits reads its data after it is issued: a VALU write of
those registers within two wait states may change what is stored. The compiler
keeps them apart for stores that it knows and sees none in asm."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qwen3.8-flash-next-fp4-local-spark_amd")
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
STATES = 2


def test_sources():
    """Every wide store in asm is followed there by `s_nop 1` or more, which is two wait states."""
    csrc, seen = os.path.join(PKG, "csrc"), 0
    for name in sorted(os.listdir(csrc)):
        path = os.path.join(csrc, name)
        if not os.path.isfile(path):
            continue
        for text in re.findall(r"asm volatile\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", open(path).read()):
            lines = [s.strip() for s in "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", text)).replace("\\n", "\n").replace("\\t", "\t").splitlines()]
            for i, line in enumerate(lines):
                if re.match(r"(global|flat|buffer|scratch)_store_dwordx[34]\b", line):
                    seen += 1
                    after = re.fullmatch(r"s_nop (\d+)", lines[i + 1]) if i + 1 < len(lines) else None
                    assert after and int(after.group(1)) + 1 >= STATES, (name, line)
    assert seen >= 1


def registers(operand):
    m = re.fullmatch(r"([va])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    lo, hi = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(lo), int(hi) + 1)}


def early_writes(lines):
    """VALU writes of a wide store's data within STATES wait states of it, in a listing's order."""
    bad, near, stores = [], [], 0
    for line in lines:
        line = line.split("//")[0].strip()
        if not line or line.endswith(":"):
            near = []                                # another block or kernel
            continue
        op, _, rest = line.partition(" ")
        args = [a.strip() for a in re.split(r",\s*(?![^\[]*\])", rest)]
        if op.startswith("v_"):
            wrote = registers(args[0]) | (registers(args[1]) if "swap" in op else set())
            bad += [(store, line) for data, store, _ in near if data & wrote]
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        near = [(data, store, age + states) for data, store, age in near if age + states < STATES]
        m = re.match(r"(global|flat|scratch|buffer)_store_dwordx[34]", op)
        if m:
            stores += 1
            near.append((registers(args[0] if m[1] == "buffer" else args[1]), line, 0))
    return bad, stores


def test_the_check_finds_one():
    store = "global_store_dwordx4 v[10:11], v[4:7], off nt"
    for between, found in (([], 1), (["s_nop 0"], 1), (["s_nop 1"], 0), (["s_mov_b32 s0, 0", "s_mov_b32 s1, 0"], 0), (["v_mov_b32_e32 v8, 0"], 1)):
        assert len(early_writes([store, *between, "v_add_f32_e32 v7, v1, v2"])[0]) == found
    assert len(early_writes([store, "v_permlane16_swap_b32_e32 v1, v5"])[0]) == 1
    assert not early_writes(["global_store_dwordx4 v10, v[4:7], s[0:1]", "v_add_f32_e32 v10, v1, v2"])[0]


def test_built_products(tmp_path):
    """The same over the code of the products of e4m3 as built, whose stores past the L2 are asm."""
    lib = os.path.join(PKG, "libfp4x.so")
    if not os.path.exists(OBJDUMP) or not os.path.exists(lib):
        pytest.skip("needs llvm-objdump and libfp4x.so")
    copy = shutil.copy(lib, tmp_path / "lib.so")
    assert subprocess.run([OBJDUMP, "--offloading", copy], capture_output=True).returncode == 0
    seen = 0
    for part in sorted(tmp_path.iterdir()):
        if not part.name.endswith("gfx950") or b"f8_tile_kernel" not in part.read_bytes():
            continue
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], capture_output=True, text=True)
        assert r.returncode == 0
        bad, stores = early_writes(r.stdout.splitlines())
        assert not bad, (len(bad), bad[0])
        seen += stores
    assert seen > 100
