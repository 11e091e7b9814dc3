"""Host-side check (no GPU needed) of the built library's device code: wait states that
the hardware wants between two instructions and that the compiler cannot keep where one of
them is inline assembly.

- A vector instruction writes a scalar register, a memory instruction reads it: 5.
- A vector instruction writes a register, a matrix instruction reads it: 2.

The compiler keeps exactly these for instructions that it knows. The code is read in the
order in which it lies; every instruction between counts as one, s_nop as what it says.
"""
import os
import re
import struct
import subprocess

import pytest

import hkq

OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", "/usr/bin/llvm-objdump") if os.path.exists(p)), None)
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
OPERAND = re.compile(r"\b([sva])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text, kinds):
    out = []
    for kind, lo, hi, one in OPERAND.findall(text):
        if kind in kinds:
            out += [(kind, r) for r in (range(int(lo), int(hi) + 1) if lo else (int(one),))]
    return out


def short_waits(lines):
    """(what, wait states, function, instruction) of every pair that is too close; also the number of loads and products read."""
    scalar, vector, now, where, seen, bad = {}, {}, 0, "", [0, 0], []
    for line in lines:
        if line[:1] != "\t":
            if line.endswith(">:\n"):
                scalar, vector, where = {}, {}, line.split("<")[-1][:-3]
            continue
        name, _, ops = line.split("//")[0].strip().partition(" ")
        if name == "s_nop":
            now += int(ops, 0) + 1
            continue
        now += 1
        if name[:2] == "v_":
            first, _, rest = ops.partition(",")
            if name.startswith("v_mfma") or name.startswith("v_smfma"):
                seen[1] += 1
                close = [now - 1 - vector[r] for r in registers(rest, "va") if now - 1 - vector.get(r, -9) < 2]
                if close:
                    bad.append(("matrix operand", min(close), where, line.strip()))
                for r in registers(first, "va"):
                    vector.pop(r, None)
                continue
            for r in registers(first, "va"):
                vector[r] = now
            if "_swap" in name:
                for r in registers(rest, "va"):
                    vector[r] = now
            for r in registers(ops.rsplit(",", 2)[0] if "_co_" in name else first, "s"):
                scalar[r] = now
        elif name.startswith(("buffer_", "global_", "flat_", "scratch_")):
            seen[0] += 1
            close = [now - 1 - scalar[r] for r in registers(ops, "s") if now - 1 - scalar.get(r, -9) < 5]
            if close:
                bad.append(("load", min(close), where, line.strip()))
            if "lds" not in ops and "store" not in name:
                for r in registers(ops.partition(",")[0], "va"):
                    vector.pop(r, None)
        elif name.startswith("ds_"):
            for r in registers(ops.partition(",")[0], "va"):
                vector.pop(r, None)
        elif name[:2] == "s_":
            for r in registers(ops.partition(",")[0], "s"):
                scalar.pop(r, None)
    return bad, seen


def test_the_reader_of_code():
    def code(*lines):
        return short_waits(["0000 <f>:\n"] + ["\t" + x + " // 0: 0\n" for x in lines])

    copy, load = "v_readfirstlane_b32 s6, v1", "buffer_load_dwordx4 v2, s[4:7], 0 offen lds"
    assert code(copy, "s_mov_b32 m0, s9", "s_nop 0", load)[0][0][:3] == ("load", 2, "f")
    assert code(copy, "s_mov_b32 m0, s9", "s_nop 3", load) == ([], [1, 0])
    assert code(copy, "s_mov_b32 s6, s9", load) == ([], [1, 0])
    perm, product = "v_perm_b32 v7, v1, v2, s0", "v_mfma_f32_16x16x32_bf16 v[0:3], v[10:13], v[4:7], v[0:3]"
    assert code(perm, "v_mov_b32_e32 v9, v8", product)[0][0][:2] == ("matrix operand", 1)
    assert code(perm, "s_nop 1", product) == ([], [0, 1])
    assert code("v_accvgpr_write_b32 a1, v9", "v_mfma_f32_32x32x16_bf16 a[0:15], v[10:13], v[4:7], a[0:15]")[0][0][1] == 0


@pytest.mark.skipif(OBJDUMP is None, reason="no disassembler")
def test_wait_states_of_the_library(tmp_path):
    with open(hkq.LIB_PATH, "rb") as f:
        lib = f.read()
    at, loads, products = lib.find(MAGIC), 0, 0
    assert at >= 0
    while at >= 0:
        n, = struct.unpack_from("<Q", lib, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(n if n < 16 else 0):  # (the name itself may stand elsewhere in the file)
            offset, size, length = struct.unpack_from("<QQQ", lib, entry)
            target = lib[entry + 24:entry + 24 + length]
            entry += 24 + length
            if b"gfx950" not in target or size == 0:
                continue
            obj = tmp_path / "device.o"
            obj.write_bytes(lib[at + offset:at + offset + size])
            with subprocess.Popen([OBJDUMP, "-d", str(obj)], stdout=subprocess.PIPE, text=True) as p:
                bad, seen = short_waits(p.stdout)
            assert p.returncode == 0
            assert not bad, f"{len(bad)} in all, first: {bad[0]}"
            loads, products = loads + seen[0], products + seen[1]
        at = lib.find(MAGIC, at + 1)
    assert loads > 1000 and products > 10000, "the library's code was not read"
