"""Host-side check (no GPU needed) of the INT4 operands that inline assembly makes: the
generated code keeps two wait states between its last write and the matrix instruction
that reads them, as the compiler does for its own instructions. Compiled without a GPU."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "amd-kernels_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

KERNEL = """
#include "w4_core.h"
using namespace hkq;
__global__ void product(const uint32_t* w, const v4i* x, v4f* out) {
    v4f c = out[threadIdx.x];
    const v4i a = x[threadIdx.x];
    const v4i b = int4_sixteenths_operand(w[threadIdx.x]);
    out[threadIdx.x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf16, a), __builtin_bit_cast(v8bf16, b), c, 0, 0, 0);
}
"""


def registers(text):
    out = set()
    for m in re.finditer(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= set(range(int(m.group(1)), int(m.group(2)) + 1)) if m.group(1) else {int(m.group(3))}
    return out


def least_distance(lines):
    """Wait states between a vector instruction's write and a matrix instruction that reads it: the least."""
    wrote, now, least = {}, 0, None
    for line in lines:
        name, _, ops = re.sub(r"[;/].*", "", line).strip().partition(" ")
        if name == "s_nop":
            now += int(ops, 0) + 1
        elif name.startswith("v_mfma"):
            now += 1
            read = registers(",".join(ops.split(",")[1:3]))
            least = min([now - 1 - wrote[r] for r in read if r in wrote] + ([] if least is None else [least]), default=None)
        elif re.match(r"[a-z]\w+$", name):
            now += 1
            if name.startswith("v_"):
                wrote.update({r: now for r in registers(ops.split(",")[0])})
    return least


def test_the_reader_of_code():
    code = ["v_perm_b32 v7, v1, v2, s0", "v_mov_b32 v9, v8", "v_mfma_f32_16x16x32_bf16 v[0:3], v[10:13], v[4:7], v[0:3]"]
    assert least_distance(code) == 1
    assert least_distance(code[:1] + ["s_nop 1"] + code[2:]) == 2
    assert least_distance(code[1:]) is None


def test_two_wait_states_before_the_matrix_instruction(tmp_path):
    (tmp_path / "product.hip").write_text(KERNEL)
    out = tmp_path / "product.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I", os.path.join(ROOT, "include"), "-I", CSRC, "--cuda-device-only", "-S", str(tmp_path / "product.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert "v_cvt_off_f32_i4" in text and "v_mfma" in text
    assert least_distance(text.splitlines()) >= 2


def test_the_kernels_use_it():
    with open(os.path.join(CSRC, "w4.hip")) as f:
        src = f.read()
    assert "int4_sixteenths<" not in src and "int4_sixteenths_operand(" in src
