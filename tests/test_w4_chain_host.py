"""Host-side check of the INT4 tiles' group sums (no GPU needed): the loop that adds a
chain's 16 values beside the next chain's matrix instructions, compiled from the kernel's
own bounds with every access checked."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd-kernels_amd", "csrc")

PROGRAM = """
#include <cstdio>
#include <vector>
#include "w4_chain.h"
int main() {
    for (int ch : {2, 4, 8}) {
        std::vector<int> added(16, 0);
        for (int s = 0; s < ch; ++s)
            for (int e = hkq::chain_added(s, ch); e < hkq::chain_added(s + 1, ch); ++e) {
                if (s == 0) return std::printf("chains of %d: value %d beside the first instruction", ch, e), 1;
                added.at(e)++;
            }
        for (int e = 0; e < 16; ++e)
            if (added[e] != 1) return std::printf("chains of %d: value %d added %d times", ch, e, added[e]), 1;
    }
}
"""


def test_each_value_of_a_chain_is_added_once(tmp_path):
    with open(os.path.join(CSRC, "w4_tile.hip")) as f:
        src = f.read()
    assert "e = chain_added(s % CH, CH); e < chain_added(s % CH + 1, CH)" in src, "the kernel's loop has other bounds"
    (tmp_path / "chain.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "chain")
    subprocess.run(["g++", "-std=c++17", "-O0", "-I", CSRC, str(tmp_path / "chain.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
