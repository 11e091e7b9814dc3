"""Host-side check (no GPU needed) of the scan that finds a workgroup's group, on bounds
whose tile counts pass 32 bits: the same steps in Python, sums held at the largest int as
the kernels hold them."""
import os

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd-kernels_amd", "csrc")
TOP = 2 ** 31 - 1


def wrap(v):
    return (v + 2 ** 31) % 2 ** 32 - 2 ** 31


def find(counts, tiles_m, at, add):
    """(group, its first tile) of row tile `at`, None past the last; `add` adds two ints."""
    total = 0
    for n in counts:
        total = add(total, n)
    if at >= min(total, tiles_m):
        return None
    before = 0
    for e, n in enumerate(counts):
        if add(before, n) > at:
            return e, before
        before = add(before, n)


def test_every_tile_of_the_grid_has_its_group():
    most = (1 << 22) // 64 + 1
    counts = [most, 0] * 32768
    for at in (0, 1, most - 1, most, 3 * most - 1):
        got = find(counts, 4 * most, at, lambda a, b: min(a + b, TOP))
        assert got == (at // most * 2, at // most * most)
        assert find(counts, 4 * most, at, lambda a, b: wrap(a + b)) is None  # what wrapped sums made of it


def test_the_kernels_hold_their_sums():
    with open(os.path.join(CSRC, "ragged.h")) as f:
        src = f.read()
    scan = src[src.index("bool ragged_tile("):src.index("ragged_most")]
    assert "__builtin_elementwise_add_sat" in src
    assert "+=" not in scan.replace("d *= 2", "").replace("e0 += 64", "") and "before + s >" not in scan
