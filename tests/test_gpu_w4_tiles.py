"""GPU tests of the products with 4-bit weights at sizes that reach each tile of many
rows, for each kind of weight, and of INT4 groups of 64 without zero points. Definitions
and tolerances are those of test_gpu_w4.py.
"""
import pytest
import torch

import hkq
from gpu_util import require_gpu
from test_gpu_w4 import KINDS, NAN, check_dense, check_grouped, rows_of, weights

pytestmark = pytest.mark.gpu

SIXTY_FOUR = ("int4", 64, False)
ALL = KINDS + [SIXTY_FOUR]

# tile, rows, columns and the sums' length (the multiple of a group below it): the last row and column tiles are ragged,
# and where groups allow it the sums end inside a unit of 128 values
DENSE = [("32x128", 33, 3449, 544), ("64x128", 33, 16683, 1056), ("64x256", 130, 16532, 1568), ("96x256", 131, 16765, 544),
         ("128x128", 66, 22327, 544), ("128x256", 194, 21780, 544)]
GROUPED = [("32x128", [36, 1], 101, 544), ("64x128", [40, 0, 30, 1, 20, 12], 5130, 1056), ("96x256", [40, 0, 3, 50, 1, 20, 10], 9020, 544),
           ("128x128", [100, 0, 1, 85], 7821, 544), ("128x256", [129, 0, 70, 7], 15451, 544)]


@pytest.mark.parametrize("kind,group,zeros", ALL)
@pytest.mark.parametrize("tile,M,N,K", DENSE, ids=[t[0] for t in DENSE])
def test_dense_tiles(tile, M, N, K, kind, group, zeros):
    require_gpu()
    check_dense(M, N, K // group * group, kind, group, zeros, pad=3, seed=M)


@pytest.mark.parametrize("kind,group,zeros", ALL)
@pytest.mark.parametrize("tile,rows,N,K", GROUPED, ids=[t[0] for t in GROUPED])
def test_grouped_tiles(tile, rows, N, K, kind, group, zeros):
    """As a layer's down projection (rows as they lie) and as its up projection (rows through the router's order)."""
    require_gpu()
    K = K // group * group
    check_grouped(rows, N, K, kind, group, zeros, pad=1, seed=7)
    check_grouped(rows, N, K, kind, group, zeros, topk=3, seed=8)


@pytest.mark.parametrize("kind,group,zeros", ALL)
def test_grouped_tiles_of_64_by_256(kind, group, zeros):
    require_gpu()
    rows = [(e * 37) % 41 for e in range(226)]
    check_grouped(rows + [4733 - sum(rows)], 129, 1568 // group * group, kind, group, zeros, seed=9)


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 40, 64, 65, 130, 300])
def test_groups_of_64_without_zero_points(M):
    require_gpu()
    for N, K in ((1, 64), (33, 192), (200, 1408), (64, 4096), (1000, 640), (13001, 576)):
        check_dense(M, N, K, *SIXTY_FOUR, seed=M + N)
    for i in range(1, 8):
        check_dense(M, 70, i * 64, *SIXTY_FOUR, pad=i, seed=i)


@pytest.mark.parametrize("rows", [[1], [0, 1, 0, 1], [5, 0, 17, 16, 1], [64, 65, 3], [200, 0, 130], [2] * 70 + [0] * 60 + [40],
                                  [700, 1, 1, 1, 0, 90], [94] * 16, [6, 9, 3, 0, 11, 7, 1, 9]], ids=lambda r: f"{len(r)}x{max(r)}")
def test_grouped_by_64_without_zero_points(rows):
    require_gpu()
    check_grouped(rows, 72, 320, *SIXTY_FOUR, topk=3, seed=1)
    check_grouped(rows, 2816, 448, *SIXTY_FOUR, first=3, tail=20, pad=2, seed=2)


@pytest.mark.parametrize("M", [3, 200])
def test_infinity_nan_and_zero_by_64_without_zero_points(M):
    require_gpu()
    q, s, _, val = weights((70, 256), *SIXTY_FOUR, 5)
    q[9], val[9] = 0x88, 0
    X = rows_of(M, 256, 6)
    clean = hkq.gemm_w4a16(X, q, s)
    assert (clean[:, 9] == 0).all()
    X[M - 1, 67] = float("inf")
    C = hkq.gemm_w4a16(X, q, s)
    v = val[:, 67]
    assert torch.equal(C[:-1], clean[:-1])
    assert torch.equal(C[-1].isnan(), v == 0) and torch.equal(C[-1][v != 0] > 0, v[v != 0] > 0) and not C[-1].isfinite().any()
    X[M - 1, 67] = NAN
    assert hkq.gemm_w4a16(X, q, s)[-1].isnan().all()
