"""GPU tests of the products over ragged groups of rows at sizes that reach their
256 x 256 tiles: the streams of tiles (sums over whole pairs of K-tiles, up to 512
groups) and the tiles by themselves (other sums, or more groups), in Y and in dX, with
data in several groups, ragged columns, sums that end inside a K-tile, and NaN in the
rows beside the groups and behind each row. Definitions and tolerances are those of
test_gpu_grouped.py.
"""
import pytest
import torch

import hkq
from gpu_util import require_gpu
from test_gpu_grouped import BF16, bf16, bounds, check

pytestmark = pytest.mark.gpu

# rows of the groups (72 more belong to none) and, for Y, columns and the sums' length
STREAMS = [([700, 0, 300, 1, 537], 7328, 384),  # 261 tiles: one each on 256 CUs, five as halves
           ([300, 1, 0, 257, 64, 180, 128], 8600, 512),  # 16 as halves; row tiles of 1, 44, 64 and 128 rows
           ([1700, 1200, 2028], 6664, 1024),  # two each, 28 as halves
           ([1700, 0, 1200, 1500], 6664, 1024)]  # 486: the last round whole
WHOLE = [([640, 0, 300, 1, 64, 17, 256], 7304, 392), ([300, 1, 0, 257, 64, 180, 70], 8568, 520), ([100, 130, 0, 257, 1, 31, 2], 8760, 1064)]


@pytest.mark.parametrize("rows,N,K", STREAMS + WHOLE, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}x{max(v)}")
def test_large_tiles(rows, N, K):
    require_gpu()
    check(rows, N, K, first=5, tail=67, pad=8, seed=K)  # Y
    check(rows, K, N, first=5, tail=67, pad=8, seed=N)  # dX


def test_large_tiles_of_many_groups():
    """More groups than the streams' table holds, on tiles by themselves."""
    require_gpu()
    rows = [180 + 7 * (e % 13) if e % 5 else 0 for e in range(512)]
    check(rows + [116389 - 72 - sum(rows)], 240, 1024, first=5, tail=67, seed=9)


@pytest.mark.parametrize("rows,N,K", [STREAMS[2], STREAMS[3], ([1024] * 8, 14336, 2048)], ids=["halves", "whole", "layer"])
def test_the_same_bits_each_time(rows, N, K):
    """Nothing about the order of the sums is left to chance: the bits of the first call in every later one, eager and
    replayed, with other work on another stream meanwhile."""
    require_gpu()
    M, E = sum(rows), len(rows)
    offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
    X, dY, W = bf16((M, K), 1).cuda(), bf16((M, N), 2).cuda(), bf16((E, N, K), 3, K ** -0.5).cuda()

    def run():
        return (hkq.grouped_gemm_bf16(X, W, offs), *hkq.grouped_gemm_backward(dY, X, W, offs))

    first = run()
    side, other = torch.cuda.Stream(), torch.ones(1 << 24, device="cuda")
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(side):
            for _ in range(8):
                other.mul_(1.0)
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for _ in range(3):
        for t in out:
            t.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_nan_and_infinity_stay_in_their_rows():
    """In a stream of tiles: an infinity and a NaN in one group's rows, each output beside theirs as without them."""
    require_gpu()
    rows, N, K = STREAMS[3]
    offs, M = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda"), sum(rows)
    X, W, dY = bf16((M, K), 1).cuda(), bf16((len(rows), N, K), 2).cuda(), bf16((M, N), 3).cuda()
    clean = hkq.grouped_gemm_bf16(X, W, offs)
    _, grad = hkq.grouped_gemm_backward(dY, X, W, offs, need_dx=False)
    X[1699, K - 1], X[1700, 0], X[3000, 7] = float("nan"), float("inf"), -float("inf")
    Y = hkq.grouped_gemm_bf16(X, W, offs)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[1699, 1700, 3000]] = True
    assert torch.equal(Y[~bad], clean[~bad]) and not Y[bad].isfinite().any()
    _, dW = hkq.grouped_gemm_backward(dY, X, W, offs, need_dx=False)
    hit = torch.zeros((len(rows), K), dtype=torch.bool, device="cuda")
    hit[0, K - 1], hit[2, 0], hit[3, 7] = True, True, True
    hit = hit[:, None, :].expand_as(dW)
    assert torch.equal(~dW.isfinite(), hit) and torch.equal(dW[~hit], grad[~hit])
    assert (dW[1] == 0).all() and dW.dtype == BF16
