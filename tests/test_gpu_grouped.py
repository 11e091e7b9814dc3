"""GPU tests of the products over ragged groups of rows and their gradients
against their definitions in 64 bits.

Tolerances, from the arithmetic (U: half a step of bf16 relative to the value,
2^-8; E: 2^-23, a step of fp32): a sum of K products in fp32 is off by at most
K E sum|products| in any order, the rounding to bf16 adds U |value|. Worst cases
add up with one sign; real errors do not, so the 2-norm of a whole output's error
is held to U as well.
"""
import pytest
import torch

import hkq
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

U, E32 = 2.0 ** -8, 2.0 ** -23
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(shape, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed)) * std).to(BF16)


def close(got, ref, mag, terms, what):
    """got against ref: sums of `terms` products whose absolute values add up to mag."""
    got = got.double()
    tol = U * ref.abs() + terms * E32 * mag + 1e-38
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {got[i]} ref {ref[i]} tol {tol[i]}")
    if ref.numel() >= 1024 and float(ref.norm()) > 0:
        assert float((got - ref).norm() / ref.norm()) <= U, what


def bounds(rows, first=0):
    o = [first]
    for r in rows:
        o.append(o[-1] + r)
    return o


def check(rows, N, K, first=0, tail=0, pad=0, seed=0):
    """Forward and both gradients with `first` rows before and `tail` rows behind the groups, rows `pad` values longer than
    they need be, everything that no product may use a NaN."""
    o = bounds(rows, first)
    M, E = o[-1] + tail, len(rows)
    nan = float("nan")

    def operand(shape, seed, std):
        t = torch.full((*shape[:-1], shape[-1] + pad), nan, dtype=BF16, device="cuda")
        v = t[..., :shape[-1]]
        v.copy_(bf16(shape, seed, std))
        return v

    X, dY, W = operand((M, K), seed, 1.0), operand((M, N), seed + 1, 1.0), operand((E, N, K), seed + 2, K ** -0.5)
    for t in (X, dY):
        t[:first] = nan
        t[o[-1]:] = nan
    offs = torch.tensor(o, dtype=torch.int32, device="cuda")

    def out(shape):
        t = torch.full((*shape[:-1], shape[-1] + pad), 7.0, dtype=BF16, device="cuda")
        return t, t[..., :shape[-1]]

    (yb, Y), (xb, dX), (wb, dW) = out((M, N)), out((M, K)), out((E, N, K))
    assert hkq.grouped_gemm_bf16(X, W, offs, Y) is Y
    got = hkq.grouped_gemm_backward(dY, X, W, offs, dX, dW)
    assert got[0] is dX and got[1] is dW
    for b, t in ((yb, Y), (xb, dX), (wb, dW)):
        assert (b[..., t.shape[-1]:] == 7.0).all(), "columns past the output written"
    for t in (Y, dX):
        assert (t[:first] == 7.0).all() and (t[o[-1]:] == 7.0).all(), "rows of no group written"
    for e in range(E):
        r = slice(o[e], o[e + 1])
        x, dy, w = X[r].double().contiguous(), dY[r].double().contiguous(), W[e].double().contiguous()
        what = f"group {e} of rows {rows}, N {N}, K {K}"
        close(Y[r], x @ w.t(), x.abs() @ w.abs().t(), K, "Y, " + what)
        close(dX[r], dy @ w, dy.abs() @ w.abs(), N, "dX, " + what)
        close(dW[e], dy.t() @ x, dy.abs().t() @ x.abs(), max(1, rows[e]), "dW, " + what)


# rows of each group: none, one, tile sizes and their neighbours, skewed, many groups (past one wave's 64)
ROWS = [[1], [0, 1, 0], [3, 0, 5, 1], [64, 63, 65, 0], [127, 128, 129], [300, 0, 1, 255], [600, 257], [1000, 1, 1, 1, 1, 1, 1, 1],
        [2] * 70 + [0] * 60 + [33, 1], [90] * 9]


@pytest.mark.parametrize("rows", ROWS, ids=lambda r: f"{len(r)}x{max(r)}")
@pytest.mark.parametrize("N,K", [(8, 8), (72, 136), (264, 520), (1408, 64), (384, 1000)])
def test_products_and_gradients(rows, N, K):
    require_gpu()
    check(rows, N, K, seed=sum(rows) + N + K)


@pytest.mark.parametrize("rows", [[3, 0, 70], [130, 0, 300, 1], [1, 1]])
def test_rows_of_no_group_and_padded_pitches(rows):
    require_gpu()
    check(rows, 200, 328, first=5, tail=67, pad=8, seed=11)
    check(rows, 520, 72, first=0, tail=300, pad=24, seed=12)


@pytest.mark.parametrize("rows,N,K", [([700, 900, 500, 30], 2816, 2048), ([94] * 16, 2048, 1408), ([6, 9, 3, 0, 11, 7, 1, 9], 4096, 3584),
                                      ([40] * 8, 4096, 4096), ([2000, 2096], 4096, 1024)])
def test_layer_sizes(rows, N, K):
    require_gpu()
    check(rows, N, K, seed=5)
