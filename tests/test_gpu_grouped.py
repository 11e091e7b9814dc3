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


def test_many_groups():
    """More groups than the table of the streaming kernels holds, and than one wave scans."""
    require_gpu()
    check([2, 0, 1] * 210, 256, 256, seed=3)
    check([0] * 700 + [300] + [0] * 100 + [290], 512, 640, seed=4)


def test_bounds_outside_the_rows():
    """Bounds below 0 and above M count as 0 and M, decreasing ones as empty groups."""
    require_gpu()
    M, N, K = 64, 40, 72
    X, W = bf16((M, K), 1).cuda(), bf16((3, N, K), 2).cuda()
    Y = torch.full((M, N), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_bf16(X, W, torch.tensor([-5, 10, 50, 1000], dtype=torch.int32, device="cuda"), Y)
    for e, r in enumerate((slice(0, 10), slice(10, 50), slice(50, 64))):
        x, w = X[r].double(), W[e].double()
        close(Y[r], x @ w.t(), x.abs() @ w.abs().t(), K, f"group {e}")
    Y.fill_(7.0)
    hkq.grouped_gemm_bf16(X, W, torch.tensor([40, 20, 20, 60], dtype=torch.int32, device="cuda"), Y)
    x, w = X[20:60].double(), W[2].double()
    close(Y[20:60], x @ w.t(), x.abs() @ w.abs().t(), K, "last group")
    assert (Y[:20] == 7.0).all() and (Y[60:] == 7.0).all()


def test_no_rows_no_sums():
    require_gpu()
    W, offs = bf16((3, 16, 24), 1).cuda(), torch.zeros(4, dtype=torch.int32, device="cuda")
    X, dY = torch.empty((0, 24), dtype=BF16, device="cuda"), torch.empty((0, 16), dtype=BF16, device="cuda")
    assert hkq.grouped_gemm_bf16(X, W, offs).shape == (0, 16)
    dX, dW = hkq.grouped_gemm_backward(dY, X, W, offs, dW=torch.full_like(W, 7.0))
    assert dX.shape == (0, 24) and (dW == 0).all()
    # K = 0: empty sums
    X, W = torch.empty((5, 0), dtype=BF16, device="cuda"), torch.empty((2, 16, 0), dtype=BF16, device="cuda")
    offs = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    Y = hkq.grouped_gemm_bf16(X, W, offs, torch.full((5, 16), 7.0, dtype=BF16, device="cuda"))
    assert (Y[:4] == 0).all() and (Y[4] == 7.0).all()


def test_only_one_gradient():
    require_gpu()
    X, W, dY = bf16((50, 64), 1).cuda(), bf16((2, 32, 64), 2).cuda(), bf16((50, 32), 3).cuda()
    offs = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    dX, dW = hkq.grouped_gemm_backward(dY, X, W, offs)
    a, none = hkq.grouped_gemm_backward(dY, X, W, offs, need_dw=False)
    assert none is None and torch.equal(a, dX)
    none, b = hkq.grouped_gemm_backward(dY, X, W, offs, need_dx=False)
    assert none is None and torch.equal(b, dW)


def test_weights_of_other_layouts():
    """Groups side by side in each row, and one weight for all groups (group stride 0)."""
    require_gpu()
    E, N, K, rows = 3, 48, 80, [40, 0, 90]
    offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
    X, dY = bf16((130, K), 1).cuda(), bf16((130, N), 2).cuda()
    W = bf16((N, E, K), 3).cuda()
    dWb = torch.full((N, E, K), 7.0, dtype=BF16, device="cuda")
    ref = hkq.grouped_gemm_bf16(X, W.transpose(0, 1).contiguous(), offs)
    assert torch.equal(hkq.grouped_gemm_bf16(X, W.transpose(0, 1), offs), ref)
    dx, dw = hkq.grouped_gemm_backward(dY, X, W.transpose(0, 1).contiguous(), offs)
    dx2, dw2 = hkq.grouped_gemm_backward(dY, X, W.transpose(0, 1), offs, dW=dWb.transpose(0, 1))
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    one = W[:, 0].contiguous()
    Y = hkq.grouped_gemm_bf16(X, one[None].expand(E, N, K), offs)
    x, w = X.double(), one.double()
    close(Y, x @ w.t(), x.abs() @ w.abs().t(), K, "one weight")


def test_nan_and_infinity_stay_in_their_rows():
    require_gpu()
    rows, N, K = [70, 130], 136, 200
    offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
    X, W, dY = bf16((200, K), 1).cuda(), bf16((2, N, K), 2).cuda(), bf16((200, N), 3).cuda()
    clean = hkq.grouped_gemm_bf16(X, W, offs)
    X[3, 199], X[150, 0], X[151, 7] = float("nan"), float("inf"), -float("inf")
    Y = hkq.grouped_gemm_bf16(X, W, offs)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[3, 150, 151]] = True
    assert torch.equal(Y[~bad], clean[~bad]) and not Y[bad].isfinite().any()
    assert torch.equal(Y[150].isnan(), (W[1, :, 0] == 0)) and torch.equal(Y[151] > 0, W[1, :, 7] < 0)
    _, dW = hkq.grouped_gemm_backward(dY, X, W, offs, need_dx=False)
    hit = torch.zeros((2, K), dtype=torch.bool, device="cuda")
    hit[0, 199], hit[1, 0], hit[1, 7] = True, True, True
    assert torch.equal(~dW.isfinite(), hit[:, None, :].expand(2, N, K))


def test_gradients_against_differences():
    """Whole numbers small enough that every sum is exact in bf16 (at most 256): the products are linear, so differences
    of the outputs are the gradients' products with the step, with nothing lost."""
    require_gpu()
    rows, N, K = [3, 0, 5, 8], 16, 8
    offs, M = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda"), sum(rows)

    def ints(shape, seed, top):
        return torch.randint(-top, top + 1, shape, generator=gen(seed)).to(BF16).cuda()

    X, W, dY = ints((M, K), 1, 3), ints((4, N, K), 2, 3), ints((M, N), 3, 1)
    dX, dW = hkq.grouped_gemm_backward(dY, X, W, offs)

    def loss(x, w):
        return float((hkq.grouped_gemm_bf16(x, w, offs).double() * dY.double()).sum())

    base = loss(X, W)
    for seed in range(8):
        sx, sw = ints((M, K), 10 + seed, 1), ints((4, N, K), 30 + seed, 1)
        assert loss(X + sx, W) - base == float((dX.double() * sx.double()).sum())
        assert loss(X, W + sw) - base == float((dW.double() * sw.double()).sum())


def test_offsets_past_32_bits():
    """Weights and their gradient of 5.4 GB, rows of 2.4 GB."""
    require_gpu()
    E, N, K = 40, 8192, 8192
    W = torch.zeros((E, N, K), dtype=BF16, device="cuda")
    W[0], W[-1] = bf16((N, K), 1, 0.01).cuda(), bf16((N, K), 2, 0.01).cuda()
    rows = [5] + [0] * (E - 2) + [70]
    offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
    X, dY = bf16((75, K), 3).cuda(), bf16((75, N), 4).cuda()
    Y = hkq.grouped_gemm_bf16(X, W, offs)
    dX, dW = hkq.grouped_gemm_backward(dY, X, W, offs)
    for e, r in ((0, slice(0, 5)), (E - 1, slice(5, 75))):
        x, dy, w = X[r].double(), dY[r].double(), W[e].double()
        close(Y[r], x @ w.t(), x.abs() @ w.abs().t(), K, "Y")
        close(dX[r], dy @ w, dy.abs() @ w.abs(), N, "dX")
        close(dW[e], dy.t() @ x, dy.abs().t() @ x.abs(), 70, "dW")
    assert (dW[1:-1] == 0).all()
    del W, dW
    M, K, N = 300000, 4096, 4096
    X = torch.zeros((M, K), dtype=BF16, device="cuda")
    X[-300:] = bf16((300, K), 5).cuda()
    W = bf16((2, N, K), 6, 0.01).cuda()
    offs = torch.tensor([0, 10, M], dtype=torch.int32, device="cuda")
    Y = hkq.grouped_gemm_bf16(X, W, offs)
    x, w = X[-300:].double(), W[1].double()
    close(Y[-300:], x @ w.t(), x.abs() @ w.abs().t(), K, "last rows")
    assert (Y[:-300] == 0).all()
    dX, dW = hkq.grouped_gemm_backward(Y, X, W, offs)
    dy = Y[-300:].double()
    close(dX[-300:], dy @ w, dy.abs() @ w.abs(), N, "dX of the last rows")
    close(dW[1], dy.t() @ x, dy.abs().t() @ x.abs(), M, "dW over the last rows")


def test_streams_and_graphs():
    """On a stream of the caller's, two at once, and captured: every replay as the eager call, with eager work between."""
    require_gpu()
    sizes = [([40, 0, 3, 200], 264, 200), ([600, 700], 512, 256), ([3, 4, 1, 0], 1408, 2048)]
    sets = []
    for i, (rows, N, K) in enumerate(sizes):
        M = sum(rows)
        offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
        sets.append((bf16((M, K), i).cuda(), bf16((len(rows), N, K), i + 10).cuda(), bf16((M, N), i + 20).cuda(), offs))

    def run(x, w, dy, offs, stream=None):
        y = hkq.grouped_gemm_bf16(x, w, offs, stream=stream)
        return (y, *hkq.grouped_gemm_backward(dy, x, w, offs, stream=stream))

    eager = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        out = [run(*s, stream=st) for s, st in zip(sets, streams)]
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = [run(*s) for s in sets]
    for _ in range(3):
        for o in out:
            for t in o:
                t.fill_(3.0)
        g.replay()
        run(*sets[0])
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    # other rows in the captured call's bounds: they are read at each replay
    sets[0][3].copy_(torch.tensor([0, 100, 100, 243, 243], dtype=torch.int32))
    eager = run(*sets[0])
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(eager, out[0]))


def test_hipkittens_module():
    require_gpu()
    import hipkittens as hk

    rows, N, K = [40, 0, 90], 48, 80
    offs = torch.tensor(bounds(rows), dtype=torch.int32, device="cuda")
    X, W, dY = bf16((130, K), 1).cuda(), bf16((3, N, K), 2).cuda(), bf16((130, N), 3).cuda()
    Y, dX, dW = torch.empty_like(dY), torch.empty_like(X), torch.empty_like(W)
    hk.moe.grouped.grouped_gemm_bf16(X, W, Y, offs)
    hk.moe.grouped.grouped_gemm_backward(dY, X, W, offs, dX, dW)
    ref = hkq.grouped_gemm_backward(dY, X, W, offs)
    assert torch.equal(Y, hkq.grouped_gemm_bf16(X, W, offs)) and torch.equal(dX, ref[0]) and torch.equal(dW, ref[1])
    with pytest.raises(ValueError, match="offs"):
        hk.moe.grouped.grouped_gemm_bf16(X, W, Y, offs[:2])
    with pytest.raises(TypeError, match="X"):
        hk.moe.grouped.grouped_gemm_bf16(X.float(), W, Y, offs)
    with pytest.raises(RuntimeError, match="overlap"):
        hk.moe.grouped.grouped_gemm_bf16(X[:, :48], W[:, :, :48], X[:, :48], offs)


def test_mixture_layer_trained_and_served():
    """A mixture layer as it is used: the router's bounds and order, gate and up projections, activation, down projection
    and the sum over a token's experts, with all gradients; then the same layer served with its weights in 4 bits. Against
    the formulas in 64 bits of the same (rounded) steps; tolerances: 2-norms, U per rounding of an intermediate (the
    activation's inputs and output, its gradients), of which at most six stand in one chain."""
    require_gpu()
    T, D, F, E, topk = 203, 512, 384, 8, 2
    x = bf16((T, D), 1).cuda()
    W1, W2 = bf16((E, 2 * F, D), 2, D ** -0.5).cuda(), bf16((E, D, F), 3, F ** -0.5).cuda()
    logits = bf16((T, E), 4, 2.0).cuda()
    r = hkq.moe_routing(logits, topk)
    offs, gather = r["token_start"], r["gather"]
    token, gate = gather.long() // topk, r["gate_scal"].double()
    xs = x[token]
    y1 = hkq.grouped_gemm_bf16(xs, W1, offs)

    def act(y):
        g, u = y[:, :F], y[:, F:]
        return g * torch.sigmoid(g) * u

    h = act(y1.float()).to(BF16)
    y2 = hkq.grouped_gemm_bf16(h, W2, offs)
    out = torch.zeros((T, D), dtype=torch.float64, device="cuda").index_add_(0, token, y2.double() * gate[:, None])
    dout = bf16((T, D), 5).cuda()
    dy2 = (dout[token].double() * gate[:, None]).to(BF16)
    dh, dW2 = hkq.grouped_gemm_backward(dy2, h, W2, offs)
    yf = y1.float().requires_grad_()
    dy1 = torch.autograd.grad(act(yf), yf, dh.float())[0].to(BF16)
    dxs, dW1 = hkq.grouped_gemm_backward(dy1, xs, W1, offs)
    # 64 bits, from x to the loss sum(out * dout)
    X, A, B = (t.double().requires_grad_() for t in (x, W1, W2))
    o = offs.tolist()
    ref = torch.zeros((T, D), dtype=torch.float64, device="cuda")
    for e in range(E):
        rows = slice(o[e], o[e + 1])
        ref = ref.index_add(0, token[rows], (act(X[token[rows]] @ A[e].t()) @ B[e].t()) * gate[rows, None])
    gx, g1, g2 = torch.autograd.grad((ref * dout.double()).sum(), (X, A, B))
    dx = torch.zeros((T, D), dtype=torch.float64, device="cuda").index_add_(0, token, dxs.double())

    def near(a, b, what, n=6):
        off = float((a.double() - b).norm() / b.norm())
        assert off <= n * U, f"{what}: {off}"

    near(out, ref.detach(), "output")
    near(dW2, g2, "dW2")
    near(dW1, g1, "dW1")
    near(dx, gx, "dx")
    # served: rows fetched through the router's order, weights in 4 bits with zero points
    (q1, s1, z1), (q2, s2, z2) = hkq.w4_quant(W1, 64, zeros=True), hkq.w4_quant(W2, 64, zeros=True)
    h4 = act(hkq.grouped_gemm_w4a16(x, q1, s1, offs, z1, gather, topk).float()).to(BF16)
    y4 = hkq.grouped_gemm_w4a16(h4, q2, s2, offs, z2)

    def values(q, s, z):
        c = torch.stack((q & 15, q >> 4), -1).flatten(-2).double().view(*s.shape, 64)
        return ((c - z.double()[..., None]) * s.double()[..., None]).flatten(-2)

    A4, B4 = values(q1, s1, z1), values(q2, s2, z2)
    for e in range(E):
        rows = slice(o[e], o[e + 1])
        ref4 = act(x.double()[token[rows]] @ A4[e].t()) @ B4[e].t()
        if rows.stop > rows.start:
            near(y4[rows], ref4, f"served group {e}", 4)
