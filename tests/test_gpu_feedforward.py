"""GPU tests of the feed-forward layer's operators against their definitions in
64 bits: residual addition + RMSNorm + quantization, products with a fused
epilogue, the gated projection pair and its backward pass.

Tolerances, from the arithmetic (U: half a step of bf16 relative to the value,
2^-8; E: 2^-23, a step of fp32):
* a sum of K products in fp32 is off by at most K E sum|products|, in any order;
* an activation moves by at most 1.13 times its argument (the largest slope of
  SiLU and GELU, with alpha <= 1.13), and its own evaluation by 2^-19 |v| (exp2
  and rcp to a few steps, the argument's rounding times the slope; GELU's
  formula to 1.5e-7);
* each rounding to bf16 adds U |value|;
* the FP8 matrix instruction adds 16 neighbouring products after cutting off what
  lies below 2^-13 of the largest of them (test_fp8_products_alignment: a product
  2^-13 of its neighbour counts, one of 2^-14 is lost, one outside the 16 is not):
  each of the 16 is off by less than 2^-13 of that largest product, which is at
  most the largest |a| times the largest |b| of the 16.
Worst cases add up with one sign. Real errors do not, so the 2-norm of a whole
output's error is held to U per rounding of it as well (a rounding's own 2-norm
is 0.43 U, the FP8 instruction's share a tenth of that).
"""
import math

import pytest
import torch

import hkq
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -23
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
ACTS = ["none", "relu", "silu", "gelu_tanh", "gelu"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(shape, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed)) * std).to(BF16)


def fp8(shape, seed):
    """E4M3FN codes of normal values and positive scales per row."""
    q = (torch.randn(shape, generator=gen(seed)) * 100.0).clamp(-448, 448).to(FP8)
    return q, 0.5 + torch.rand(shape[0], generator=gen(seed + 1))


def act64(v, name, alpha=1.0):
    """(value, slope) in float64."""
    if name == "none":
        return v, torch.ones_like(v)
    if name == "relu":
        return v.clamp_min(0), (v > 0).double()
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return v * phi, phi + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        z, dz = alpha * v, torch.full_like(v, alpha)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        z, dz = c * (v + 0.044715 * v ** 3), c * (1 + 3 * 0.044715 * v ** 2)
    s = torch.sigmoid(z)
    return v * s, s + v * s * (1 - s) * dz


def close(got, ref, tol, what, roundings=1):
    got = got.detach().double().to(ref.device)
    assert got.shape == ref.shape, f"{what}: {got.shape} vs {ref.shape}"
    if roundings and ref.numel() >= 1024:  # enough values for a norm to say something
        off = float(torch.linalg.norm(got - ref) / torch.linalg.norm(ref))
        assert off <= roundings * U, f"{what}: 2-norm of the error {off} of the result's"
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {got[i]} "
                             f"ref {ref[i]} tol {tol[i]}")


def guarded(M, N, ld, dtype=BF16, fill=7.0, device="cuda"):
    """(whole buffer of M + 2 rows of ld filled with `fill`, view of its rows 1 .. M, N columns)."""
    buf = torch.full((M + 2, ld), fill, device=device).to(dtype)
    return buf, buf[1:M + 1, :N]


def untouched(buf, M, N, fill=7.0):
    b = buf.float()
    assert (b[0] == fill).all() and (b[M + 1] == fill).all(), "rows around the output written"
    assert (b[1:M + 1, N:] == fill).all(), "columns past the output written"


# ------------------------------------------------------- residual + norm + quantization

def norm_ref(x, res, w, eps, group, qmax):
    h = x if res is None else (x.float() + res.float()).to(BF16)
    v = h.double()
    y = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w.double()
    g = y.view(y.shape[0], -1, group or y.shape[1])
    s = (g.abs().amax(2) / qmax).clamp_min(1e-10)
    return h, y, s, (g / s[:, :, None]).view(y.shape)


def check_norm(x, res, w, eps, group, kind, q, s, h):
    qmax = 448.0 if kind == hkq.KIND_FP8 else 127.0
    M, D = x.shape
    rh, y, rs, rq = norm_ref(x, res, w, eps, group, qmax)
    if res is not None:
        assert torch.equal(h.cpu().view(torch.int16), rh.view(torch.int16)), "h"
    # the fp32 sum of squares is off by D E relative at most, its root by half
    # of that, and seven further roundings reach s and the codes' argument
    slack = (D / 2 + 8) * E
    s = s.cpu().double().view(rs.shape)
    assert ((s - rs).abs() <= slack * rs).all(), "scales"
    q = q.cpu().float().double()
    if kind == hkq.KIND_FP8:  # half a step of e4m3: 2^-4 of the value, 2^-10 among the subnormal codes
        tol = torch.maximum(rq.abs() * 2.0 ** -4, torch.full_like(rq, 2.0 ** -10)) + 2 * slack * rq.abs()
    else:
        tol = torch.full_like(rq, 0.5) + 2 * slack * rq.abs()
    close(q, rq, tol, "codes", roundings=0)


@pytest.mark.parametrize("kind", [hkq.KIND_FP8, hkq.KIND_INT8])
@pytest.mark.parametrize("M,D,group,residual", [
    (1, 8, 0, True), (3, 40, 0, True), (5, 512, 128, True), (4, 520, 0, False), (9, 1024, 128, True), (7, 2048, 0, True),
    (2, 2056, 0, True), (6, 2176, 128, False), (33, 4096, 0, True), (5, 4096, 128, True), (3, 4104, 0, True),
    (17, 7168, 128, True), (4, 8192, 0, False), (3, 8200, 0, True), (2, 16384, 0, True), (2, 16384, 128, True)])
def test_add_rmsnorm_quant(kind, M, D, group, residual):
    require_gpu()
    x, w = bf16((M, D), M + D, 1.5), (1 + 0.2 * torch.randn(D, generator=gen(D))).to(BF16)
    res = bf16((M, D), M + D + 1, 2.0) if residual else None
    if M > 2:
        x[1] = 0
        if residual:
            res[1] = 0  # a row of zeros: scale 1e-10, codes 0
    q, s, h = hkq.add_rmsnorm_quant(x.cuda(), w.cuda(), None if res is None else res.cuda(), 1e-5, kind, group)
    torch.cuda.synchronize()
    assert (h is None) == (res is None)
    check_norm(x, res, w, 1e-5, group, kind, q, s, h)


def test_add_rmsnorm_quant_strides_in_place_and_neighbours():
    """Pitched rows, h written over the residual (and over x), nothing written around the outputs."""
    require_gpu()
    M, D = 11, 2048
    x, res, w = bf16((M, D), 1), bf16((M, D), 2), bf16((D,), 3)
    for over in ("residual", "x", "own"):
        xb, xv = guarded(M, D, D + 24)
        rb, rv = guarded(M, D, D + 8 if over != "x" else D + 24)
        xv.copy_(x), rv.copy_(res)
        hb, hv = {"residual": (rb, rv), "x": (xb, xv)}.get(over) or guarded(M, D, D + 16)
        qb, qv = guarded(M, D, D + 32, FP8)
        sb, sv = guarded(M, D // 128, D // 128 + 3, torch.float32)
        hkq.add_rmsnorm_quant(xv, w.cuda(), rv, 1e-6, hkq.KIND_FP8, 128, h=hv, q=qv, s=sv)
        torch.cuda.synchronize()
        check_norm(x, res, w, 1e-6, 128, hkq.KIND_FP8, qv, sv, hv)
        for buf, n in ((xb, D), (rb, D), (hb, D), (qb, D), (sb, D // 128)):
            untouched(buf, M, n)


@pytest.mark.parametrize("D", [512, 4096])
def test_add_rmsnorm_quant_rows_alone_and_together(D):
    """A row's codes do not depend on the other rows of the call."""
    require_gpu()
    x, res, w = bf16((37, D), 4).cuda(), bf16((37, D), 5).cuda(), bf16((D,), 6).cuda()
    q, s, h = hkq.add_rmsnorm_quant(x, w, res)
    for m in (0, 17, 36):
        q1, s1, h1 = hkq.add_rmsnorm_quant(x[m:m + 1], w, res[m:m + 1])
        assert torch.equal(q1.view(torch.uint8)[0], q.view(torch.uint8)[m]) and s1[0] == s[m] and torch.equal(h1[0], h[m])


@pytest.mark.parametrize("kind", [hkq.KIND_FP8, hkq.KIND_INT8])
@pytest.mark.parametrize("group", [0, 128])
def test_add_rmsnorm_quant_nan_and_inf_reach_the_scales(kind, group):
    require_gpu()
    M, D = 5, 512
    x, w = bf16((M, D), 7), torch.ones(D, dtype=BF16)
    x[1, 3], x[2, 200], x[3, 7] = float("nan"), float("inf"), -float("inf")
    _, s, _ = hkq.add_rmsnorm_quant(x.cuda(), w.cuda(), torch.zeros_like(x).cuda(), 1e-6, kind, group)
    s = s.cpu().view(M, -1)
    assert torch.isfinite(s[0]).all() and torch.isfinite(s[4]).all()
    assert torch.isnan(s[1]).all()                      # the row's norm is NaN
    g = 200 // 128 if group else 0                      # x / inf: NaN where x is infinite, zeros elsewhere
    assert torch.isnan(s[2, g]) and torch.isnan(s[3, 0])
    w[300] = float("nan")                               # a NaN weight: its own group, or the row
    _, s, _ = hkq.add_rmsnorm_quant(x[:1].cuda(), w.cuda(), None, 1e-6, kind, group)
    assert torch.isnan(s.view(-1)).cpu().tolist() == ([False, False, True, False] if group else [True])


def test_add_rmsnorm_quant_no_rows():
    require_gpu()
    e = torch.empty((0, 256), dtype=BF16, device="cuda")
    q, s, h = hkq.add_rmsnorm_quant(e, bf16((256,), 1).cuda(), e)
    assert q.shape == (0, 256) and s.shape == (0,) and h.shape == (0, 256)


# ----------------------------------------------------------------- fused epilogue

def sums(kind, A, B, sa=None, sb=None):
    """(products' sums, their error bound) in float64."""
    a, b = A.double(), B.double()
    v, t = a @ b.t(), a.abs() @ b.abs().t()
    if kind == "a8w8":
        f = sa.double()[:, None] * sb.double()[None, :]
        # blocks of 16 products: 16 times 2^-13 of the largest
        blocks = [x.abs().view(x.shape[0], -1, 16).amax(2) for x in (a, b)]
        return v * f, f * ((A.shape[1] + 4) * E * t + 16 * 2.0 ** -13 * (blocks[0] @ blocks[1].t()))
    return v, (A.shape[1] + 4) * E * t


def test_fp8_products_alignment():
    """What the bound of FP8 sums takes from the instruction: next to products
    of +-2^16, one of 2^3 (2^-13 of them) or more is added in full; a smaller one
    is lost beside them, and is added in full 16 places on."""
    require_gpu()
    rows = 17
    for place in (2, 17):
        A, B = torch.zeros(rows, 64), torch.zeros(32, 64)
        A[:, 0] = A[:, 1] = 256
        A[:, place] = 2.0 ** (8 - torch.arange(rows).float())
        B[:, 0], B[:, 1], B[:, place] = 256, -256, 1
        one = torch.ones(rows, device="cuda"), torch.ones(32, device="cuda")
        got = hkq.gemm_a8w8(A.to(FP8).cuda(), B.to(FP8).cuda(), *one).float().cpu()[:, 0] / A[:, place]
        assert got.tolist() == ([1.0] * 6 + [0.0] * 11 if place == 2 else [1.0] * rows)


def epilogue_ref(v, err, bias, act, alpha, res):
    if bias is not None:
        v, err = v + bias.double(), err + E * (v.abs() + bias.double().abs())
    o, tol = act64(v, act, alpha)[0], 1.13 * err + (2.0 ** -19 * v.abs() if act not in ("none", "relu") else 0)
    if res is not None:
        o = o + res.double()
        tol = tol + E * (o.abs() + res.double().abs())
    return o, tol + U * o.abs()


def operands(kind, M, N, K, seed):
    if kind == "a8w8":
        (A, sa), (B, sb) = fp8((M, K), seed), fp8((N, K), seed + 10)
        return A, B, sa / 100, sb / (100 * math.sqrt(K))
    return bf16((M, K), seed), bf16((N, K), seed + 10, 1 / math.sqrt(K)), None, None


def epilogue(kind, A, B, sa, sb, **kw):
    if kind == "a8w8":
        return hkq.gemm_a8w8_epilogue(A, B, sa, sb, **kw)
    return hkq.gemm_bf16_epilogue(A, B, **kw)


# every tile size of the plan: one row to long prefills, ragged in each direction
EPI_SHAPES = [(1, 4, 64), (1, 256, 512), (4, 1000, 4096), (16, 516, 256), (31, 4096, 1024), (33, 2052, 576), (64, 1028, 2048),
              (100, 1028, 512), (129, 4100, 320), (160, 4096, 1024), (300, 2056, 1024), (333, 1284, 8192), (520, 4104, 256),
              (1025, 4100, 128), (2050, 4108, 192)]


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("M,N,K", EPI_SHAPES)
def test_epilogue_shapes(kind, M, N, K):
    require_gpu()
    A, B, sa, sb = operands(kind, M, N, K, M + N + K)
    act = ACTS[(M + N // 4) % 5]
    bias, res = bf16((N,), 3), bf16((M, N), 4, 2.0)
    cu = [t if t is None else t.cuda() for t in (A, B, sa, sb)]
    buf, C = guarded(M, N, N + 4)
    epilogue(kind, *cu, bias=bias.cuda(), act=act, residual=res.cuda(), C=C)
    torch.cuda.synchronize()
    v, err = sums(kind, A, B, sa, sb)
    close(C, *epilogue_ref(v, err, bias, act, 1.0, res), f"{kind} {M}x{N}x{K} {act}")
    untouched(buf, M, N)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M", [3, 70, 700])
def test_epilogue_parts(kind, act, bias, residual, M):
    require_gpu()
    N, K = 520, 256
    A, B, sa, sb = operands(kind, M, N, K, M)
    b = bf16((N,), 3) if bias else None
    r = bf16((M, N), 4, 2.0) if residual else None
    cu = [t if t is None else t.cuda() for t in (A, B, sa, sb, b, r)]
    C = epilogue(kind, *cu[:4], bias=cu[4], act=act, residual=cu[5], alpha=1.1)
    torch.cuda.synchronize()
    v, err = sums(kind, A, B, sa, sb)
    close(C, *epilogue_ref(v, err, b, act, 1.1, r), f"{kind} {act}")


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("M,N,K", [(9, 260, 256), (130, 1028, 256), (700, 1284, 128), (128, 1028, 8192)])
def test_epilogue_residual_in_place_and_pitches(kind, M, N, K):
    """The residual in C's own place, in rows that are 8- but not 16-byte aligned."""
    require_gpu()
    A, B, sa, sb = operands(kind, M, N, K, 5)
    res = bf16((M, N), 4, 2.0)
    buf, C = guarded(M, N, N + 8)
    C = C[:, :]
    C.copy_(res)
    cu = [t if t is None else t.cuda() for t in (A, B, sa, sb)]
    epilogue(kind, *cu, act="silu", residual=C, C=C)
    torch.cuda.synchronize()
    v, err = sums(kind, A, B, sa, sb)
    close(C, *epilogue_ref(v, err, None, "silu", 1.0, res), kind)
    untouched(buf, M, N)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
def test_epilogue_split_k_repeats(kind):
    """K split over workgroups: the same bits each time, whatever the workspace held before, and with none."""
    require_gpu()
    M, N, K = 128, 1024, 14336
    A, B, sa, sb = operands(kind, M, N, K, 6)
    bias, res = bf16((N,), 3), bf16((M, N), 4)
    cu = [t if t is None else t.cuda() for t in (A, B, sa, sb)]
    kw = dict(bias=bias.cuda(), act="gelu", residual=res.cuda())
    assert int(getattr(hkq.lib(), f"hkq_gemm_{kind}_workspace")(M, N, K)) > 0
    first = epilogue(kind, *cu, **kw)
    for _ in range(3):
        torch.randn(1 << 20, device="cuda")
        assert torch.equal(epilogue(kind, *cu, **kw), first)
    v, err = sums(kind, A, B, sa, sb)
    want = epilogue_ref(v, err, bias, "gelu", 1.0, res)
    close(first, *want, "split")
    close(epilogue(kind, *cu, split=False, **kw), *want, "unsplit")


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("M,N,K", [(3, 1000, 512), (40, 4100, 1024), (100, 5632, 2048), (300, 1036, 1024), (300, 14340, 512),
                                   (1024, 1024, 1024), (1100, 7172, 512), (500, 4096, 14336)])
def test_epilogue_residual_in_place(kind, M, N, K):
    """The residual as C gives the bits of a residual of its own, in every tile size."""
    require_gpu()
    A, B, sa, sb = (t if t is None else t.cuda() for t in operands(kind, M, N, K, M + N))
    res, bias = bf16((M, N), 7).cuda(), bf16((N,), 8).cuda()
    call = (lambda **kw: hkq.gemm_a8w8_epilogue(A, B, sa, sb, **kw)) if kind == "a8w8" else \
        (lambda **kw: hkq.gemm_bf16_epilogue(A, B, **kw))
    want = call(bias=bias, act="silu", residual=res)
    buf, C = guarded(M, N, N + 4)
    C.copy_(res)
    call(bias=bias, act="silu", residual=C, C=C)
    torch.cuda.synchronize()
    assert torch.equal(C, want)
    untouched(buf, M, N)


# grids of the streaming kernel (whole tiles over several rounds and a last round
# in halves; its K-tiles come in eights: K a multiple of 512 bf16 or 1024 FP8
# values) and of 192-row tiles, ragged in both directions, rows of C pitched
LARGE = {"a8w8": [(2300, 14340, 1024), (601, 14340, 2048), (1100, 6152, 1088)],
         "bf16": [(2300, 14340, 512), (601, 14340, 1024), (1100, 6152, 544)]}


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("act,bias,residual", [("gelu", True, True), ("silu", True, False), ("none", False, True)])
def test_epilogue_large_tiles(kind, which, act, bias, residual):
    """The reference in 64 bits on the GPU."""
    require_gpu()
    M, N, K = LARGE[kind][which]
    A, B, sa, sb = (t if t is None else t.cuda() for t in operands(kind, M, N, K, M + which))
    b = bf16((N,), 3).cuda() if bias else None
    rbuf = bf16((M, N + 4), 4, 2.0).cuda()  # rows 8-, not 16-byte aligned
    r = rbuf[:, :N] if residual else None
    buf, C = guarded(M, N, N + 4 if which != 1 else N + 12)
    epilogue(kind, A, B, sa, sb, bias=b, act=act, residual=r, C=C)
    v, err = sums(kind, A, B, sa, sb)
    close(C, *epilogue_ref(v, err, b, act, 1.0, r), f"{kind} {M}x{N}x{K} {act}")
    untouched(buf, M, N)


def test_epilogue_special_values():
    """Saturated activations, infinities and NaN as in the formulas."""
    require_gpu()
    vals = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 5.0, -5.0, 30.0, -30.0, 1e4, -1e4, 3e38, -3e38, float("inf"), float("nan")])
    K = 32
    A = torch.zeros((len(vals), K), dtype=BF16)
    A[:, 0] = vals.to(BF16)
    B = torch.zeros((4, K), dtype=BF16)
    B[:, 0] = 1
    # (an infinite operand meets the other columns' zeros: every one of its sums is NaN)
    for act in ACTS:
        C = hkq.gemm_bf16_epilogue(A.cuda(), B.cuda(), act=act).cpu().double()
        v = A[:, :1].double().expand(-1, 4).clone()
        ref = act64(v, act)[0]
        for i in range(len(vals)):
            if i >= 12:
                assert torch.isnan(C[i]).all() or (i == 12 and torch.isinf(C[i]).all()), (act, i, C[i])
                continue
            assert torch.isfinite(C[i]).all(), (act, float(vals[i]), C[i])
            assert ((C[i] - ref[i]).abs() <= U * ref[i].abs() + 2.0 ** -19 * v[i].abs().clamp_max(1e4)).all(), (act, float(vals[i]), C[i])


def test_epilogue_no_rows_or_columns():
    require_gpu()
    A, B = bf16((0, 64), 1).cuda(), bf16((8, 64), 2).cuda()
    assert hkq.gemm_bf16_epilogue(A, B, act="silu").shape == (0, 8)
    assert hkq.gemm_bf16_epilogue(B, A, act="silu").shape == (8, 0)


# --------------------------------------------------------------------- gated pair

def halves(y, interleaved):
    F = y.shape[1] // 2
    return (y[:, 0::2], y[:, 1::2]) if interleaved else (y[:, :F], y[:, F:])


def gated_ref(y, err, act, alpha, interleaved):
    (g, u), (eg, eu) = halves(y, interleaved), halves(err, interleaved)
    a = act64(g, act, alpha)[0]
    ea = 1.13 * eg + (2.0 ** -19 * g.abs() if act not in ("none", "relu") else 0)
    h = a * u
    return h, U * h.abs() + (1 + E) * (ea * u.abs() + a.abs() * eu + ea * eu) + 3 * E * h.abs()


# one token to long prefills; features ragged against every tile width
GATED_SHAPES = [(1, 8, 64), (1, 256, 512), (5, 520, 4096), (16, 1000, 256), (17, 4096, 512), (31, 264, 576), (48, 2048, 1024),
                (100, 1032, 512), (129, 2056, 320), (200, 4096, 256), (300, 1032, 1024), (520, 2056, 256), (1030, 2056, 128),
                (2050, 2056, 192)]


def gated(kind, A, W, sa, sw, **kw):
    if kind == "a8w8":
        return hkq.gated_ffn_a8w8(A, W, sa, sw, **kw)
    return hkq.gated_ffn_bf16(A, W, **kw)


@pytest.mark.parametrize("kind", ["a8w8", "bf16", "bf16_save"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,F,K", GATED_SHAPES)
def test_gated_shapes(kind, interleaved, M, F, K):
    require_gpu()
    save, kind = kind.endswith("save"), kind[:4]
    A, W, sa, sw = operands(kind, M, 2 * F, K, M + F + K)
    act = ACTS[(M + F // 8) % 5]
    cu = [t if t is None else t.cuda() for t in (A, W, sa, sw)]
    hbuf, H = guarded(M, F, F + 12)
    kw = {}
    if save:
        ybuf, kw["Y"] = guarded(M, 2 * F, 2 * F + 4)
    gated(kind, *cu, act=act, interleaved=interleaved, H=H, **kw)
    torch.cuda.synchronize()
    y, err = sums(kind, A, W, sa, sw)
    close(H, *gated_ref(y, err, act, 1.0, interleaved), f"{kind} {M}x{F}x{K} {act}")
    untouched(hbuf, M, F)
    if save:
        close(kw["Y"], y, err + U * y.abs(), "kept projections")
        untouched(ybuf, M, 2 * F)


# workgroups of 8 features and of 16, one and several groups of rows, 32 x 32 tiles
# over a long K and with a half K-tile at its end
@pytest.mark.parametrize("kind", ["a8w8", "bf16_save"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,F,K", [(1, 2048, 4096), (4, 1000, 2048), (8, 4000, 512), (2, 14336, 4096), (16, 2048, 128),
                                   (24, 2040, 8192), (33, 504, 1088), (63, 1024, 2816), (64, 512, 4096)])
def test_gated_few_rows(kind, interleaved, M, F, K):
    require_gpu()
    save, kind = kind.endswith("save"), kind[:4]
    A, W, sa, sw = (t if t is None else t.cuda() for t in operands(kind, M, 2 * F, K, M + F + K))
    hbuf, H = guarded(M, F, F + 8)
    kw = {}
    if save:
        ybuf, kw["Y"] = guarded(M, 2 * F, 2 * F + 8)
    gated(kind, A, W, sa, sw, act="gelu_tanh", interleaved=interleaved, H=H, **kw)
    y, err = sums(kind, A, W, sa, sw)
    close(H, *gated_ref(y, err, "gelu_tanh", 1.0, interleaved), f"{kind} {M}x{F}x{K}")
    untouched(hbuf, M, F)
    if save:
        close(kw["Y"], y, err + U * y.abs(), "kept projections")
        untouched(ybuf, M, 2 * F)


@pytest.mark.parametrize("kind", ["a8w8", "bf16", "bf16_save"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("which,act", [(0, "silu"), (1, "gelu_tanh"), (2, "gelu")])
def test_gated_large_tiles(kind, interleaved, which, act):
    require_gpu()
    save, kind = kind.endswith("save"), kind[:4]
    M, N, K = LARGE[kind][which]
    F = N // 16 * 8
    A, W, sa, sw = (t if t is None else t.cuda() for t in operands(kind, M, 2 * F, K, M + which))
    hbuf, H = guarded(M, F, F + 8)
    kw = {}
    if save:
        ybuf, kw["Y"] = guarded(M, 2 * F, 2 * F + 4)
    gated(kind, A, W, sa, sw, act=act, interleaved=interleaved, H=H, **kw)
    y, err = sums(kind, A, W, sa, sw)
    close(H, *gated_ref(y, err, act, 1.0, interleaved), f"{kind} {M}x{F}x{K} {act}")
    untouched(hbuf, M, F)
    if save:
        close(kw["Y"], y, err + U * y.abs(), "kept projections")
        untouched(ybuf, M, 2 * F)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [2, 40, 600])
def test_gated_activations_and_pitches(kind, act, M):
    """Weight and activation rows apart from each other, alpha of SiLU."""
    require_gpu()
    F, K = 264, 256
    A, W, sa, sw = operands(kind, M, 2 * F, K, M)
    Wp = torch.zeros((2 * F, K + 64), dtype=W.dtype)
    Ap = torch.zeros((M, K + 32), dtype=A.dtype)
    if kind == "a8w8":  # codes of NaN between the rows: none may reach a sum
        Wp.view(torch.uint8).fill_(0x7F), Ap.view(torch.uint8).fill_(0x7F)
    else:
        Wp.fill_(float("nan")), Ap.fill_(float("nan"))
    Wp[:, :K], Ap[:, :K] = W, A
    cu = [t if t is None else t.cuda() for t in (sa, sw)]
    y, err = sums(kind, A, W, sa, sw)
    for interleaved in (False, True):
        H = gated(kind, Ap.cuda()[:, :K], Wp.cuda()[:, :K], *cu, act=act, alpha=0.9, interleaved=interleaved)
        torch.cuda.synchronize()
        close(H, *gated_ref(y, err, act, 0.9, interleaved), f"{kind} {act}")


# ------------------------------------------------------------------- its backward

def backward_ref(dH, X, W, Y, act, alpha, interleaved):
    (g, u), dh = halves(Y.double(), interleaved), dH.double()
    a, slope = act64(g, act, alpha)
    dg, du = dh * u * slope, dh * a
    # the slope's evaluation: a few steps of its terms, |g| of them growing with the argument
    eg = (dh * u).abs() * (1 + g.abs() + 0.2 * g.abs() ** 3 * (act == "gelu_tanh")) * 2.0 ** -18 if act not in ("none", "relu") else 0 * g
    ea = dh.abs() * g.abs() * 2.0 ** -19
    eg, eu = U * dg.abs() + eg + 4 * E * dg.abs(), U * du.abs() + ea + 4 * E * du.abs()
    F = g.shape[1]

    def join(p, q):
        return torch.stack((p, q), 2).reshape(p.shape[0], 2 * F) if interleaved else torch.cat((p, q), 1)

    dy, ey, w, x = join(dg, du), join(eg, eu), W.double(), X.double()
    dx, tx = dy @ w, ey @ w.abs() + (2 * F + 4) * E * ((dy.abs() + ey) @ w.abs())
    dw, tw = dy.t() @ x, ey.t() @ x.abs() + (X.shape[0] + 4) * E * ((dy.abs() + ey).t() @ x.abs())
    return (dx, tx + U * dx.abs()), (dw, tw + U * dw.abs())


BWD_SHAPES = [(1, 8, 32), (3, 40, 64), (64, 256, 256), (65, 136, 288), (129, 520, 256), (300, 1032, 544), (7, 2816, 512),
              (1001, 1408, 1024), (2050, 328, 2080), (520, 4104, 4128)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,F,K", BWD_SHAPES)
def test_backward_shapes(interleaved, M, F, K):
    require_gpu()
    act = ACTS[(M + F // 8 + interleaved) % 5]
    X, W, Y, dH = bf16((M, K), 1), bf16((2 * F, K), 2, 0.05), bf16((M, 2 * F), 3, 1.5), bf16((M, F), 4, 0.3)
    xb, dX = guarded(M, K, K + 8)
    wb, dW = guarded(2 * F, K, K + 4)
    hkq.gated_ffn_backward(dH.cuda(), X.cuda(), W.cuda(), Y.cuda(), act=act, interleaved=interleaved, dX=dX, dW=dW)
    torch.cuda.synchronize()
    rx, rw = backward_ref(dH, X, W, Y, act, 1.0, interleaved)
    close(dX, *rx, f"dX {M}x{F}x{K} {act}", 2)
    close(dW, *rw, f"dW {M}x{F}x{K} {act}", 2)
    untouched(xb, M, K)
    untouched(wb, 2 * F, K)


# the streaming kernel over several rounds (K-tiles in eights), 128 x 256 tiles,
# an odd count of tokens whose last K-tile holds one row
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,F,K,act", [(2048, 2048, 4096, "silu"), (4096, 4352, 2080, "gelu_tanh"), (1025, 4352, 4096, "gelu"),
                                       (2300, 2056, 2048, "relu")])
def test_backward_large_tiles(interleaved, M, F, K, act):
    """The reference in 64 bits on the GPU."""
    require_gpu()
    X, W, Y, dH = bf16((M, K), 1).cuda(), bf16((2 * F, K), 2, 0.05).cuda(), bf16((M, 2 * F), 3, 1.5).cuda(), bf16((M, F), 4, 0.3).cuda()
    xb, dX = guarded(M, K, K + 8)
    wb, dW = guarded(2 * F, K, K + 8)
    hkq.gated_ffn_backward(dH, X, W, Y, act=act, interleaved=interleaved, dX=dX, dW=dW)
    rx, rw = backward_ref(dH, X, W, Y, act, 1.0, interleaved)
    close(dX, *rx, f"dX {M}x{F}x{K} {act}", 2)
    close(dW, *rw, f"dW {M}x{F}x{K} {act}", 2)
    untouched(xb, M, K)
    untouched(wb, 2 * F, K)


# few tokens of a wide layer: dX's K split over 256 x 256 tiles; rows and columns
# that end inside a tile, a last part shorter than the others
@pytest.mark.parametrize("M,F,K,interleaved", [(600, 8200, 3328, False), (1300, 8200, 3232, True), (513, 8192, 3296, False)])
def test_backward_parts(M, F, K, interleaved):
    """The reference in 64 bits on the GPU; the same bits again from a workspace that held NaN."""
    require_gpu()
    X, W, Y, dH = bf16((M, K), 1).cuda(), bf16((2 * F, K), 2, 0.05).cuda(), bf16((M, 2 * F), 3, 1.5).cuda(), bf16((M, F), 4, 0.3).cuda()
    xb, dX = guarded(M, K, K + 8)
    hkq.gated_ffn_backward(dH, X, W, Y, interleaved=interleaved, dX=dX, need_dw=False)
    n = hkq.lib().hkq_gated_ffn_backward_workspace(M, F, K)
    assert n >= M * 4 * F + 2 * 4 * (M // 256 + 1) * 256 * K  # two parts at least
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    again = torch.empty((M, K), dtype=BF16, device="cuda")
    hkq.call("hkq_gated_ffn_backward", dH.data_ptr(), None, W.data_ptr(), Y.data_ptr(), again.data_ptr(), None, M, F, K,
             F, K, K, 2 * F, K, K, hkq.ACTIVATIONS["silu"], 1.0, int(interleaved), ws.data_ptr(), n,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(again, dX)
    rx, _ = backward_ref(dH, X[:, :32], W, Y, "silu", 1.0, interleaved)
    close(dX, *rx, f"dX {M}x{F}x{K}", 2)
    untouched(xb, M, K)


@pytest.mark.parametrize("act", ACTS)
def test_backward_activations_pitches_and_one_gradient(act):
    """NaN between the operands' rows reaches nothing; either gradient alone gives the same bits."""
    require_gpu()
    M, F, K = 77, 200, 160

    def pitched(t, extra):
        b = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), dtype=BF16, device="cuda")
        v = b[:, :t.shape[1]]
        v.copy_(t)
        return v

    X, W, Y, dH = bf16((M, K), 1), bf16((2 * F, K), 2, 0.1), bf16((M, 2 * F), 3, 2.0), bf16((M, F), 4)
    ops = pitched(dH, 8), pitched(X, 16), pitched(W, 24), pitched(Y, 40)
    dX, dW = hkq.gated_ffn_backward(*ops, act=act, alpha=0.8)
    torch.cuda.synchronize()
    rx, rw = backward_ref(dH, X, W, Y, act, 0.8, False)
    close(dX, *rx, "dX", 2)
    close(dW, *rw, "dW", 2)
    only_x = hkq.gated_ffn_backward(*ops, act=act, alpha=0.8, need_dw=False)
    only_w = hkq.gated_ffn_backward(*ops, act=act, alpha=0.8, need_dx=False)
    assert only_x[1] is None and only_w[0] is None
    assert torch.equal(only_x[0], dX) and torch.equal(only_w[1], dW)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu"])
def test_backward_against_differences(act):
    """dX and dW along random directions against central differences of the
    forward in 64 bits: sum(dH * H(X + t V, W + t Z)) moves by t (<dX, V> + <dW, Z>).
    The step's own error is of order t^2; the gradients' bound is the one above,
    summed over the direction."""
    require_gpu()
    M, F, K = 20, 72, 64
    X, W, dH = bf16((M, K), 1), bf16((2 * F, K), 2, 0.15), bf16((M, F), 4)
    H, Y = hkq.gated_ffn_bf16(X.cuda(), W.cuda(), act=act, save=True)
    dX, dW = hkq.gated_ffn_backward(dH.cuda(), X.cuda(), W.cuda(), Y, act=act)
    V, Z = torch.randn((M, K), generator=gen(5)).double(), torch.randn((2 * F, K), generator=gen(6)).double() * 0.15

    def loss(t):
        y = (X.double() + t * V) @ (W.double() + t * Z).t()
        return float((dH.double() * act64(y[:, :F], act)[0] * y[:, F:]).sum())

    t = 1e-4
    num = (loss(t) - loss(-t)) / (2 * t)
    got = float((dX.cpu().double() * V).sum() + (dW.cpu().double() * Z).sum())
    # Y is kept in bf16: its rounding moves the slopes, by U |y| times the second derivatives
    # (below 1.2), on top of the gradients' own bound
    (rx, tx), (rw, tw) = backward_ref(dH, X, W, Y.cpu(), act, 1.0, False)
    g, u = halves(Y.cpu().double(), False)
    dg, du = dH.double().abs() * U * (1.2 * g.abs() * u.abs() + 1.13 * u.abs()), dH.double().abs() * 1.13 * U * g.abs()
    w, x = W.double().abs(), X.double().abs()
    tol = float(((tx + dg @ w[:F] + du @ w[F:]) * V.abs()).sum() + ((tw + torch.cat((dg, du), 1).t() @ x) * Z.abs()).sum())
    assert abs(got - num) <= tol + 1e-5 * abs(num), (got, num, tol)
    # the bound adds every rounding with one sign; their signs are random, so the
    # sum stays within a small share of it, unless a term is missing
    assert abs(got - num) <= 0.05 * tol + 1e-5 * abs(num), (got, num, tol)


@pytest.mark.parametrize("act", ACTS)
def test_backward_slopes_at_the_ends(act):
    """Activations that saturate have slopes 1 and 0 far out; "none" and ReLU
    also at infinities and NaN (ReLU passes a NaN's gradient on). One token with
    X of ones: row f of dW is the projection's gradient itself, exactly."""
    require_gpu()
    inf, nan, big = float("inf"), float("nan"), 2.0 ** 127
    g = torch.tensor([big, -big, 0.0, -0.0, 1e4, -1e4, 2.0 ** 60, -2.0 ** 60])
    if act in ("none", "relu"):
        g = torch.cat((g, torch.tensor([inf, -inf, nan, 1.0, -1.0, 2.0, -2.0, 0.5])))
    F, K = len(g), 32
    u, dh = torch.full((1, F), 2.0), torch.full((1, F), 0.25)
    Y = torch.cat((g.to(BF16)[None], u.to(BF16)), 1).cuda()
    _, dW = hkq.gated_ffn_backward(dh.to(BF16).cuda(), torch.ones(1, K, dtype=BF16).cuda(),
                                   torch.zeros(2 * F, K, dtype=BF16).cuda(), Y, act=act, need_dx=False)
    g = g.to(BF16).double()
    slope = torch.ones(F).double() if act == "none" else (~(g <= 0)).double()
    if act not in ("none", "relu"):
        slope[g == 0] = 0.5
    value = g if act == "none" else torch.where(g <= 0, torch.zeros_like(g), g)
    want = torch.cat((0.5 * slope, 0.25 * value))[:, None].expand(2 * F, K)
    assert torch.equal(torch.nan_to_num(dW.cpu().double(), nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_backward_without_tokens_or_features():
    require_gpu()
    X, W = bf16((0, 64), 1).cuda(), bf16((32, 64), 2).cuda()
    dX, dW = hkq.gated_ffn_backward(bf16((0, 16), 3).cuda(), X, W, bf16((0, 32), 4).cuda())
    assert dX.shape == (0, 64) and dW.shape == (32, 64) and not dW.any()
    X, W = bf16((0, 2048), 1).cuda(), bf16((16384, 2048), 2).cuda()  # as many tiles as a large layer has
    wb, dW = guarded(16384, 2048, 2056)
    hkq.gated_ffn_backward(bf16((0, 8192), 3).cuda(), X, W, bf16((0, 16384), 4).cuda(), dW=dW)
    assert not dW.any()
    untouched(wb, 16384, 2048)
    X, W = bf16((5, 64), 1).cuda(), bf16((0, 64), 2).cuda()
    dX, dW = hkq.gated_ffn_backward(bf16((5, 0), 3).cuda(), X, W, bf16((5, 0), 4).cuda())
    assert dX.shape == (5, 64) and not dX.any() and dW.shape == (0, 64)


# -------------------------------------------------------------- together, streams, graphs

def test_outputs_belong_to_the_stream_of_the_call():
    """Outputs and workspaces of a call on another stream are that stream's memory:
    they are not a block that work pending on the current stream still uses."""
    require_gpu()
    M, K, F = 256, 512, 1024
    x, w = bf16((M, K), 1).cuda(), bf16((2 * F, K), 2, 0.05).cuda()
    dh = bf16((M, F), 3).cuda()
    want = hkq.gated_ffn_bf16(x, w, save=True)
    want += hkq.gated_ffn_backward(dh, x, w, want[1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        # blocks of the outputs' sizes, freed here while the current stream is still to write them
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            busy = busy @ busy * 1e-4
        junk = [torch.full_like(t, 3.0) for t in want]
        del junk
        H, Y = hkq.gated_ffn_bf16(x, w, save=True, stream=side)
        got = (H, Y) + hkq.gated_ffn_backward(dh, x, w, Y, stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))



def layer_fp8(x, res, w, w1, s1, w2, s2, stream=None):
    """A serving step's dense feed-forward layer: the new stream and the layer's own output."""
    q, s, h = hkq.add_rmsnorm_quant(x, w, res, stream=stream)
    H = hkq.gated_ffn_a8w8(q, w1, s, s1, stream=stream)
    q2, sq2 = hkq.per_token_quant(H, stream=stream)
    return hkq.gemm_a8w8_epilogue(q2, w2, sq2, s2, residual=h, stream=stream), q, s, h, H, q2, sq2


@pytest.mark.parametrize("M", [1, 24, 300])
def test_feedforward_layer_fp8(M):
    """Norm, gated pair, quantizer, down projection with the residual: each step
    within its bound of the definition on the step's own inputs, and the chain
    captured in a graph and on another stream with the same bits."""
    require_gpu()
    K, F = 512, 1024
    x, res, w = bf16((M, K), 1), bf16((M, K), 2), bf16((K,), 3)
    (w1, s1), (w2, s2) = fp8((2 * F, K), 4), fp8((K, F), 5)
    s1, s2 = s1 / (100 * math.sqrt(K)), s2 / (100 * math.sqrt(F))
    args = [t.cuda() for t in (x, res, w, w1, s1, w2, s2)]
    out, q, s, h, H, q2, sq2 = layer_fp8(*args)
    torch.cuda.synchronize()
    check_norm(x, res, w, 1e-6, 0, hkq.KIND_FP8, q, s, h)
    y, err = sums("a8w8", q.cpu(), w1, s.cpu(), s1)
    close(H, *gated_ref(y, err, "silu", 1.0, False), "H")
    v, err = sums("a8w8", q2.cpu(), w2, sq2.cpu(), s2)
    close(out, *epilogue_ref(v, err, None, "none", 1.0, h.cpu()), "out")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = layer_fp8(*args, stream=side)[0]
    side.synchronize()
    assert torch.equal(other, out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer_fp8(*args)[0]
    for k in range(4):
        args[0].copy_(torch.roll(x, k, 1))
        want = layer_fp8(*args)[0]
        torch.cuda.synchronize()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {k}"


def test_feedforward_training_step():
    """Forward with the projections kept, down projection with the residual, and
    the gradients: the first-order change of a loss in 64 bits, eager, on another
    stream and captured."""
    require_gpu()
    M, K, F = 130, 256, 512
    x, w1, w2 = bf16((M, K), 1).cuda(), bf16((2 * F, K), 2, 0.06).cuda(), bf16((K, F), 3, 0.05).cuda()
    dout = bf16((M, K), 4).cuda()
    w2t = w2.t().contiguous()

    def step(stream=None):
        H, Y = hkq.gated_ffn_bf16(x, w1, save=True, stream=stream)
        out = hkq.gemm_bf16_epilogue(H, w2, residual=x, stream=stream)
        dH = hkq.gemm_bf16(dout, w2t, stream=stream)  # dout . w2
        dX, dW = hkq.gated_ffn_backward(dH, x, w1, Y, stream=stream)
        return out, H, Y, dH, dX, dW

    out, H, Y, dH, dX, dW = step()
    torch.cuda.synchronize()
    c = [t.cpu() for t in (x, w1, w2, H, Y, dH)]
    y, err = sums("bf16", c[0], c[1])
    close(H, *gated_ref(y, err, "silu", 1.0, False), "H")
    v, err = sums("bf16", c[3], c[2])
    close(out, *epilogue_ref(v, err, None, "none", 1.0, c[0]), "out")
    rx, rw = backward_ref(c[5], c[0], c[1], c[4], "silu", 1.0, False)
    close(dX, *rx, "dX", 2)
    close(dW, *rw, "dW", 2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, (out, H, Y, dH, dX, dW)))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    keep = x.clone()
    for k in range(4):
        x.copy_(torch.roll(keep, k, 1))
        want = step()
        torch.cuda.synchronize()
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {k}"


def test_modules_give_the_same_bytes():
    """The pybind modules against the tensor layer over the C ABI."""
    require_gpu()
    import hipkittens as hk

    M, K, F = 70, 256, 128
    x, res, w = bf16((M, K), 1).cuda(), bf16((M, K), 2).cuda(), bf16((K,), 3).cuda()
    for kind, group in ((hkq.KIND_FP8, 0), (hkq.KIND_INT8, 128)):
        q, s, h = hkq.add_rmsnorm_quant(x, w, res, 1e-6, kind, group)
        q2, s2, h2 = torch.empty_like(q), torch.empty_like(s), torch.empty_like(h)
        hk.fused_add_rmsnorm_quant_fwd(x, res, w, h2, q2, s2, 1e-6, group)
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s) and torch.equal(h2, h)
    q, s, _ = hkq.add_rmsnorm_quant(x, w, res)
    wq, ws = (t.cuda() for t in fp8((2 * F, K), 4))
    H = torch.empty((M, F), dtype=BF16, device="cuda")
    hk.ffn.gated.gated_ffn_a8w8(q, wq, s, ws, H, act="gelu", interleaved=True)
    assert torch.equal(H, hkq.gated_ffn_a8w8(q, wq, s, ws, act="gelu", interleaved=True))
    C = torch.empty((M, 2 * F), dtype=BF16, device="cuda")
    bias, r2 = bf16((2 * F,), 5).cuda(), bf16((M, 2 * F), 6).cuda()
    hk.fused_gemm.a8w8_epilogue.dispatch(q, wq, s, ws, C, bias, r2, "silu", 0.5)
    assert torch.equal(C, hkq.gemm_a8w8_epilogue(q, wq, s, ws, bias, "silu", r2, 0.5))
    wb = bf16((2 * F, K), 7, 0.1).cuda()
    hk.fused_gemm.a16w16_epilogue.dispatch(x, wb, C, residual=r2, act="relu")
    assert torch.equal(C, hkq.gemm_bf16_epilogue(x, wb, act="relu", residual=r2))
    Y = torch.empty_like(C)
    hk.ffn.gated.gated_ffn_bf16(x, wb, H, Y)
    want = hkq.gated_ffn_bf16(x, wb, save=True)
    assert torch.equal(H, want[0]) and torch.equal(Y, want[1])
    dX, dW = torch.empty_like(x), torch.empty_like(wb)
    hk.ffn.gated.gated_ffn_backward(H, x, wb, Y, dX, dW)
    want = hkq.gated_ffn_backward(H, x, wb, Y)
    assert torch.equal(dX, want[0]) and torch.equal(dW, want[1])


# ------------------------------------------------------------- outputs over operands

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,F,K", [(5, 32, 64), (1001, 1408, 1024), (600, 8200, 3328)])
def test_backward_outputs_over_operands(interleaved, M, F, K):
    """dX in X's place, dW in W's, dX in Y's memory: the bits of outputs of their own."""
    require_gpu()
    ops = bf16((M, F), 4, 0.3), bf16((M, K), 1), bf16((2 * F, K), 2, 0.05), bf16((M, 2 * F), 3, 1.5)
    dH, X, W, Y = (t.cuda() for t in ops)
    dX, dW = hkq.gated_ffn_backward(dH, X, W, Y, interleaved=interleaved)
    x = X.clone()
    got = hkq.gated_ffn_backward(dH, x, W, Y, interleaved=interleaved, dX=x)
    assert torch.equal(got[0], dX) and torch.equal(got[1], dW), "dX over X"
    w = W.clone()
    got = hkq.gated_ffn_backward(dH, X, w, Y, interleaved=interleaved, dW=w)
    assert torch.equal(got[0], dX) and torch.equal(got[1], dW), "dW over W"
    both = torch.cat((Y, X), 1)  # rows of Y followed by rows of X: dX goes over Y's
    if K <= 2 * F:
        got = hkq.gated_ffn_backward(dH, both[:, 2 * F:], W, both[:, :2 * F], interleaved=interleaved, dX=both[:, :K])
        assert torch.equal(got[0], dX) and torch.equal(got[1], dW), "dX over Y"
        assert torch.equal(both[:, 2 * F:], X)


def test_backward_outputs_beside_operands():
    """Columns of one buffer side by side share no element: not refused."""
    require_gpu()
    M, F, K = 70, 72, 64
    dH, X, W, Y = bf16((M, F), 4, 0.3).cuda(), bf16((M, K), 1).cuda(), bf16((2 * F, K), 2, 0.05).cuda(), bf16((M, 2 * F), 3).cuda()
    dX, dW = hkq.gated_ffn_backward(dH, X, W, Y)
    xs, ws = torch.cat((X, X), 1), torch.cat((W, W), 1)
    got = hkq.gated_ffn_backward(dH, xs[:, K:], ws[:, :K], Y, dX=xs[:, :K], dW=ws[:, K:])
    assert torch.equal(got[0], dX) and torch.equal(got[1], dW)
    assert torch.equal(xs[:, K:], X) and torch.equal(ws[:, :K], W)


def test_backward_of_neither_gradient():
    """No workspace is taken where nothing is asked for."""
    require_gpu()
    M, F, K = 512, 1024, 512
    dH, X, W, Y = bf16((M, F), 4).cuda(), bf16((M, K), 1).cuda(), bf16((2 * F, K), 2).cuda(), bf16((M, 2 * F), 3).cuda()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    assert hkq.gated_ffn_backward(dH, X, W, Y, need_dx=False, need_dw=False) == (None, None)
    assert torch.cuda.max_memory_allocated() == before


def test_outputs_beside_operands():
    """Outputs in the columns beside their operands' share no element: not refused, and nothing else is written."""
    require_gpu()
    M, K, F = 70, 64, 64
    x, res, w = bf16((M, K), 1).cuda(), bf16((M, K), 2).cuda(), bf16((K,), 3).cuda()
    W = bf16((2 * F, K), 4, 0.1).cuda()
    q, s, h = hkq.add_rmsnorm_quant(x, w, res)
    both = torch.cat((x, res, res), 1)
    q2, s2, _ = hkq.add_rmsnorm_quant(both[:, :K], w, both[:, K:2 * K], h=both[:, 2 * K:])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    assert torch.equal(both, torch.cat((x, res, h), 1))
    H, Y = hkq.gated_ffn_bf16(x, W, save=True)
    both = torch.cat((x, torch.zeros_like(H), torch.zeros_like(Y)), 1)
    hkq.gated_ffn_bf16(both[:, :K], W, H=both[:, K:K + F], Y=both[:, K + F:])
    assert torch.equal(both, torch.cat((x, H, Y), 1))
    C = hkq.gemm_bf16_epilogue(x, W, act="silu", residual=Y)
    both = torch.cat((x, Y, torch.zeros_like(Y)), 1)
    hkq.gemm_bf16_epilogue(both[:, :K], W, act="silu", residual=both[:, K:K + 2 * F], C=both[:, K + 2 * F:])
    assert torch.equal(both, torch.cat((x, Y, C), 1))


# ------------------------------------------------------------- operands past 32 bits

def sampled(n, k, *marks):
    """k indices of n: the first, the last, those around each mark, others."""
    at = {0, n - 1, *(i for m in marks for i in (m - 1, m) if 0 <= i < n)}
    at |= set(torch.randint(0, n, (k,), generator=gen(n)).tolist())
    return torch.tensor(sorted(at), device="cuda")


def gpu_bf16(shape, seed, std=1.0):
    """Normal values made on the GPU, a block of rows at a time."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(shape, dtype=BF16, device="cuda")
    step = max(1, (1 << 28) // shape[1])
    for i in range(0, shape[0], step):
        n = min(step, shape[0] - i)
        out[i:i + n] = torch.randn((n, shape[1]), generator=g, device="cuda") * std
    return out


def columns(t, f, F):
    """Columns f of both halves of [.., 2F]."""
    return torch.cat((t[:, f], t[:, F + f]), 1)


# dW's sums over tokens whose gradients (the K-tiles' memory rows) pass 4 GiB: on
# K groups of 128 x 64 tiles, the streaming kernel (K-tiles in eights) and the
# one-tile kernel; dX's over 4 GiB of weights, in parts of K
@pytest.mark.parametrize("M,F,K", [(70001, 16384, 64), (66048, 16384, 512), (66049, 16384, 512), (300, 1 << 20, 1056)])
def test_gated_operands_past_32_bits(M, F, K):
    """Forward with the projections kept, and both gradients: rows and columns on
    either side of 2^31 and 2^32 bytes into each tensor, and random ones."""
    require_gpu()
    torch.cuda.empty_cache()
    X, W, dH = gpu_bf16((M, K), 1), gpu_bf16((2 * F, K), 2, 1 / math.sqrt(K)), gpu_bf16((M, F), 3, 0.3)
    H, Y = hkq.gated_ffn_bf16(X, W, save=True)
    assert max(Y.numel(), W.numel()) * 2 > 1 << 32
    marks = [(1 << b) // (2 * w) for b in (31, 32) for w in (F, 2 * F, K)]
    m, f = sampled(M, 12, *marks), sampled(F, 12, *(x for k in marks for x in (k, k - F)))
    w = torch.cat((W[f], W[F + f]))
    y = X[m].double() @ w.double().t()
    err = (K + 4) * E * (X[m].double().abs() @ w.double().abs().t())
    close(columns(Y[m], f, F), y, err + U * y.abs(), "Y")
    close(H[m][:, f], *gated_ref(y, err, "silu", 1.0, False), "H")
    del H
    dX, dW = hkq.gated_ffn_backward(dH, X, W, Y)
    _, rw = backward_ref(dH[:, f], X, w, columns(Y, f, F), "silu", 1.0, False)
    close(torch.cat((dW[f], dW[F + f])), *rw, "dW", 2)
    want = torch.zeros((len(m), K), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    step = 1 << 16
    for i in range(0, F, step):  # a range of features at a time
        n = torch.arange(i, min(F, i + step), device="cuda")
        (dx, tx), _ = backward_ref(dH[m][:, n], X[m][:, :32], torch.cat((W[n], W[F + n])), columns(Y[m], n, F), "silu", 1.0, False)
        want += dx
        # the bound of 2n summed products, scaled to that of all 2F
        tol += (tx - U * dx.abs()) * ((2 * F + 4) / (2 * len(n) + 4))
    close(dX[m], want, tol + U * want.abs(), "dX", 2)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("M,N,K", [(70001, 32768, 64), (66049, 32776, 1024)])
def test_epilogue_operands_past_32_bits(kind, M, N, K):
    """C and the residual of more than 4 GiB, the residual also in C's place."""
    require_gpu()
    torch.cuda.empty_cache()
    A, B, sa, sb = (t if t is None else t.cuda() for t in operands(kind, M, N, K, 3))
    res, bias = gpu_bf16((M, N), 4, 2.0), bf16((N,), 5).cuda()
    C = epilogue(kind, A, B, sa, sb, bias=bias, act="silu", residual=res)
    marks = [(1 << b) // (2 * N) for b in (31, 32)]
    m, n = sampled(M, 40, *marks), sampled(N, 40)
    a, b = (t.view(torch.uint8)[i].view(t.dtype) for t, i in ((A, m), (B, n)))
    v, err = sums(kind, a, b, *(() if sa is None else (sa[m], sb[n])))
    close(C[m][:, n], *epilogue_ref(v, err, bias[n], "silu", 1.0, res[m][:, n]), kind)
    assert torch.equal(epilogue(kind, A, B, sa, sb, bias=bias, act="silu", residual=res, C=res), C)


# a row of 8 columns per wave, at the most rows of one launch, and rows whose
# offsets pass 2^32 bytes
@pytest.mark.parametrize("kind,M,D,group", [(hkq.KIND_INT8, (1 << 26) - 4, 8, 0), (hkq.KIND_FP8, 270001, 8192, 128)])
def test_add_rmsnorm_quant_most_rows(kind, M, D, group):
    require_gpu()
    torch.cuda.empty_cache()
    x, res, w = gpu_bf16((M, D), 1), gpu_bf16((M, D), 2, 2.0), bf16((D,), 3)
    q, s, h = hkq.add_rmsnorm_quant(x, w.cuda(), res, 1e-6, kind, group)
    m = sampled(M, 200, *((1 << b) // (2 * D) for b in (31, 32)), *((1 << b) // D for b in (31, 32)))
    q = q.view(torch.uint8)[m].view(q.dtype)
    check_norm(x[m].cpu(), res[m].cpu(), w, 1e-6, group, kind, q, s[m], h[m])
