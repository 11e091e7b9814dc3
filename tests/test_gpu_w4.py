"""GPU tests of 4-bit weights: quantizer and dequantizer against the formulas, and the
products, dense and grouped, against their definition in 64 bits.

Tolerances of the products, from the arithmetic (U: half a step of bf16 relative to
the value, 2^-8; E: 2^-23, a step of fp32): a sum of K products in fp32 is off by at
most K E sum|products| in any order, the scales of the groups add one rounding each,
the rounding to bf16 adds U |value|. Worst cases add up with one sign; real errors do
not, so the 2-norm of a whole output's error is held to U as well.
"""
import pytest
import torch

import hkq
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

U, E32 = 2.0 ** -8, 2.0 ** -23
BF16 = torch.bfloat16
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf16(shape, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed)) * std).to(BF16)


# ------------------------------------------------------------------ quantizer

def quant_ref(w, group, zeros):
    """The formulas in fp32 on the CPU: (codes, scales, zero points)."""
    v = w.float().view(*w.shape[:-1], -1, group)
    tiny = 2.0 ** -126
    if zeros:
        lo, hi = v.amin(-1).clamp_max(0.0), v.amax(-1).clamp_min(0.0)
        s = (hi / 15.0 - lo / 15.0).to(BF16)
        inv = torch.where(s.float() >= tiny, 1.0 / s.float(), torch.zeros(()))
        z = torch.round(-lo * inv).clamp(0, 15)
        c = (torch.round(v * inv[..., None]) + z[..., None]).clamp(0, 15)
        return c.to(torch.uint8).flatten(-2), s, z.to(torch.uint8)
    s = (v.abs().amax(-1) / 7.0).to(BF16)
    inv = torch.where(s.float() >= tiny, 1.0 / s.float(), torch.zeros(()))
    c = torch.round(v * inv[..., None]).clamp(-8, 7) + 8
    return c.to(torch.uint8).flatten(-2), s, None


def unpack(q):
    return torch.stack((q & 15, q >> 4), -1).flatten(-2)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", [(1, 128), (3, 384), (257, 1408), (2, 5, 256), (1000, 128)])
def test_quantizer(shape, group, zeros):
    require_gpu()
    w = bf16(shape, sum(shape) + group, 0.02)
    w.view(-1, shape[-1])[0, :32] = 0.0  # with group 32 a whole group
    w.view(-1, shape[-1])[-1, -32:] = 0.3  # one value only, one sign
    got = hkq.w4_quant(w.cuda(), group, zeros)
    c, s, z = quant_ref(w, group, zeros)
    assert torch.equal(unpack(got[0].cpu()), c), "codes"
    assert torch.equal(got[1].cpu().view(torch.int16), s.view(torch.int16)), "scales"
    if zeros:
        assert torch.equal(got[2].cpu(), z), "zero points"
    back = hkq.w4_dequant(*got)
    off = z.float()[..., None] if zeros else 8.0
    ref = ((c.float().view(*s.shape, group) - off) * s.float()[..., None]).to(BF16).flatten(-2)
    assert torch.equal(back.cpu().view(torch.int16), ref.view(torch.int16)), "values"
    step = s.float().repeat_interleave(group, -1)
    # half a step, and what bf16 scales (2^-8 of up to 15 steps) and values add
    assert ((back.cpu().float() - w.float()).abs() <= step * (0.5 + 2 * 15 * U) + 1e-30).all()


def test_quantizer_special_groups_and_pitches():
    require_gpu()
    inf, G = float("inf"), 32
    w = bf16((9, 64), 3)
    w[0, 5] = NAN
    w[1, 40] = inf
    w[2, 3], w[2, 4] = inf, -inf
    w[3, :32] = 0.0
    w[4, :32] = 2.0 ** -130  # a scale below 2^-126: codes of zero
    w[5, :32] = 3.3895e38  # the largest magnitude
    w[6, :32] = -3.3895e38
    w[7, :16], w[7, 16:32] = 3.3895e38, -3.3895e38
    for zeros in (False, True):
        big = torch.full((9, 96), 9.0, dtype=BF16, device="cuda")
        big[:, :64] = w
        q = torch.full((9, 40), 77, dtype=torch.uint8, device="cuda")
        s = torch.full((9, 5), 5.0, dtype=BF16, device="cuda")
        z = torch.full((9, 5), 99, dtype=torch.uint8, device="cuda") if zeros else None
        hkq.w4_quant(big[:, :64], G, zeros, q[:, :32], s[:, :2], None if z is None else z[:, :2])
        assert (q[:, 32:] == 77).all() and (s[:, 2:] == 5.0).all() and (z is None or (z[:, 2:] == 99).all())
        v = hkq.w4_dequant(q[:, :32], s[:, :2], None if z is None else z[:, :2]).cpu().float()
        assert v[0, :32].isnan().all() and not v[0, 32:].isnan().any()
        assert not v[1, 32:].isfinite().any() and v[1, :32].isfinite().all()
        assert not v[2, :32].isfinite().any()
        assert (v[3, :32] == 0).all() and (v[4, :32] == 0).all()
        for r in (5, 6, 7):
            ok = (v[r, :32] - w[r, :32].float()).abs() <= 3.3895e38 * 0.04
            assert ok.all() or not zeros or r == 7  # 15 steps of a scale rounded up may pass the largest value
        c, s_ref, z_ref = quant_ref(w[3:5], G, zeros)
        assert torch.equal(unpack(q[3:5, :32].cpu()), c)


# ------------------------------------------------------------------- products

KINDS = [("int4", 128, False), ("int4", 128, True), ("int4", 64, True), ("int4", 32, False), ("int4", 32, True), ("mx", 32, False)]
MIDS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_of_experts_apart(zeros):
    """Halves of experts' rows in one buffer, quantized on another stream: what the experts
    give one by one, and nothing between them written."""
    both = bf16((3, 10, 256), 12).cuda()
    q = torch.full((3, 10, 128), 0xA5, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for half in (slice(0, 5), slice(5, 10)):
        got = hkq.w4_quant(both[:, half], 128, zeros, q=q[:, half], stream=stream)
        back = hkq.w4_dequant(*got, stream=stream)
        stream.synchronize()
        assert got[0].data_ptr() == q[:, half].data_ptr()
        for e in range(3):
            one = hkq.w4_quant(both[e, half].contiguous(), 128, zeros)
            assert all(torch.equal(a[e].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, one))
            assert torch.equal(back[e], hkq.w4_dequant(*one))
        if half.start == 0:
            assert (q[:, 5:] == 0xA5).all()


def weights(shape, kind, group, zeros, seed, pad=0):
    """Random codes, scales and zero points on the GPU, `pad` scales (NaN), and 16 pad bytes, past each row; and the values."""
    *lead, K = shape
    g = gen(seed)
    code = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8)
    G = K // group
    if kind == "mx":
        s = torch.randint(118, 124, (*lead, G), generator=g, dtype=torch.uint8)
        val = (MIDS[code.long()].view(*lead, G, group) * torch.pow(2.0, s.double() - 127)[..., None]).view(shape)
        z = None
    else:
        s = ((0.5 + torch.rand((*lead, G), generator=g)) / 64).to(BF16)
        z = torch.randint(0, 16, (*lead, G), generator=g, dtype=torch.uint8) if zeros else None
        off = z.double()[..., None] if zeros else 8.0
        val = ((code.double().view(*lead, G, group) - off) * s.double()[..., None]).view(shape)
    q = code[..., 0::2] | (code[..., 1::2] << 4)

    def padded(t, n, fill):
        if t is None:
            return None
        b = torch.full((*t.shape[:-1], t.shape[-1] + n), fill, dtype=t.dtype, device="cuda")
        b[..., :t.shape[-1]] = t.cuda()
        return b[..., :t.shape[-1]]

    return padded(q, 16 if pad else 0, 255), padded(s, pad, 255 if kind == "mx" else NAN), padded(z, pad, 255), val.cuda()


def close(got, ref, mag, terms, what):
    got = got.double()
    tol = U * ref.abs() + (terms + 8) * E32 * mag + 1e-38
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {got[i]} ref {ref[i]} tol {tol[i]}")
    if ref.numel() >= 1024:
        assert float((got - ref).norm() / ref.norm()) <= U, what


def rows_of(M, K, seed, pad=0):
    X = torch.full((M, K + pad), NAN, dtype=BF16, device="cuda")
    X[:, :K] = bf16((M, K), seed)
    return X[:, :K]


def check_dense(M, N, K, kind, group, zeros, pad=0, seed=0):
    q, s, z, val = weights((N, K), kind, group, zeros, seed + 1, pad)
    X = rows_of(M, K, seed, 8 if pad else 0)
    buf = torch.full((M + 2, N + pad), 7.0, dtype=BF16, device="cuda")
    C = buf[1:M + 1, :N]
    assert hkq.gemm_w4a16(X, q, s, z, C) is C
    x = X.double().contiguous()
    close(C, x @ val.t(), x.abs() @ val.abs().t(), K, f"{M}x{N}x{K} {kind} {group} {zeros}")
    assert (buf[0] == 7.0).all() and (buf[M + 1] == 7.0).all() and (buf[:, N:] == 7.0).all(), "written around the output"


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 40, 64, 65, 130, 300])
def test_dense(M, kind, group, zeros):
    require_gpu()
    for N, K in ((1, group), (33, 3 * group), (200, 1408), (64, 4096), (1000, 640)):
        check_dense(M, N, K, kind, group, zeros, seed=M + N)


@pytest.mark.parametrize("kind,group,zeros", KINDS)
def test_dense_short_and_ragged_k(kind, group, zeros):
    require_gpu()
    for i in range(1, 12):
        for M in (1, 20, 150):
            check_dense(M, 70, i * group, kind, group, zeros, pad=i, seed=i)


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 14336), (16, 14336, 4096), (48, 4096, 4096), (200, 4096, 2048), (600, 2816, 2048),
                                   (1030, 1408, 4096), (3, 13001, 544), (7, 13001, 544), (12, 13001, 544), (29, 13001, 544)])
def test_dense_layer_sizes(M, N, K, kind, group, zeros):
    """Many columns (the last four: ragged ones) take more of them per workgroup."""
    require_gpu()
    K = K // group * group
    check_dense(M, N, K, kind, group, zeros, seed=3)


def check_grouped(rows, N, K, kind, group, zeros, first=0, tail=0, topk=0, pad=0, seed=0):
    o = [first]
    for r in rows:
        o.append(o[-1] + r)
    M, E = o[-1] + tail, len(rows)
    q, s, z, val = weights((E, N, K), kind, group, zeros, seed + 1, pad)
    offs = torch.tensor(o, dtype=torch.int32, device="cuda")
    if topk:
        T = (M + topk - 1) // topk
        gather = torch.randperm(T * topk, generator=gen(seed + 2))[:M].to(torch.int32)
        if M > 2:
            gather[1], gather[2] = -1, T * topk + 5  # rows outside X: zeros
        X = rows_of(T, K, seed, pad * 8)
        x = torch.cat((X.double(), torch.zeros((1, K), dtype=torch.float64, device="cuda")))
        src = torch.where((gather >= 0) & (gather < T * topk), gather // topk, T).cuda().long()
        x, gather = x[src], gather.cuda()
    else:
        X, gather = rows_of(M, K, seed, pad * 8), None
        X[:first] = NAN
        X[o[-1]:] = NAN
        x = X.double().contiguous()
    buf = torch.full((M + 2, N + pad), 7.0, dtype=BF16, device="cuda")
    Y = buf[1:M + 1, :N]
    assert hkq.grouped_gemm_w4a16(X, q, s, offs, z, gather, max(1, topk), Y) is Y
    for e in range(E):
        r = slice(o[e], o[e + 1])
        close(Y[r], x[r] @ val[e].t(), x[r].abs() @ val[e].abs().t(), K, f"group {e} of {rows} {N}x{K} {kind} {group} {zeros}")
    assert (Y[:first] == 7.0).all() and (Y[o[-1]:] == 7.0).all(), "rows of no group written"
    assert (buf[0] == 7.0).all() and (buf[M + 1] == 7.0).all() and (buf[:, N:] == 7.0).all(), "written around the output"


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("rows", [[1], [0, 1, 0, 1], [5, 0, 17, 16, 1], [64, 65, 3], [200, 0, 130], [2] * 70 + [0] * 60 + [40],
                                  [700, 1, 1, 1, 0, 90]], ids=lambda r: f"{len(r)}x{max(r)}")
def test_grouped(rows, kind, group, zeros):
    require_gpu()
    check_grouped(rows, 72, 5 * group, kind, group, zeros, topk=3, seed=1)
    check_grouped(rows, 130, 2 * group, kind, group, zeros, first=3, tail=20, pad=2, seed=2)


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("rows,N,K,topk", [([1, 0, 0, 0, 0, 1, 0, 0], 28672, 1024, 2), ([94] * 16, 2816, 2048, 6), ([6, 9, 3, 0, 11, 7, 1, 9], 4096, 3584, 2)])
def test_grouped_layer_sizes(rows, N, K, topk, kind, group, zeros):
    require_gpu()
    check_grouped(rows, N, K, kind, group, zeros, topk=topk, seed=4)


@pytest.mark.parametrize("kind,group,zeros", KINDS)
def test_grouped_short_groups_of_many_columns(kind, group, zeros):
    """Means of 3 to 16 rows, where streams and tiles take over from each other."""
    require_gpu()
    check_grouped([3, 9, 0, 5, 33, 1, 2, 17, 4, 0, 6, 8, 3, 1, 40, 2], 5632, 1024, kind, group, zeros, first=2, tail=3, topk=3, seed=21)
    check_grouped([3, 2, 4, 0, 5, 17, 1, 3], 4104, 1152, kind, group, zeros, tail=1, seed=22)


def test_mxfp4_scales():
    """Every e8m0 code, 255 as NaN; products with one value of X, so that nothing cancels."""
    require_gpu()
    K, N = 256, 256
    code = torch.arange(16, dtype=torch.uint8).repeat(16)
    q = (code[0::2] | (code[1::2] << 4)).repeat(N, 1).cuda()
    s = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, K // 32).cuda()
    val = MIDS[code.long()][None] * torch.pow(2.0, torch.arange(256).double() - 127)[:, None]
    for k in (1, 7, 9, 15):
        for M in (1, 40, 300):
            X = torch.zeros((M, K), dtype=BF16, device="cuda")
            X[:, k] = 1.0
            C = hkq.gemm_w4a16(X, q, s).cpu().double()
            ref = val[:, k].float().to(BF16).double()  # beyond the largest bf16: an infinity
            # the operand is bf16: below its smallest normal number a value may be flushed
            ok = (C[:, :255] == ref[:255]) | ((ref[:255].abs() < 2.0 ** -126) & (C[:, :255].abs() < 2.0 ** -126))
            fin = torch.isfinite(torch.tensor(6.0) * torch.pow(2.0, torch.arange(255).double() - 127).float())
            assert ok[:, fin].all(), (k, M, (~ok[:, fin]).nonzero()[:4])
            assert C[:, 255].isnan().all()


def test_weights_of_other_layouts():
    """Groups side by side in each row, one weight for all groups, scales of odd pitch."""
    require_gpu()
    E, N, K, rows = 3, 40, 160, [5, 0, 70]
    q, s, z, val = weights((N, E, K), "int4", 32, True, 1)
    offs = torch.tensor([0, 5, 5, 75], dtype=torch.int32, device="cuda")
    X = rows_of(75, K, 2)
    Y = hkq.grouped_gemm_w4a16(X, q.transpose(0, 1), s.transpose(0, 1), offs, z.transpose(0, 1))
    ref = hkq.grouped_gemm_w4a16(X, q.transpose(0, 1).contiguous(), s.transpose(0, 1).contiguous(), offs, z.transpose(0, 1).contiguous())
    assert torch.equal(Y, ref)
    one = [t[:, 0].contiguous()[None].expand(E, N, -1) for t in (q, s, z)]
    Y = hkq.grouped_gemm_w4a16(X, one[0], one[1], offs, one[2])
    close(Y, X.double() @ val[:, 0].t(), X.double().abs() @ val[:, 0].abs().t(), K, "one weight")


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("M", [1, 7, 16, 30, 100])
def test_nan_infinity_and_zero_weights(M, kind, group, zeros):
    """An infinity in X gives what the weight at its place makes of it: a signed infinity, or NaN where that is zero; it and
    a NaN stay in their rows. Weights of zero give zeros, whatever X."""
    require_gpu()
    N, K = 70, 4 * group
    q, s, z, val = weights((N, K), kind, group, zeros, 5)
    q[9] = 0 if kind == "mx" else 0x88
    if z is not None:
        z[9] = 8
    val[9] = 0
    X = rows_of(M, K, 6)
    clean = hkq.gemm_w4a16(X, q, s, z)
    assert (clean[:, 9] == 0).all()
    at = group + 3
    X[M - 1, at] = float("inf")
    C = hkq.gemm_w4a16(X, q, s, z)
    assert torch.equal(C[:-1], clean[:-1])
    v = val[:, at]
    assert torch.equal(C[-1].isnan(), v == 0) and torch.equal(C[-1][v != 0] > 0, v[v != 0] > 0) and not C[-1].isfinite().any()
    X[M - 1, at] = NAN
    assert hkq.gemm_w4a16(X, q, s, z)[-1].isnan().all()
    # a NaN scale reaches the outputs of its column only (test_mxfp4_scales: MXFP4's)
    if kind == "int4":
        X[M - 1, at] = 1.0
        s[3, 1] = NAN
        C = hkq.gemm_w4a16(X, q, s, z)
        assert C[:, 3].isnan().all() and C[:, :3].isfinite().all() and C[:, 4:].isfinite().all()


def test_no_rows_no_sums():
    require_gpu()
    q, s, z, _ = weights((24, 64), "int4", 32, True, 1)
    X = torch.empty((0, 64), dtype=BF16, device="cuda")
    assert hkq.gemm_w4a16(X, q, s, z).shape == (0, 24)
    offs = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert hkq.grouped_gemm_w4a16(X, q[None], s[None], offs, z[None]).shape == (0, 24)
    empty = [t[:, :0] for t in (q, s)]
    for M in (1, 20, 100):
        C = hkq.gemm_w4a16(torch.empty((M, 0), dtype=BF16, device="cuda"), *empty, C=torch.full((M, 24), 7.0, dtype=BF16, device="cuda"))
        assert (C == 0).all()


@pytest.mark.parametrize("M", [3, 300])
def test_gather_from_no_rows(M):
    """An X without rows, whatever its pitch: every gathered row counts as zeros."""
    N, K = 64, 256
    Q = torch.full((1, N, K // 2), 0x21, dtype=torch.uint8, device="cuda")
    S = torch.ones((1, N, K // 128), dtype=torch.bfloat16, device="cuda")
    X = torch.ones((4, 2 * K), dtype=torch.bfloat16, device="cuda")
    offs = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    gather = torch.arange(M, dtype=torch.int32, device="cuda") - 1
    for pitch in (K, 2 * K, 1 << 20):
        Y = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
        hkq.call("hkq_grouped_gemm_w4a16", X.data_ptr(), Q.data_ptr(), S.data_ptr(), 0, Y.data_ptr(), offs.data_ptr(), gather.data_ptr(),
                 M, 0, 1, N, K, 1, pitch, K // 2, N * K // 2, K // 128, N * K // 128, N, 128, hkq.W4_INT4, 0, 0,
                 torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert (Y == 0).all()


@pytest.mark.parametrize("kind,group,zeros", [("int4", 64, True), ("mx", 32, False)])
def test_offsets_past_32_bits(kind, group, zeros):
    """Codes of 5.4 GB, rows and outputs of 2.4 GB."""
    require_gpu()
    E, N, K = 80, 16384, 8192
    q, s, z, val = weights((64, K), kind, group, zeros, 1)
    Q = torch.zeros((E, N, K // 2), dtype=torch.uint8, device="cuda")
    S = torch.zeros((E, N, K // group), dtype=s.dtype, device="cuda")
    Z = torch.zeros((E, N, K // group), dtype=torch.uint8, device="cuda") if zeros else None
    for e in (0, E - 1):
        Q[e, -64:], S[e, -64:] = q, s
        if zeros:
            Z[e, -64:] = z
    for rows in ([1] + [0] * (E - 2) + [3], [70] + [0] * (E - 2) + [130]):
        M = sum(rows)
        offs = torch.tensor([0] + [rows[0]] * (E - 1) + [M], dtype=torch.int32, device="cuda")
        X = rows_of(M, K, 2)
        Y = hkq.grouped_gemm_w4a16(X, Q, S, offs, Z)
        close(Y[:, -64:], X.double() @ val.t(), X.double().abs() @ val.abs().t(), K, "last columns")
    del Q, S, Z
    M, K, N = 300000, 4096, 4096
    q, s, z, val = weights((N, K), kind, group, zeros, 3)
    X = torch.zeros((M, K), dtype=BF16, device="cuda")
    X[-300:] = bf16((300, K), 4)
    C = hkq.gemm_w4a16(X, q, s, z)
    x = X[-300:].double()
    close(C[-300:], x @ val.t(), x.abs() @ val.abs().t(), K, "last rows")
    assert (C[:-300] == 0).all()


def test_streams_and_graphs():
    """On a stream of the caller's, several at once, and captured: every replay as the eager call, with eager work between."""
    require_gpu()
    sets = []
    for i, (M, N, K, (kind, group, zeros)) in enumerate([(1, 512, 1024, KINDS[1]), (13, 300, 640, KINDS[4]), (40, 256, 384, KINDS[5]),
                                                         (200, 520, 512, KINDS[0])]):
        q, s, z, _ = weights((2, N, K), kind, group, zeros, i)
        offs = torch.tensor([0, M // 3, M], dtype=torch.int32, device="cuda")
        sets.append((rows_of(M, K, i + 9), q, s, z, offs))
    w = bf16((96, 256), 30).cuda()

    def run(x, q, s, z, offs, stream=None):
        a = hkq.gemm_w4a16(x, q[0], s[0], z[0] if z is not None else None, stream=stream)
        b = hkq.grouped_gemm_w4a16(x, q, s, offs, z, stream=stream)
        c = hkq.w4_quant(w, 64, True, stream=stream)
        return (a, b, *c, hkq.w4_dequant(*c, stream=stream))

    eager = [run(*t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        out = [run(*t, stream=st) for t, st in zip(sets, streams)]
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        out = [run(*t) for t in sets]
    for _ in range(3):
        for o in out:
            for t in o:
                t.fill_(3)
        g.replay()
        run(*sets[0])
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_hipkittens_module():
    require_gpu()
    import hipkittens as hk

    w, X = bf16((48, 256), 1).cuda(), rows_of(20, 256, 2)
    q, s, z = (torch.empty((48, n), dtype=t, device="cuda") for n, t in ((128, torch.uint8), (4, BF16), (4, torch.uint8)))
    hk.w4.w4_quant(w, q, s, z)
    ref = hkq.w4_quant(w, 64, True)
    assert all(torch.equal(a, b) for a, b in zip((q, s, z), ref))
    out, C = torch.empty_like(w), torch.empty((20, 48), dtype=BF16, device="cuda")
    hk.w4.w4_dequant(q, s, out, z)
    hk.w4.gemm_w4a16(X, q, s, C, z)
    assert torch.equal(out, hkq.w4_dequant(q, s, z)) and torch.equal(C, hkq.gemm_w4a16(X, q, s, z))
    offs = torch.tensor([0, 7, 20], dtype=torch.int32, device="cuda")
    Q, S = torch.stack((q, q.flip(0))), torch.stack((s, s.flip(0)))
    gather = torch.randperm(20, generator=gen(3)).to(torch.int32).cuda()
    Y = torch.empty((20, 48), dtype=BF16, device="cuda")
    hk.w4.grouped_gemm_w4a16(X[:10], Q, S, Y, offs, gather=gather, topk=2)
    assert torch.equal(Y, hkq.grouped_gemm_w4a16(X[:10], Q, S, offs, None, gather, 2))
    mq, ms = hkq.mx_quant(w, True)
    hk.w4.gemm_w4a16(X, mq, ms, C)
    assert torch.equal(C, hkq.gemm_w4a16(X, mq, ms))
    with pytest.raises(ValueError, match="scale per"):
        hk.w4.gemm_w4a16(X, q, s[:, :1].contiguous(), C)
    with pytest.raises(TypeError, match="Q"):
        hk.w4.gemm_w4a16(X, q.float(), s, C)
    with pytest.raises(ValueError, match="zero points"):
        hk.w4.gemm_w4a16(X, mq, ms, C, ms)


def test_quantized_weights_through_the_products():
    """w4_quant's and mx_quant's outputs as the products take them."""
    require_gpu()
    w, X = bf16((200, 512), 1, 0.05).cuda(), rows_of(37, 512, 2)
    for group, zeros in ((32, True), (64, False), (128, True), (128, False)):
        t = hkq.w4_quant(w, group, zeros)
        c = unpack(t[0]).double().view(200, -1, group)
        val = ((c - (t[2].double()[..., None] if zeros else 8.0)) * t[1].double()[..., None]).view(200, 512)
        close(hkq.gemm_w4a16(X, *t), X.double() @ val.t(), X.double().abs() @ val.abs().t(), 512, f"{group} {zeros}")
    q, s = hkq.mx_quant(w, True)
    val = hkq.mx_dequant(q, s, 512, True).double()
    close(hkq.gemm_w4a16(X, q, s), X.double() @ val.t(), X.double().abs() @ val.abs().t(), 512, "mx")
