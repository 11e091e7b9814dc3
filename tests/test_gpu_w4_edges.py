"""GPU tests of the 4-bit weights at the edges of what their calls take: the largest
values, expert stacks past one call's rows, scales at any address, ends of the e8m0
range, more tiles than one launch holds."""
import pytest
import torch

import hkq
from gpu_util import require_gpu
from test_gpu_w4 import BF16, MIDS, bf16, close, quant_ref, unpack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_of_the_largest_values(group, zeros):
    """Near the largest bf16: codes, scales and zero points as the formulas give them, and values bf16((code - zero) * scale),
    an infinity exactly where that passes the largest bf16."""
    require_gpu()
    top = 3.3895e38
    w = bf16((6, 2 * group), 3)
    w[0, :group], w[1, group:] = top, -top
    w[2, :group // 2], w[2, group // 2:group] = top, -top
    w[3, 5], w[4, group + 1] = top, -top
    w[5, ::3], w[5, 1::3] = top, -0.5 * top
    assert w.isfinite().all()
    c, s, z = quant_ref(w, group, zeros)
    assert s.isfinite().all() and int(c.max()) == 15
    got = hkq.w4_quant(w.cuda(), group, zeros)
    assert torch.equal(unpack(got[0].cpu()), c), "codes"
    assert torch.equal(got[1].cpu().view(torch.int16), s.view(torch.int16)), "scales"
    assert not zeros or torch.equal(got[2].cpu(), z), "zero points"
    off = z.float()[..., None] if zeros else 8.0
    ref = ((c.float().view(*s.shape, group) - off) * s.float()[..., None]).to(BF16).flatten(-2)
    back = hkq.w4_dequant(*got).cpu()
    assert torch.equal(back.view(torch.int16), ref.view(torch.int16)), "values"
    fin = ref.isfinite()
    assert ((back.float() - w.float()).abs()[fin] <= (s.float().repeat_interleave(group, -1) * (0.5 + 2 * 15 * 2.0 ** -8))[fin]).all()


@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_of_more_rows_than_a_call_takes(zeros):
    """2^22 rows of two experts: past one call's limit, so one for each."""
    require_gpu()
    w = torch.zeros((2, 1 << 21, 32), dtype=BF16, device="cuda")
    rows = [0, 1, 77777, (1 << 21) - 1]
    w[:, rows] = bf16((2, 4, 32), 1).cuda()
    got = hkq.w4_quant(w, 32, zeros)
    c, s, z = quant_ref(w[:, rows].cpu(), 32, zeros)
    assert torch.equal(unpack(got[0][:, rows].cpu()), c) and torch.equal(got[1][:, rows].cpu(), s)
    assert not zeros or torch.equal(got[2][:, rows].cpu(), z)
    back = hkq.w4_dequant(*got)
    assert torch.equal(back[:, rows], torch.stack([hkq.w4_dequant(*(t[e][rows].contiguous() for t in got)) for e in range(2)]))
    assert (back[:, 2:77777] == 0).all()


def test_quantizer_of_one_row_of_each_expert():
    """A row of each expert's matrix, the experts 2^22 values apart, and one row for all of them."""
    require_gpu()
    whole = bf16((3, 4, 1 << 20), 2).cuda()
    for w in (whole[:, 1:2, :256], whole[:1, :1, :256].expand(3, 1, 256)):
        got = hkq.w4_quant(w, 64, True)
        ref = hkq.w4_quant(w.contiguous(), 64, True)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
        assert torch.equal(hkq.w4_dequant(*got), hkq.w4_dequant(*ref))


@pytest.mark.parametrize("M", [1, 7, 16, 30, 100, 300])
def test_mxfp4_scales_at_any_address(M):
    """e8m0 scales are bytes: rows of any pitch from any address."""
    require_gpu()
    N, K = 133, 416
    g = torch.Generator().manual_seed(M)
    code = torch.randint(0, 16, (2, N, K), generator=g, dtype=torch.uint8)
    sc = torch.randint(118, 124, (2, N, K // 32), generator=g, dtype=torch.uint8)
    q = (code[..., 0::2] | (code[..., 1::2] << 4)).cuda()
    val = (MIDS[code.long()].view(2, N, -1, 32) * torch.pow(2.0, sc.double() - 127)[..., None]).view(2, N, K).cuda()
    X = bf16((M, K), M + 1).cuda()
    x, offs = X.double(), torch.tensor([0, M // 3, M], dtype=torch.int32, device="cuda")
    for at in (1, 2, 3):
        for pitch in (13, 14, 16):
            buf = torch.full((at + 2 * N * pitch,), 255, dtype=torch.uint8, device="cuda")
            S = buf.as_strided((2, N, K // 32), (N * pitch, pitch, 1), at)
            S.copy_(sc)
            close(hkq.gemm_w4a16(X, q[0], S[0]), x @ val[0].t(), x.abs() @ val[0].abs().t(), K, f"{at} {pitch}")
            Y = hkq.grouped_gemm_w4a16(X, q, S, offs)
            for e, r in enumerate((slice(0, M // 3), slice(M // 3, M))):
                close(Y[r], x[r] @ val[e].t(), x[r].abs() @ val[e].abs().t(), K, f"group {e}, {at} {pitch}")


@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_mxfp4_ends_of_the_scales(M):
    """A code by itself in its row, under each scale byte: exact down to the smallest (2^-128, below bf16's normal numbers),
    up to where a value is 2^128 or more and the weight an infinity, as mx_dequant has it. Powers of two as X."""
    require_gpu()
    N, K = 255 * 16, 64
    e, c = torch.arange(255).repeat_interleave(16), torch.arange(16, dtype=torch.uint8).repeat(255)
    val = MIDS[c.long()] * torch.pow(2.0, e.double() - 127)
    over = val.abs() >= 2.0 ** 128
    assert sorted(set(e[over].tolist())) == [253, 254] and int(over.sum()) == 4 + 8
    s = e.to(torch.uint8)[:, None].expand(N, 2).contiguous().cuda()
    for k in (0, 13, 39, 63):
        q = torch.zeros((N, K // 2), dtype=torch.uint8)
        q[:, k // 2] = c << (4 * (k % 2))
        q = q.cuda()
        w = hkq.mx_dequant(q, s, K).cpu().double()
        assert torch.equal(w[:, k], torch.where(over, val.sign() * float("inf"), val))
        for x in (1.0, -2.0 ** -20, 2.0 ** 60, 2.0 ** -3):
            X = torch.full((M, K), x, dtype=BF16, device="cuda")
            # one rounding of the exact product (fp32 holds it or rounds as bf16 does: two significant bits)
            ref = torch.where(over, val.sign() * x * float("inf"), val * x).float().to(BF16)
            C = hkq.gemm_w4a16(X, q, s).cpu()
            Y = hkq.grouped_gemm_w4a16(X, q[None], s[None], torch.tensor([0, M], dtype=torch.int32, device="cuda")).cpu()
            assert torch.equal(C, ref.expand(M, N)) and torch.equal(Y, C), (k, x)
    X[:] = 0.0
    C = hkq.gemm_w4a16(X, q, s).cpu()
    assert torch.equal(C.isnan(), over.expand(M, N)) and (C[:, ~over] == 0).all()
