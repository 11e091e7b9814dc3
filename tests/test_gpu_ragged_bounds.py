"""GPU tests of bounds that are none: groups that all claim all rows, so many that their
tile counts add up past 32 bits. Nothing outside the operands is read or written."""
import pytest
import torch

import hkq
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("M", [(1 << 22) + 8, 3 << 21, 9 << 20])
def test_every_second_group_claims_all_rows(M):
    """65535 groups of one weight, bounds 0, M, 0, M, ..: the row tiles add up past 2^31. Rows are the weight's product,
    whoever computes them."""
    require_gpu()
    E, N, K = 65535, 8, 32
    offs = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offs[1::2] = M
    X = torch.zeros((M, K), dtype=BF16, device="cuda")
    X[:, 0] = (torch.arange(M, device="cuda") % 251).to(BF16)
    w = torch.zeros((N, K), dtype=BF16, device="cuda")
    w[:, 0] = torch.arange(N, device="cuda").to(BF16) / 8
    want = (X[:, :1].float() * w[:, 0].float()).to(BF16)
    buf = torch.full((M + 2, N), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_bf16(X, w[None].expand(E, N, K), offs, buf[1:-1])
    assert torch.equal(buf[1:-1], want) and (buf[0] == 7.0).all() and (buf[-1] == 7.0).all()
    q = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
    q[:, 0] = 0x88 + torch.arange(N, dtype=torch.uint8, device="cuda") % 8
    s = torch.full((N, 1), 0.125, dtype=BF16, device="cuda")
    buf.fill_(7.0)
    hkq.grouped_gemm_w4a16(X, q[None].expand(E, N, K // 2), s[None].expand(E, N, 1), offs, Y=buf[1:-1])
    assert torch.equal(buf[1:-1], want) and (buf[0] == 7.0).all() and (buf[-1] == 7.0).all()


def test_short_tiles():
    """The same on the 16-row tiles of short groups."""
    require_gpu()
    E, N, K = 65535, 64, 32
    M = 17 * E - 1
    offs = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offs[1::2] = M
    X = torch.ones((M, K), dtype=BF16, device="cuda")
    q = torch.full((N, K // 2), 0x99, dtype=torch.uint8, device="cuda")
    s = torch.full((N, 1), 0.125, dtype=BF16, device="cuda")
    buf = torch.full((M + 2, N), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_w4a16(X, q[None].expand(E, N, K // 2), s[None].expand(E, N, 1), offs, Y=buf[1:-1])
    assert (buf[1:-1] == 4.0).all() and (buf[0] == 7.0).all() and (buf[-1] == 7.0).all()
