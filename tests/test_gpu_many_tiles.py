"""GPU tests of products over so many groups and columns that their tiles pass what one
launch holds (2^32 threads). Whole numbers, exact in bf16 and fp32."""
import pytest
import torch

import hkq
from gpu_util import require_gpu
from test_gpu_w4 import MIDS

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(shape, seed, top=2):
    return torch.randint(-top, top + 1, shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def one_row_each(E):
    return torch.arange(E + 1, dtype=torch.int32, device="cuda")


def test_grouped_products_and_dx():
    require_gpu()
    E, C, S = 4096, 262208, 8  # 4097 column tiles of 64
    x, w = ints((E, S), 1), ints((C, S), 2)
    want = (x.float() @ w.float().t()).to(BF16)
    Y = torch.full((E, C), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_bf16(x, w[None].expand(E, C, S), one_row_each(E), Y)
    assert torch.equal(Y, want)
    Y.fill_(7.0)
    wt = w.t().contiguous()
    hkq.grouped_gemm_backward(x, torch.empty((E, C), dtype=BF16, device="cuda"), wt[None].expand(E, S, C), one_row_each(E), dX=Y, need_dw=False)
    assert torch.equal(Y, want)


def test_weight_gradients():
    """65535 groups of 258 tiles, three of them with rows."""
    require_gpu()
    E, N, K = 65535, 8, 66048
    rows = {0: 3, 40000: 2, 65534: 4}
    count = torch.zeros(E, dtype=torch.int32)
    for e, n in rows.items():
        count[e] = n
    offs = torch.cat((torch.zeros(1, dtype=torch.int32), count.cumsum(0).to(torch.int32))).cuda()
    X, dY = ints((9, K), 3), ints((9, N), 4)
    dW = torch.full((E, N, K), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_backward(dY, X, torch.zeros((1, 1, K), dtype=BF16, device="cuda").expand(E, N, K), offs, dW=dW, need_dx=False)
    at = 0
    for e, n in rows.items():
        assert torch.equal(dW[e], (dY[at:at + n].float().t() @ X[at:at + n].float()).to(BF16)), e
        dW[e] = 0
        at += n
    assert not any(bool(part.view(torch.int32).any()) for part in dW.split(2048))


@pytest.mark.parametrize("kind", ["int4", "mx"])
@pytest.mark.parametrize("rows,N", [(1, 65576), (3, 524360)], ids=["short", "tiles"])
def test_w4_products(rows, N, kind):
    """Every group's rows are the same, and so is its weight."""
    require_gpu()
    E, K = 4096, 32
    code = torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(5), dtype=torch.uint8)
    q = (code[:, 0::2] | (code[:, 1::2] << 4)).cuda()
    if kind == "mx":
        val, s = MIDS[code.long()], torch.full((N, 1), 127, dtype=torch.uint8, device="cuda")
    else:
        val, s = code.double() - 8, torch.ones((N, 1), dtype=BF16, device="cuda")
    x = ints((rows, K), 6, 1)
    want = (x.float() @ val.float().cuda().t()).to(BF16)
    Y = torch.full((E, rows, N), 7.0, dtype=BF16, device="cuda")
    hkq.grouped_gemm_w4a16(x.repeat(E, 1), q[None].expand(E, N, K // 2), s[None].expand(E, N, 1), one_row_each(E) * rows,
                           Y=Y.view(E * rows, N))
    assert all(bool((part == want).all()) for part in Y.split(512))
