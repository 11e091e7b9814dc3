"""Host-side check (no GPU needed) of how stacks of experts' weights are handed to the
4-bit quantizer: rows of one call below 2^22, at pitches that it takes, never a copy."""
import pytest
import torch

import hkq


def stack(E, N, K, stride_e, stride_n):
    return torch.empty(1, dtype=torch.bfloat16, device="meta").as_strided((E, N, K), (stride_e, stride_n, 1))


@pytest.mark.parametrize("t,calls", [
    (stack(3, 5, 64, 320, 64), 1), (stack(3, 5, 64, 640, 128), 1), (stack(3, 5, 64, 321, 64), 3), (stack(3, 5, 64, 0, 64), 3),
    (stack(1, 5, 64, 7, 64), 1), (stack(3, 1, 64, 640, 9), 1), (stack(3, 1, 64, 1 << 22, 64), 3), (stack(3, 1, 64, 0, 64), 3),
    (stack(1, 1, 64, 0, 0), 1), (stack(2, 1 << 21, 32, 32 << 21, 32), 2), (stack(2, (1 << 21) - 1, 32, 32 * ((1 << 21) - 1), 32), 1),
    (stack(2, 2, 64, 2 << 22, 1 << 22), 2), (stack(0, 5, 64, 0, 64), 1), (stack(4, 0, 64, 0, 64), 1)])
def test_rows_of_one_call(t, calls):
    rows, = hkq._experts(t)
    assert len(rows) == calls and sum(r.shape[0] for r in rows) == t.shape[0] * t.shape[1]
    for r in rows:
        assert r.dim() == 2 and r.shape[0] < 1 << 22
        if calls == 1 and r.shape[0] > 1:
            assert t.shape[2] <= r.stride(0) < 1 << 22 and r._base is not None


def test_one_tensor_apart_takes_all_apart():
    both = hkq._experts(stack(3, 5, 64, 320, 64), stack(3, 5, 32, 170, 32))
    assert [len(rows) for rows in both] == [3, 3]
