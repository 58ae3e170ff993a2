"""Column sums over many row blocks of one slice: what the sum of the blocks rounds away in the same direction each time is not lost."""
import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad", [0, 1])
def test_sums_of_constant_columns(cuda, pad):
    """640 blocks in one slice (75 tiles of 256 kept columns by 128).  A block adds two chains of 32 numbers: 32 roundings of its sum at most, and the sum of the blocks is rounded
    once.  One chain over the blocks in float32 would be off by up to 154 roundings here."""
    import torch
    n, m, cols = 640 * 64, 1280, 1920
    a = A.act8_pack(torch.ones(n, m, device=cuda))
    value = (1 + torch.arange(cols + 2 * pad, device=cuda, dtype=torch.float64) / (cols + 2 * pad) * 2.0 ** -12).float()
    grad = value.expand(n, cols + 2 * pad).contiguous()[:, pad:pad + cols]
    _, db = A.act8_weight_grad(a, grad)
    want = grad[0].double() * n
    assert float(((db.double() - want).abs() / want).max()) <= 34 * F.U


def test_infinite_columns_in_many_blocks(cuda):
    import torch
    n, m, cols = 100 * 64, 1280, 1920
    a = A.act8_pack(torch.ones(n, m, device=cuda))
    grad = torch.ones(n, cols, device=cuda)
    grad[70, 3], grad[900, 5], grad[5000, 5], grad[n - 1, 7] = float("inf"), float("inf"), float("-inf"), float("nan")
    grad[:, 9] = -3e38                                            # beyond the largest float within two rows
    _, db = A.act8_weight_grad(a, grad)
    want = torch.full((cols,), float(n), device=cuda)
    want[3], want[5], want[7], want[9] = float("inf"), float("nan"), float("nan"), float("-inf")
    assert torch.equal(torch.nan_to_num(db, nan=-1.0), torch.nan_to_num(want, nan=-1.0)) and torch.equal(torch.isnan(db), torch.isnan(want))
