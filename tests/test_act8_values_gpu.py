"""What a checkpoint of unusual codes stands for is the same in every call over it."""
import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F

pytestmark = pytest.mark.gpu


def _product(a, grad):
    """(X^T G, column sums, bound, bound) in float64 with infinities and NaN where the products and sums have them; the bounds are of the finite terms."""
    x, g = A.act8_unpack(a).cpu().numpy().astype(np.float64), grad.cpu().numpy().astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, sums = np.zeros((x.shape[1], g.shape[1])), np.zeros(g.shape[1])
        for xi, gi in zip(x, g):                       # no library product: its zeros times infinity are not always NaN
            want += xi[:, None] * gi[None, :]
            sums += gi
        fx, fg = np.where(np.isfinite(x), x, 0), np.where(np.isfinite(g), g, 0)
    _, bound, _, bound_b = F.weight_grad(fx, fg)
    return want, sums, bound, bound_b


def _same(got, want, bound):
    got = got.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    live = np.isfinite(want)
    assert (np.abs(got[live] - want[live]) <= bound[live]).all()


@pytest.mark.parametrize("n,m,cols", [(3, 40, 5), (200, 130, 132), (70, 300, 17)])
def test_nan_codes_are_nan_in_the_weight_gradient(cuda, n, m, cols):
    """A checkpoint put together from the caller's own codes: 0x7f and 0xff are e4m3's NaN at any scale, next to every other code."""
    import torch
    rng = np.random.default_rng(n)
    blocks = -(-m // 32)
    codes = torch.from_numpy(rng.integers(0, 256, (n, blocks * 32)).astype(np.uint8)).to(cuda)
    codes = torch.where(codes & 127 == 127, codes - 1, codes)
    scales = torch.from_numpy(rng.choice(np.array([120, 127, 134, 135, 140], np.uint8), (blocks, (n + 15) // 16 * 16))).to(cuda)
    for k in range(8):                                 # each place of a word, both signs
        codes[rng.integers(n), (5 * k) % m] = 0x7f + 128 * (k & 1)
    a = A.Act8(codes, scales, m)
    grad = torch.from_numpy(rng.standard_normal((n, cols)).astype(np.float32)).to(cuda)
    want, sums, bound, bound_b = _product(a, grad)
    assert 0 < np.isnan(want[:, 0]).sum() <= 8 and np.isnan(want).all(1).sum() == np.isnan(want[:, 0]).sum()
    dw, db = A.act8_weight_grad(a, grad)
    _same(dw, want, bound)
    _same(db, sums, bound_b)
    mask = A.act8_unpack(a) > 0
    assert torch.equal(A.act8_relu_backward(torch.ones(n, m, device=cuda), a) > 0, mask)
