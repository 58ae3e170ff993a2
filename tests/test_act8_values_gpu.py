"""What a checkpoint of unusual codes and a gradient of unusual numbers stand for is the same in every call: NaN codes, infinities, what lies next to the largest float."""
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


@pytest.mark.parametrize("n,m,cols,pad", [(5, 33, 8, 0), (150, 130, 64, 0), (150, 100, 61, 1), (300, 260, 129, 3)])
def test_gradients_of_infinity_and_next_to_the_largest_float(cuda, n, m, cols, pad):
    import torch
    rng = np.random.default_rng(m)
    x = (2.0 ** -20 * (1 + rng.random((n, m)))).astype(np.float32) * rng.choice(np.array([-1, 1], np.float32), (n, m))
    x[rng.random((n, m)) < 0.05] = 0
    g = rng.standard_normal((n, cols + 2 * pad)).astype(np.float32)
    top = np.float32(3.4028235e38)
    edge = np.uint32(0x7f7f8000).view(np.float32)                 # the first number that bfloat16 rounds to infinity
    put = [np.inf, -np.inf, top, -top, edge, np.nextafter(edge, np.float32(0)), np.uint32(0x7f7f0001).view(np.float32), -np.uint32(0x7f7fabcd).view(np.float32)]
    for k, v in enumerate(put):
        g[rng.integers(n), pad + k % cols] = v
    if cols > len(put) + 2:                                       # infinities of both signs, and NaN, in a column
        g[0, pad + len(put)], g[n - 1, pad + len(put)], g[n // 2, pad + len(put) + 1] = np.inf, -np.inf, np.nan
    a, grad = A.act8_pack(torch.from_numpy(x).to(cuda)), torch.from_numpy(g).to(cuda)[:, pad:pad + cols]
    want, sums, bound, bound_b = _product(a, grad)
    assert np.isinf(want).any() and np.isnan(want).any() and np.isfinite(want[:, 2:8]).all()
    dw, db = A.act8_weight_grad(a, grad)
    _same(dw, want, bound)
    _same(db, sums, bound_b)
