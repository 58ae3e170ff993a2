"""8-bit checkpoints: codes, scales and values equal to a float64 restatement, the ReLU mask, and the weight gradient over the kept values."""
import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F

pytestmark = pytest.mark.gpu


def _np(t):
    return t.float().cpu().numpy()


def _hard(rng, n, cols):
    """Values over many binades, ties, zeros of both signs, subnormal numbers, the largest float, blocks of zeros."""
    x = (rng.standard_normal((n, cols)) * 2.0 ** rng.integers(-30, 30, (n, 1))).astype(np.float32)
    x.flat[::7] = (rng.integers(-40, 41, x.flat[::7].size) / 32).astype(np.float32)
    for v in (0.0, -0.0, 448.0, -464.0, 465.0, 1e-45, -1e-40, 3.4e38, 2.0 ** -126):
        x.flat[rng.integers(0, x.size, max(1, x.size // 60))] = v
    x[rng.integers(0, n, max(1, n // 8))] = 0
    return x


@pytest.mark.parametrize("n,cols", [(1, 1), (3, 4), (4, 31), (5, 32), (17, 33), (64, 128), (33, 384), (9, 100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["whole", "aligned", "odd"])
def test_pack_and_unpack(cuda, n, cols, dtype, layout):
    import torch
    rng = np.random.default_rng(n * 100 + cols)
    pad = dict(whole=0, aligned=8, odd=3)[layout]
    x = torch.from_numpy(_hard(rng, n, cols + 2 * pad)).to(cuda).to(torch.bfloat16 if dtype == "bf16" else torch.float32)[:, pad:pad + cols]
    codes, scales, values = F.pack(x.float().cpu().numpy())
    a = A.act8_pack(x)
    assert a.shape == (n, cols)
    assert np.array_equal(a.codes.cpu().numpy(), codes) and np.array_equal(a.scales.cpu().numpy()[:, :n], scales)
    got = A.act8_unpack(a).cpu().numpy()
    assert np.array_equal(got.astype(np.float64), values, equal_nan=True)
    fine = x.float().cpu().numpy().astype(np.float64)
    step = 2.0 ** (np.repeat(scales.T[:, :, None].astype(np.float64), 32, 2).reshape(n, -1)[:, :cols] - 127 - 9)
    with np.errstate(invalid="ignore"):
        assert ((np.abs(got - fine) <= np.maximum(np.abs(fine) / 16, step)) | np.isnan(values)).all()
        assert (((got != 0) == (fine != 0)) | np.isnan(values)).all() and ((np.sign(got) == np.sign(fine)) | np.isnan(values)).all()


def test_a_block_with_infinity_or_nan_is_nan(cuda):
    import torch
    x = torch.ones(6, 70, device=cuda)
    x[1, 3], x[2, 40], x[4, 69] = float("inf"), float("nan"), float("-inf")
    got = A.act8_unpack(A.act8_pack(x))
    want = torch.ones_like(x)
    want[1, :32] = want[2, 32:64] = want[4, 64:] = float("nan")
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])
    dw, db = A.act8_weight_grad(A.act8_pack(x), torch.ones(6, 5, device=cuda))
    assert torch.isnan(dw).all() and torch.equal(db, torch.full((5,), 6.0, device=cuda))
    clean = torch.ones(6, 70, device=cuda)
    clean[1, 3] = float("nan")                                   # one block of one row: its 32 rows of the gradient
    dw, _ = A.act8_weight_grad(A.act8_pack(clean), torch.ones(6, 5, device=cuda))
    assert torch.isnan(dw[:32]).all() and torch.equal(dw[32:], torch.full((38, 5), 6.0, device=cuda))
    assert not A.act8_relu_backward(torch.ones_like(x), A.act8_pack(x))[1, :32].any()


@pytest.mark.parametrize("n,cols", [(1, 1), (7, 31), (50, 512), (33, 130), (4, 4)])
@pytest.mark.parametrize("layout", ["whole", "aligned", "odd"])
def test_relu_mask(cuda, n, cols, layout):
    import torch
    rng = np.random.default_rng(cols)
    h = torch.relu(torch.from_numpy(_hard(rng, n, cols)).to(cuda))
    pad = dict(whole=0, aligned=8, odd=3)[layout]
    grad = torch.randn(n, cols + 2 * pad, device=cuda)[:, pad:pad + cols]
    a = A.act8_pack(h)
    want = torch.where(h > 0, grad, torch.zeros_like(grad))
    assert torch.equal(A.act8_relu_backward(grad, a), want)
    if layout == "whole":
        same = grad.clone()
        assert A.act8_relu_backward(same, a, out=same) is same and torch.equal(same, want)


def _weight_case(torch, cuda, n, m, cols, seed, pad=0, spread=0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, m)).astype(np.float32)
    g = rng.standard_normal((n, cols + 2 * pad)).astype(np.float32)
    if spread:
        x *= 2.0 ** rng.integers(-spread, spread, (n, 1))
        g *= 2.0 ** rng.integers(-spread, spread, g.shape)
    a = A.act8_pack(torch.from_numpy(x.astype(np.float32)).to(cuda))
    grad = torch.from_numpy(g.astype(np.float32)).to(cuda)[:, pad:pad + cols]
    return a, grad


def _check_weight(a, grad):
    dw, db = A.act8_weight_grad(a, grad)
    values = _np(A.act8_unpack(a))
    want, bound, want_b, bound_b = F.weight_grad(values, _np(grad))
    assert dw.shape == want.shape and (np.abs(_np(dw) - want) <= bound).all(), float((np.abs(_np(dw) - want) / np.maximum(bound, 1e-300)).max())
    assert (np.abs(_np(db) - want_b) <= bound_b).all()
    return dw, db


@pytest.mark.parametrize("n,m,cols", [(1, 1, 1), (2, 33, 5), (15, 16, 16), (64, 128, 128), (63, 129, 127), (65, 130, 4), (128, 256, 64), (200, 257, 129),
                                      (300, 384, 1536), (257, 1536, 384), (1000, 64, 256), (5000, 100, 68), (20_003, 128, 128), (3, 700, 300)])
def test_weight_gradient(cuda, n, m, cols):
    import torch
    a, grad = _weight_case(torch, cuda, n, m, cols, n + m)
    dw, db = _check_weight(a, grad)
    again = A.act8_weight_grad(a, grad)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])                       # repeatable bit for bit
    out = torch.full((m, cols), float("nan"), device=cuda)
    got, none = A.act8_weight_grad(a, grad, out=out, bias_grad=False)
    assert got is out and none is None and torch.equal(out, dw)
    # the usual accuracy, not only the worst case of any order: the relative error of the whole matrix stays a few roundings
    want = _np(A.act8_unpack(a)).astype(np.float64).T @ _np(grad).astype(np.float64)
    assert np.linalg.norm(_np(dw) - want) <= 16 * F.U * np.sqrt(max(np.log2(n + 1), 1)) * np.linalg.norm(np.abs(_np(A.act8_unpack(a))).T.astype(np.float64) @ np.abs(_np(grad)))


@pytest.mark.parametrize("n,m,cols,pad", [(500, 96, 64, 8), (500, 96, 61, 3), (130, 300, 200, 1)])
def test_weight_gradient_of_strided_rows(cuda, n, m, cols, pad):
    import torch
    _check_weight(*_weight_case(torch, cuda, n, m, cols, 5, pad=pad))


def test_weight_gradient_over_many_binades(cuda):
    """Rows of every size next to one another: each entry stays within the bound of its own terms."""
    import torch
    _check_weight(*_weight_case(torch, cuda, 700, 128, 128, 8, spread=20))
    _check_weight(*_weight_case(torch, cuda, 90, 40, 24, 9, spread=45))


def test_no_rows(cuda):
    import torch
    a = A.act8_pack(torch.empty(0, 40, device=cuda))
    assert A.act8_unpack(a).shape == (0, 40) and A.act8_relu_backward(torch.empty(0, 40, device=cuda), a).shape == (0, 40)
    dw, db = A.act8_weight_grad(a, torch.empty(0, 8, device=cuda))
    assert not dw.any() and not db.any() and dw.shape == (40, 8)


def test_captured_and_replayed(cuda):
    import torch
    x, y, g = torch.randn(700, 128, device=cuda), torch.randn(700, 256, device=cuda), torch.randn(700, 256, device=cuda)

    def step():
        a, h = A.act8_pack(x), A.act8_pack(torch.relu(y))
        masked = A.act8_relu_backward(g, h)
        return (A.act8_unpack(a), masked) + A.act8_weight_grad(a, masked)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in (x, y, g):
        t.copy_(torch.randn_like(t))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
