"""qk_norm_rope and its backward against float64: head widths that fill a group of lanes, leave some idle or take two pieces, head counts that do not fill a
task, grouped keys, strided and unaligned rows, types, in place, positions outside the tables."""
import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _rows(torch, cuda, n, cols, dtype, layout, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    if layout == "whole":
        return torch.randn(n, cols, device=cuda, generator=gen).to(t)
    pad = 8 if layout == "aligned" else 3
    return torch.randn(n, cols + 2 * pad, device=cuda, generator=gen).to(t)[:, pad:pad + cols]


def _np(t):
    return t.float().cpu().numpy()


def _close(got, want, bound, dtype):
    tol = bound + 1e-40
    if dtype == "bf16":
        tol = tol * (1 + F.BF16) + F.BF16 * np.abs(want)
    assert got.shape == want.shape and (np.abs(_np(got).astype(np.float64) - want) <= tol).all(), float((np.abs(_np(got) - want) / tol).max())


@pytest.mark.parametrize("hd", [2, 16, 20, 32, 48, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (5, 4, 4), (131, 6, 2), (70, 9, 3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["whole", "aligned", "odd"])
def test_both_directions(cuda, hd, n, hq, hk, dtype, layout):
    import torch
    q, k = _rows(torch, cuda, n, hq * hd, dtype, layout, 1), _rows(torch, cuda, n, hk * hd, dtype, layout, 2)
    dq, dk = _rows(torch, cuda, n, hq * hd, dtype, layout, 3), _rows(torch, cuda, n, hk * hd, dtype, layout, 4)
    gains = [1 + 0.2 * torch.randn(hd, device=cuda) for _ in range(2)]
    cos, sin = F.rope_table(50, hd)
    c, s = torch.from_numpy(cos).to(cuda), torch.from_numpy(sin).to(cuda)
    pos = torch.randint(0, 50, (n,), device=cuda, dtype=torch.int32)
    p = pos.cpu().numpy()
    y = A.qk_norm_rope(q, k, *gains, pos, c, s, eps=EPS)
    for got, x, g in zip(y, (q, k), gains):
        assert got.dtype == x.dtype
        _close(got, *F.norm_rope(_np(x), _np(g), p, cos, sin, EPS), dtype)
    sums = [torch.full((hd,), 2.0, device=cuda) for _ in range(2)]
    dx = A.qk_norm_rope_backward(dq, dk, q, k, *gains, pos, c, s, *sums, eps=EPS)
    for got, acc, d, x, g in zip(dx, sums, (dq, dk), (q, k), gains):
        want, bound, dg, dg_bound = F.norm_rope_backward(_np(d), _np(x), _np(g), p, cos, sin, EPS)
        _close(got, want, bound, dtype)
        assert (np.abs(_np(acc).astype(np.float64) - 2.0 - dg) <= dg_bound + F.U * (2 + np.abs(dg))).all()       # added to what was there
    again = [torch.full((hd,), 2.0, device=cuda) for _ in range(2)]
    dx2 = A.qk_norm_rope_backward(dq, dk, q, k, *gains, pos, c, s, *again, eps=EPS)
    assert all(torch.equal(a, b) for a, b in zip(dx + tuple(sums), dx2 + tuple(again)))                          # repeatable bit for bit


@pytest.mark.parametrize("hd", [32, 128])
def test_outputs_of_another_type_and_in_place(cuda, hd):
    import torch
    n, h = 37, 3
    x = torch.randn(n, 3 * h * hd, device=cuda)                     # q, k and v of one projection
    q, k = x[:, :h * hd], x[:, h * hd:2 * h * hd]
    cos, sin = [torch.from_numpy(t).to(cuda) for t in F.rope_table(64, hd)]
    pos = torch.arange(n, device=cuda, dtype=torch.int32)
    want = A.qk_norm_rope(q, k, None, None, pos, cos, sin)
    got = A.qk_norm_rope(q, k, None, None, pos, cos, sin, k_dtype=torch.bfloat16)
    assert got[1].dtype == torch.bfloat16 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1].bfloat16())
    dy = [torch.randn(n, h * hd, device=cuda) for _ in range(2)]
    ref = A.qk_norm_rope_backward(*dy, q, k, None, None, pos, cos, sin)
    over = [d.clone() for d in dy]
    assert all(torch.equal(a, b) for a, b in zip(ref, A.qk_norm_rope_backward(*over, q, k, None, None, pos, cos, sin, q_out=over[0], k_out=over[1])))
    low = A.qk_norm_rope_backward(dy[0].bfloat16(), dy[1].bfloat16(), q, k, None, None, pos, cos, sin)           # gradients of the other type
    full = A.qk_norm_rope_backward(dy[0].bfloat16().float(), dy[1].bfloat16().float(), q, k, None, None, pos, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(low, full))
    v = x[:, 2 * h * hd:].clone()
    A.qk_norm_rope(q, k, None, None, pos, cos, sin, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(x[:, 2 * h * hd:], v)              # and nothing beside them


@pytest.mark.parametrize("hd,pad", [(32, 8), (32, 3), (40, 2), (128, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("out_dtype", ["f32", "bf16"])
def test_outputs_in_columns_of_wider_rows(cuda, hd, pad, dtype, out_dtype):
    """Outputs of both types written into column ranges, on and off 16-byte boundaries, leave what lies beside them."""
    import torch
    n, hq, hk = 29, 5, 2
    t = torch.bfloat16 if out_dtype == "bf16" else torch.float32
    q, k = _rows(torch, cuda, n, hq * hd, dtype, "whole", 1), _rows(torch, cuda, n, hk * hd, dtype, "whole", 2)
    cos, sin = [torch.from_numpy(x).to(cuda) for x in F.rope_table(16, hd)]
    pos = torch.randint(0, 16, (n,), device=cuda, dtype=torch.int32)
    wide = [torch.full((n, h * hd + 2 * pad), 7.0, device=cuda, dtype=t) for h in (hq, hk)]
    views = [w[:, pad:w.shape[1] - pad] for w in wide]
    A.qk_norm_rope(q, k, None, None, pos, cos, sin, q_out=views[0], k_out=views[1])
    for got, w, x in zip(views, wide, (q, k)):
        _close(got, *F.norm_rope(_np(x), None, pos.cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), 1e-6), out_dtype)
        assert bool((w[:, :pad] == 7).all()) and bool((w[:, -pad:] == 7).all())
    if dtype == out_dtype:
        dy = [_rows(torch, cuda, n, h * hd, "f32", "odd", 3) for h in (hq, hk)]
        A.qk_norm_rope_backward(*dy, q, k, None, None, pos, cos, sin, q_out=views[0], k_out=views[1])
        want = A.qk_norm_rope_backward(*dy, q, k, None, None, pos, cos, sin)
        for got, w, x, d in zip(views, wide, (q, k), dy):
            _close(got, *F.norm_rope_backward(_np(d), _np(x), None, pos.cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), 1e-6)[:2], out_dtype)
            assert bool((w[:, :pad] == 7).all()) and bool((w[:, -pad:] == 7).all())
        assert want[0].dtype == q.dtype
    y = A.qk_norm_rope(q, k, None, None, pos, cos, sin, k_dtype=t)
    assert y[0].dtype == q.dtype and y[1].dtype == t


def test_zero_rows_positions_outside_the_tables_and_infinities(cuda):
    import torch
    hd, n = 32, 6
    cos, sin = [torch.from_numpy(t).to(cuda) for t in F.rope_table(10, hd)]
    x = torch.randn(n, hd, device=cuda)
    x[1] = 0
    x[2, 4] = float("nan")
    x[3, 4] = float("inf")
    pos = torch.tensor([0, 3, 3, 3, -5, 99], device=cuda, dtype=torch.int32)
    y, _ = A.qk_norm_rope(x, x, None, None, pos, cos, sin)
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 4, 5]]).all()
    near, _ = A.qk_norm_rope(x, x, None, None, pos.clamp(0, 9), cos, sin)
    assert torch.equal(y[[0, 1, 4, 5]], near[[0, 1, 4, 5]])
    dx, _ = A.qk_norm_rope_backward(torch.ones_like(x), torch.ones_like(x), x, x, None, None, pos, cos, sin)
    assert torch.isfinite(dx[[0, 1, 4, 5]]).all()
    none = A.qk_norm_rope(x[:0], x[:0], None, None, pos[:0], cos, sin)
    assert none[0].shape == (0, hd)
    empty = A.qk_norm_rope_backward(x[:0], x[:0], x[:0], x[:0], None, None, pos[:0], cos, sin, *[torch.ones(hd, device=cuda) for _ in range(2)])
    assert empty[0].shape == (0, hd)


def test_gradients_against_differences(cuda):
    """Central differences of a float64 restatement at the operator's own gradients."""
    import torch
    rng = np.random.default_rng(0)
    n, h, hd = 3, 2, 16
    x, dy, g = rng.standard_normal((n, h * hd)), rng.standard_normal((n, h * hd)), 1 + 0.3 * rng.standard_normal(hd)
    cos, sin = F.rope_table(8, hd)
    pos = np.array([0, 5, 7])
    x, dy, g = [a.astype(np.float32) for a in (x, dy, g)]
    t = lambda a: torch.from_numpy(a).to(cuda)  # noqa: E731
    sums = [torch.zeros(hd, device=cuda) for _ in range(2)]
    dx, _ = A.qk_norm_rope_backward(t(dy), t(dy), t(x), t(x), t(g), t(g), t(pos.astype(np.int32)), t(cos), t(sin), *sums, eps=EPS)

    def f(x, g):
        return float((F.norm_rope(x, g, pos, cos, sin, EPS)[0] * dy).sum())

    x, g, step = x.astype(np.float64), g.astype(np.float64), 1e-5
    for a, got in ((x, _np(dx)), (g, _np(sums[0]))):
        for i in range(0, a.size, 5):
            old = a.flat[i]
            a.flat[i] = old + step
            up = f(x, g)
            a.flat[i] = old - step
            down = f(x, g)
            a.flat[i] = old
            assert abs((up - down) / (2 * step) - got.flat[i]) < 1e-5 * max(1.0, np.abs(got).max())


def test_many_rows_and_a_captured_call(cuda):
    import torch
    n, h, hd = 50_001, 4, 32
    q, k = [torch.randn(n, h * hd, device=cuda) for _ in range(2)]
    cos, sin = F.rope_table(128, hd)
    c, s = torch.from_numpy(cos).to(cuda), torch.from_numpy(sin).to(cuda)
    pos = torch.randint(0, 128, (n,), device=cuda, dtype=torch.int32)
    dq, dk = [torch.randn(n, h * hd, device=cuda) for _ in range(2)]
    sums = [torch.zeros(hd, device=cuda) for _ in range(2)]
    dx = A.qk_norm_rope_backward(dq, dk, q, k, None, None, pos, c, s, *sums)
    take = np.r_[0:3, 25_000:25_003, n - 3:n]
    for d, x, got, acc in ((dq, q, dx[0], sums[0]), (dk, k, dx[1], sums[1])):
        want, bound, _, _ = F.norm_rope_backward(_np(d)[take], _np(x)[take], None, pos.cpu().numpy()[take], cos, sin, 1e-6)
        _close(got[torch.from_numpy(take).to(cuda)], want, bound, "f32")
        _, _, dg, dgb = F.norm_rope_backward(_np(d), _np(x), None, pos.cpu().numpy(), cos, sin, 1e-6)
        assert (np.abs(_np(acc) - dg) <= dgb).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = A.qk_norm_rope(q, k, None, None, pos, c, s)
        back = A.qk_norm_rope_backward(dq, dk, q, k, None, None, pos, c, s)
    q.copy_(torch.randn_like(q))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(y, A.qk_norm_rope(q, k, None, None, pos, c, s)))
    assert all(torch.equal(a, b) for a, b in zip(back, A.qk_norm_rope_backward(dq, dk, q, k, None, None, pos, c, s)))
