"""Gain gradients over so many rows that a thread's sums leave their registers several times, on numbers for which everything is exact: x of +-1 (a root mean square
of 1), quarter turns for the rotation, integer gradients.  A lost, doubled or wrongly placed row shows."""
import numpy as np
import pytest

import agpt_b200 as A

pytestmark = pytest.mark.gpu


def _case(torch, cuda, n, hq, hk, hd, dtype, pad):
    gen = torch.Generator(device=cuda).manual_seed(n + hd)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32

    def rows(cols, lo, hi, odd=False):
        v = torch.randint(lo, hi + 1, (n, cols + 2 * pad), device=cuda, generator=gen)
        return (2 * v + 1 if odd else v).to(t)[:, pad:pad + cols]

    q, k = rows(hq * hd, -1, 0, True), rows(hk * hd, -1, 0, True)          # +-1
    dq, dk = rows(hq * hd, -4, 4), rows(hk * hd, -4, 4)
    # position p turns by p quarters
    cos = torch.tensor([1.0, 0.0, -1.0, 0.0], device=cuda)[:, None].expand(4, hd).contiguous()
    sin = torch.tensor([0.0, 1.0, 0.0, -1.0], device=cuda)[:, None].expand(4, hd).contiguous()
    pos = torch.randint(0, 4, (n,), device=cuda, generator=gen, dtype=torch.int32)
    return q, k, dq, dk, cos, sin, pos


def _turn(torch, v, cos, sin):
    a, b = v[..., 0::2], v[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _want(torch, x, dy, cos, sin, pos, hd):
    """(y, dx, dgain) in float64: exact"""
    n = x.shape[0]
    c, s = cos.double()[pos.long()][:, None, 0::2], sin.double()[pos.long()][:, None, 0::2]
    v, w = x.double().reshape(n, -1, hd), _turn(torch, dy.double().reshape(n, -1, hd), c, -s)
    return _turn(torch, v, c, s).reshape(n, -1), (w - v * (w * v).mean(2, keepdim=True)).reshape(n, -1), (w * v).sum((0, 1))


# rounds of a thread on 148 SMs: 85 of 4736 rows, 86 of 352, 127 of 2368 (rows off 16-byte boundaries), 96 of 1576, 113 of 1776
@pytest.mark.parametrize("n,hq,hk,hd,dtype,pad", [(400_003, 4, 4, 32, "f32", 0), (30_011, 32, 8, 128, "bf16", 0), (300_007, 4, 4, 32, "f32", 3), (150_001, 3, 1, 256, "f32", 0),
                                                  (200_003, 2, 1, 64, "bf16", 1)])
def test_exact_sums(cuda, n, hq, hk, hd, dtype, pad):
    import torch
    q, k, dq, dk, cos, sin, pos = _case(torch, cuda, n, hq, hk, hd, dtype, pad)
    y = A.qk_norm_rope(q, k, None, None, pos, cos, sin, eps=1e-12)
    sums = [torch.full((hd,), 3.0, device=cuda) for _ in range(2)]
    dx = A.qk_norm_rope_backward(dq, dk, q, k, None, None, pos, cos, sin, *sums, eps=1e-12)
    for x, dy, got_y, got_dx, got in ((q, dq, y[0], dx[0], sums[0]), (k, dk, y[1], dx[1], sums[1])):
        want_y, want_dx, want = _want(torch, x, dy, cos, sin, pos, hd)
        assert 4 * n * hq < 1 << 24 and float(want.abs().max()) > 100
        assert torch.equal(got_y.double(), want_y)                         # so the reciprocal root of 1 is 1
        assert torch.equal(got_dx, want_dx.float().to(q.dtype)) and torch.equal(got.double(), want + 3)
    alone = torch.zeros(hd, device=cuda)                                   # one of the two
    A.qk_norm_rope_backward(dq, dk, q, k, None, None, pos, cos, sin, None, alone, eps=1e-12)
    assert torch.equal(alone + 3, sums[1])
