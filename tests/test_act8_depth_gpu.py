"""The weight gradient over slices of ten row blocks and more, where every stage and accumulator of its pipeline is used again, on numbers whose sums are exact in
float32: whatever order they are added in, a lost, doubled or mispaired row shows."""
import numpy as np
import pytest

import agpt_b200 as A

pytestmark = pytest.mark.gpu


# blocks of 64 rows a slice on 148 SMs: 34 to 35; 10 to 11 twice (one accumulator at a time); 52 to 53 twice (groups of 160 and of 97 or 120 kept columns); 22 to 23 twice
@pytest.mark.parametrize("n,m,cols", [(20_003, 512, 1024), (100_003, 128, 128), (100_003, 100, 65), (20_003, 257, 1500), (20_003, 280, 1500), (12_800, 64, 1920), (12_864, 200, 1920)])
@pytest.mark.parametrize("pad", [0, 1])
def test_exact_sums(cuda, n, m, cols, pad):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(n + m)
    x = torch.randint(-2, 3, (n, m), device=cuda, generator=gen)
    g = torch.randint(-4, 5, (n, cols + 2 * pad), device=cuda, generator=gen)
    # rows of 18 bits, for the second and third part of a split, far apart and at the end
    rows = torch.cat([torch.arange(1, n, n // 19, device=cuda), torch.tensor([n - 1], device=cuda)])
    g[rows] = torch.randint(-(1 << 18) + 1, 1 << 18, (rows.numel(), cols + 2 * pad), device=cuda, generator=gen)
    grad = g.float()[:, pad:pad + cols]
    # any partial sum stays below 2^24
    assert 2 * (4 * n + rows.numel() * (1 << 18)) < 1 << 24
    a = A.act8_pack(x.float())
    assert torch.equal(A.act8_unpack(a), x.float())
    dw, db = A.act8_weight_grad(a, grad)
    want = x.double().t() @ grad.double()                         # exact in float64
    assert torch.equal(dw.double(), want) and torch.equal(db.double(), grad.double().sum(0))
    assert float(want.abs().amin(1).max()) > 0 and float(want.abs().max()) > 1 << 17
