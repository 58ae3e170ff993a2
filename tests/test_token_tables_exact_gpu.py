"""The table's gradient on integers: every partial sum is exact in float32, so the sums of a token are equal to the integer ones however many rows, warps, blocks and
joins they run over; a lost or doubled row or piece shows."""
import numpy as np
import pytest

import agpt_b200 as A
from tests.test_token_tables_gpu import _ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["one", "zipf", "distinct", "halves"])
@pytest.mark.parametrize("n,vocab,d", [
    (512, 40, 65), (513, 40, 65), (2049, 2, 128), (5000, 7, 20), (9001, 3, 260), (20_011, 500, 132), (32_768, 1000, 12),
    (32_769, 2047, 12), (33_001, 2048, 65), (70_000, 3, 8), (150_001, 70_000, 36), (400_003, 5, 128),
])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_integer_sums(cuda, kind, n, vocab, d, dtype):
    import torch
    rng = np.random.default_rng(n + d)
    if kind == "halves":          # two long runs and what lies between, borders off every run of places
        ids = np.where(np.arange(n) < n // 2 + 3, 0, vocab - 1)
        ids[n // 3::97] = vocab // 2
        rng.shuffle(ids)
    else:
        ids = _ids(kind, n, vocab, rng)
    ids = torch.from_numpy(ids).to(cuda)
    gen = torch.Generator(device=cuda).manual_seed(n)
    whole = torch.randint(-8, 9, (n, d), device=cuda, generator=gen)
    grad = whole.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    live = (ids >= 0) & (ids < vocab)
    want = torch.zeros(vocab, d, dtype=torch.float64, device=cuda).index_add_(0, ids[live].long(), whole[live].double())
    got = A.embedding_grad_sorted(grad, ids.to(torch.int32), vocab, 2.0)
    assert torch.equal(got.double(), 2 * want) and bool(want.any())
    old = torch.randint(-99, 100, (vocab, d), device=cuda, generator=gen).float()
    more = old.clone()
    assert A.embedding_grad_sorted(grad, ids.to(torch.int64), vocab, 1.0, out=more, accumulate=True) is more
    assert torch.equal(more.double(), want + old.double())
    wider = torch.zeros(n, d + 5, dtype=grad.dtype, device=cuda)          # rows off 16-byte boundaries
    wider[:, 3:d + 3] = grad
    rounded = torch.full((vocab, d), 7.0, dtype=torch.bfloat16, device=cuda)
    A.embedding_grad_sorted(wider[:, 3:d + 3], ids.to(torch.int32), vocab, 1.0, out=rounded)
    assert torch.equal(rounded, want.float().bfloat16())                  # one rounding of the exact sum
