"""embedding_lookup and embedding_grad_sorted against float64, at the borders of their ways: few rows in one launch, rows ordered in one cluster and by many blocks, every number of
passes of both sorts, whole and odd pieces of a row, runs of a token inside a warp, across warps, across blocks and over all of them."""
import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F

pytestmark = pytest.mark.gpu


def _types(torch, name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _ids(kind, n, vocab, rng):
    if kind == "one":
        return np.full(n, vocab // 2)
    if kind == "distinct":
        return rng.permutation(max(n, vocab))[:n] % vocab
    if kind == "outside":
        return rng.choice(np.array([-1, vocab, vocab + 7, -2 ** 31, 2 ** 31 - 1]), n)
    zipf = np.minimum((np.exp(rng.random(n) * np.log(vocab + 1.0)) - 1).astype(np.int64), vocab - 1)
    return np.where(rng.random(n) < 0.05, -1, zipf)


@pytest.mark.parametrize("n,vocab,d", [(1, 1, 4), (7, 5, 1), (33, 1400, 384), (300, 65, 130), (5, 70_000, 16), (1000, 3, 1024)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_lookup_is_the_rounded_product(cuda, n, vocab, d, dtype, wide):
    import torch
    rng = np.random.default_rng(n + d)
    table = torch.randn(vocab, d, device=cuda).to(_types(torch, dtype))
    ids = torch.from_numpy(_ids("zipf", n, vocab, rng)).to(cuda).to(torch.int64 if wide else torch.int32)
    live = (ids >= 0) & (ids < vocab)
    for scale in (1.0, 0.3):
        want = torch.where(live[:, None], table[ids.long().clamp(0, vocab - 1)].float() * scale, 0.0).to(table.dtype)
        assert torch.equal(A.embedding_lookup(table, ids, scale), want)
    # a column range of a wider table whose rows start off every boundary, and an output given by the caller
    wider = torch.randn(vocab, d + 3, device=cuda).to(_types(torch, dtype))
    out = torch.full((n, d), 7.0, device=cuda, dtype=table.dtype)
    assert A.embedding_lookup(wider[:, 1:d + 1], ids, 2.0, out=out) is out
    assert torch.equal(out, torch.where(live[:, None], wider[:, 1:d + 1][ids.long().clamp(0, vocab - 1)].float() * 2.0, 0.0).to(table.dtype))


def _check_grad(torch, grad, ids, vocab, scale, out=None, **kw):
    want, bound = F.table_grad(grad.float().cpu().numpy(), ids.cpu().numpy(), vocab, scale)
    old = out.float().cpu().numpy().astype(np.float64) if kw.get("accumulate") else 0.0
    got = A.embedding_grad_sorted(grad, ids, vocab, scale, out=out, **kw)
    g = got.float().cpu().numpy().astype(np.float64)
    tol = bound + 2 * F.U * (np.abs(want) + np.abs(old))
    if got.dtype == torch.bfloat16:
        tol = tol * (1 + F.BF16) + F.BF16 * np.abs(want + old)
    assert (np.abs(g - (want + old)) <= tol).all()
    return got


@pytest.mark.parametrize("kind", ["zipf", "one", "distinct", "outside"])
@pytest.mark.parametrize("n,vocab,d", [
    (0, 5, 8), (1, 1, 4), (2, 3, 1), (300, 1400, 384), (512, 40, 65), (513, 40, 65),          # both sides of the few-rows border
    (1025, 1, 33), (1024, 255, 128), (4097, 256, 36), (5000, 70_000, 20), (3001, 20_000_000, 4),       # one cluster: passes of eight bits, one to four
    (20_011, 500, 132), (32_768, 1000, 12),
    (32_769, 2047, 12), (33_001, 2048, 20), (40_000, 70_000, 9), (33_333, 5_000_000, 4),     # many blocks: passes of up to eleven bits, one to three
    (70_000, 3, 8),                                                                          # runs of a token over many blocks of the sums
])
def test_gradient(cuda, kind, n, vocab, d):
    import torch
    n = min(n, 5000) if kind == "outside" else n
    rng = np.random.default_rng(n * 7 + d)
    grad = torch.from_numpy(rng.standard_normal((n, d)).astype(np.float32)).to(cuda)
    ids = torch.from_numpy(_ids(kind, n, vocab, rng)).to(cuda)
    a = _check_grad(torch, grad, ids.to(torch.int32), vocab, 0.7)
    assert torch.equal(a, A.embedding_grad_sorted(grad, ids.to(torch.int64), vocab, 0.7))          # int64 ids; repeatable bit for bit


@pytest.mark.parametrize("n,d", [(200, 72), (3000, 72), (3000, 71), (6000, 264)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("out_dtype", ["f32", "bf16"])
def test_gradient_types_strides_and_accumulation(cuda, n, d, dtype, out_dtype):
    import torch
    rng = np.random.default_rng(d + n)
    vocab = 801
    ids = torch.from_numpy(_ids("zipf", n, vocab, rng)).to(cuda).to(torch.int32)
    wider = torch.randn(n, d + 9, device=cuda).to(_types(torch, dtype))
    for grad in (wider[:, 8:d + 8], wider[:, 1:d + 1], wider[:, :d].contiguous()):
        out = torch.full((vocab, d), float("nan"), device=cuda, dtype=_types(torch, out_dtype))      # every row is written
        _check_grad(torch, grad, ids, vocab, 1.5, out=out)
        out = torch.randn(vocab, d, device=cuda).to(_types(torch, out_dtype))
        kept = out.clone()
        _check_grad(torch, grad, ids, vocab, 1.5, out=out, accumulate=True)
        absent = torch.ones(vocab, dtype=torch.bool, device=cuda)
        absent[ids[(ids >= 0)].long()] = False
        assert torch.equal(out[absent], kept[absent])                                                # rows of absent tokens are left as they are


def test_infinities_and_nan_stay_in_their_token(cuda):
    import torch
    n, vocab, d = 4000, 700, 64
    ids = torch.arange(n, device=cuda, dtype=torch.int32) % vocab
    grad = torch.ones(n, d, device=cuda)
    grad[5, 3], grad[9, 7] = float("inf"), float("nan")
    got = A.embedding_grad_sorted(grad, ids, vocab)
    assert torch.isinf(got[5, 3]) and torch.isnan(got[9, 7]) and int((~torch.isfinite(got)).sum()) == 2
    ids[5] = ids[9] = -1                                       # padded rows are not read into any sum
    assert torch.isfinite(A.embedding_grad_sorted(grad, ids, vocab)).all()
    few = A.embedding_grad_sorted(grad[:300], ids[:300], vocab)
    assert torch.isfinite(few).all()


def test_gradient_is_the_lookups_derivative(cuda):
    """<d out, lookup(E + h D) - lookup(E)> / h = <grad, D>: the lookup is linear."""
    import torch
    torch.manual_seed(3)
    n, vocab, d = 2000, 1200, 96
    emb, dirn, dy = [torch.randn(s, d, device=cuda) for s in (vocab, vocab, n)]
    ids = torch.randint(-1, vocab, (n,), device=cuda, dtype=torch.int32)
    diff = (A.embedding_lookup(emb + dirn, ids, 3.0).double() - A.embedding_lookup(emb, ids, 3.0).double())
    left, right = (diff * dy.double()).sum(), (A.embedding_grad_sorted(dy, ids, vocab, 3.0).double() * dirn.double()).sum()
    # every term is off by a few roundings of its own size
    assert abs(left - right) <= 16 * F.U * 3.0 * float(((emb.abs() + dirn.abs()).double()[ids.clamp(min=0).long()] * dy.abs().double()).sum())


def test_streams_and_graphs(cuda):
    """A captured call is replayed on new contents, beside another capture and an eager call on another stream."""
    import torch
    n, vocab, d = 3000, 900, 64
    ids = [torch.randint(0, vocab, (n,), device=cuda, dtype=torch.int32) for _ in range(2)]
    grads = [torch.randn(n, d, device=cuda) for _ in range(2)]
    A.embedding_grad_sorted(grads[0], ids[0], vocab)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(A.embedding_grad_sorted(grads[k], ids[k], vocab))
        graphs.append(g)
    for k in range(2):
        grads[k].copy_(torch.randn(n, d, device=cuda))
        ids[k].copy_(torch.randint(0, vocab, (n,), device=cuda, dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(outs[k], A.embedding_grad_sorted(grads[k], ids[k], vocab))
