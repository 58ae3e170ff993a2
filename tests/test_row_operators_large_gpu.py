"""The row operators past 2^31 elements: the last rows of a large call are those of a call on these rows alone."""
import pytest

import agpt_b200 as A

pytestmark = pytest.mark.gpu
ROWS, COLS, TAIL = (1 << 21) + 64, 1024, 64          # 2^31 + 65536 elements


@pytest.fixture(autouse=True)
def _memory_back():
    yield
    import torch
    torch.cuda.empty_cache()


def _zeros_but_tail(torch, rows, cols, dtype, cuda, seed):
    x = torch.zeros(rows, cols, device=cuda, dtype=dtype)
    x[-TAIL:] = torch.randn(TAIL, cols, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(dtype)
    return x


def test_token_tables(cuda):
    import torch
    vocab = 1500
    table = torch.randn(vocab, COLS, device=cuda).bfloat16()
    ids = torch.randint(0, vocab, (ROWS,), device=cuda, dtype=torch.int32)
    rows = A.embedding_lookup(table, ids, 2.0)
    assert torch.equal(rows[-TAIL:], A.embedding_lookup(table, ids[-TAIL:], 2.0)) and torch.equal(rows[:TAIL], A.embedding_lookup(table, ids[:TAIL], 2.0))
    del rows
    grad = _zeros_but_tail(torch, ROWS, COLS, torch.bfloat16, cuda, 1)
    # zeros change no sum, and the last rows of a token come in the same order
    assert torch.equal(A.embedding_grad_sorted(grad, ids, vocab), A.embedding_grad_sorted(grad[-TAIL:], ids[-TAIL:], vocab))


def test_query_and_key_norms(cuda):
    import torch
    hd, hk = 128, 2
    q, k = torch.randn(ROWS, COLS, device=cuda, dtype=torch.bfloat16), torch.randn(ROWS, hk * hd, device=cuda, dtype=torch.bfloat16)
    cos, sin = torch.randn(64, hd, device=cuda), torch.randn(64, hd, device=cuda)
    pos = torch.randint(0, 64, (ROWS,), device=cuda, dtype=torch.int32)
    y = A.qk_norm_rope(q, k, None, None, pos, cos, sin)
    want = A.qk_norm_rope(q[-TAIL:], k[-TAIL:], None, None, pos[-TAIL:], cos, sin)
    assert all(torch.equal(a[-TAIL:], b) for a, b in zip(y, want))
    dx = A.qk_norm_rope_backward(*y, q, k, None, None, pos, cos, sin)
    want = A.qk_norm_rope_backward(y[0][-TAIL:], y[1][-TAIL:], q[-TAIL:], k[-TAIL:], None, None, pos[-TAIL:], cos, sin)
    assert all(torch.equal(a[-TAIL:], b) for a, b in zip(dx, want))


def test_8_bit_checkpoints(cuda):
    import torch
    x = torch.randn(ROWS, COLS, device=cuda, dtype=torch.bfloat16)
    a, tail = A.act8_pack(x), A.act8_pack(x[-TAIL:])
    assert torch.equal(a.codes[-TAIL:], tail.codes) and torch.equal(a.scales[:, ROWS - TAIL:ROWS], tail.scales[:, :TAIL])
    del x
    assert torch.equal(A.act8_unpack(a)[-TAIL:], A.act8_unpack(tail))
    grad = torch.randn(ROWS, COLS, device=cuda)
    assert torch.equal(A.act8_relu_backward(grad, a, out=grad)[-TAIL:], A.act8_relu_backward(grad[-TAIL:], tail))
    del grad
    # the last 64 rows are a row block of their own in both calls
    grad = _zeros_but_tail(torch, ROWS, 16, torch.float32, cuda, 2)
    assert all(torch.equal(u, v) for u, v in zip(A.act8_weight_grad(a, grad), A.act8_weight_grad(tail, grad[-TAIL:])))
    wide = _zeros_but_tail(torch, ROWS, COLS + 1, torch.float32, cuda, 3)[:, 1:]      # off 16-byte boundaries
    few = A.Act8(a.codes[:, :32].contiguous(), a.scales[:1].contiguous(), 32)
    few_tail = A.Act8(tail.codes[:, :32].contiguous(), tail.scales[:1].contiguous(), 32)
    assert all(torch.equal(u, v) for u, v in zip(A.act8_weight_grad(few, wide), A.act8_weight_grad(few_tail, wide[-TAIL:])))
