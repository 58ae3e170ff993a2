"""Queries and keys that share one gain, and its one gradient; accumulators that overlap in another way are refused."""
import ctypes as C

import pytest

import agpt_b200 as A


def test_overlapping_accumulators_are_refused():
    """Before any launch, on addresses that are never read."""
    L, some = A.lib(), C.c_void_p(1 << 20)

    def call(dq_gain, dk_gain, hd=32, workspace=None):
        return L.agpt_b200_qk_norm_rope_backward(some, 64, some, 64, 0, some, 64, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, hd, 1e-6, some, 64, some, 64,
                                                 C.c_void_p(dq_gain), C.c_void_p(dk_gain), workspace, 0, None)
    at = 1 << 21
    for other in (at + 4, at + 31 * 4, at - 4, at - 31 * 4):
        assert call(at, other) == -1 and b"overlap" in L.agpt_b200_last_error()
    for other in (at, at + 32 * 4, at - 32 * 4):                  # one tensor, or neighbours: what is missing is the workspace
        assert call(at, other) == -1 and b"workspace" in L.agpt_b200_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("n,hq,hk,hd", [(1, 1, 1, 2), (3000, 4, 4, 32), (20_011, 6, 2, 128), (701, 3, 1, 250)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_gradient_takes_both_sums(cuda, n, hq, hk, hd, dtype):
    import torch
    from tests import row_forms as F
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    gen = torch.Generator(device=cuda).manual_seed(n)
    q, k, dq, dk = [torch.randn(n, h * hd, device=cuda, generator=gen).to(t) for h in (hq, hk, hq, hk)]
    gain = 1 + 0.2 * torch.randn(hd, device=cuda, generator=gen)
    cos, sin = [torch.from_numpy(x).to(cuda) for x in F.rope_table(64, hd)]
    pos = torch.randint(0, 64, (n,), device=cuda, generator=gen, dtype=torch.int32)
    apart = [torch.zeros(hd, device=cuda) for _ in range(2)]
    dx = A.qk_norm_rope_backward(dq, dk, q, k, gain, gain, pos, cos, sin, *apart)
    old = torch.randn(hd, device=cuda, generator=gen)
    for _ in range(3):
        both = old.clone()
        got = A.qk_norm_rope_backward(dq, dk, q, k, gain, gain, pos, cos, sin, both, both)
        assert torch.equal(both, old + apart[0] + apart[1])       # in this order, bit for bit
        assert all(torch.equal(a, b) for a, b in zip(got, dx))
    assert bool((apart[1] != 0).all())
