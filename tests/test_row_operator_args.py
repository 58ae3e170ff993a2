"""What the row operators refuse, and the restatements their GPU tests are held to.  Nothing here needs a GPU: the checks come before any launch."""
import ctypes as C

import numpy as np
import pytest

import agpt_b200 as A
from tests import row_forms as F


def test_host_tensors_are_refused():
    import torch
    x, ids = torch.zeros(4, 32), torch.zeros(4, dtype=torch.int32)
    cos, sin = [torch.from_numpy(t) for t in F.rope_table(8, 32)]
    for call in (lambda: A.embedding_lookup(x, ids), lambda: A.embedding_grad_sorted(x, ids, 9), lambda: A.qk_norm_rope(x, x, None, None, ids, cos, sin),
                 lambda: A.qk_norm_rope_backward(x, x, x, x, None, None, ids, cos, sin), lambda: A.act8_pack(x),
                 lambda: A.Act8(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 16, dtype=torch.uint8), 32)):
        with pytest.raises(A.AgptError):
            call()


def test_the_library_refuses_before_it_launches():
    L, some = A.lib(), C.c_void_p(256)          # an address that is never read
    bad = [
        L.agpt_b200_embedding_lookup(None, 8, 0, some, 0, some, 4, 8, 10, 1.0, None),
        L.agpt_b200_embedding_lookup(some, 4, 0, some, 0, some, 4, 8, 10, 1.0, None),            # rows overlap
        L.agpt_b200_embedding_lookup(some, 8, 2, some, 0, some, 4, 8, 10, 1.0, None),            # no such type
        L.agpt_b200_embedding_grad_sorted(some, 8, 0, some, 0, None, 0, 4, 8, 10, 1.0, 0, some, 1 << 30, None),
        L.agpt_b200_embedding_grad_sorted(some, 8, 0, some, 0, some, 5, 4, 8, 10, 1.0, 0, some, 1 << 30, None),
        L.agpt_b200_embedding_grad_sorted(some, 8, 0, some, 0, some, 0, 100_000, 8, 10, 1.0, 0, some, 16, None),       # workspace too small
        L.agpt_b200_embedding_grad_sorted(some, 8, 0, some, 0, some, 0, 100_000, 8, 10, 1.0, 0, None, 1 << 30, None),
        L.agpt_b200_qk_norm_rope(some, 64, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, 33, 1e-6, some, 66, 0, some, 66, 0, None),       # odd head_dim
        L.agpt_b200_qk_norm_rope(some, 64, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, 32, 0.0, some, 64, 0, some, 64, 0, None),        # eps
        L.agpt_b200_qk_norm_rope(some, 63, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, 32, 1e-6, some, 64, 0, some, 64, 0, None),       # stride
        L.agpt_b200_qk_norm_rope(some, 64, some, 64, 0, None, None, some, some, some, 0, 4, 2, 2, 32, 1e-6, some, 64, 0, some, 64, 0, None),       # empty tables
        L.agpt_b200_qk_norm_rope(some, 64, some, 64, 0, None, None, None, some, some, 8, 4, 2, 2, 32, 1e-6, some, 64, 0, some, 64, 0, None),
        L.agpt_b200_qk_norm_rope_backward(some, 64, some, 64, 0, some, 64, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, 32, 1e-6, some, 64, some, 64, some,
                                          some, None, 0, None),                                                                                  # no workspace
        L.agpt_b200_qk_norm_rope_backward(some, 64, some, 64, 7, some, 64, some, 64, 0, None, None, some, some, some, 8, 4, 2, 2, 32, 1e-6, some, 64, some, 64, None,
                                          None, None, 0, None),
        L.agpt_b200_act8_pack(some, 31, 0, some, some, 4, 32, None),
        L.agpt_b200_act8_pack(some, 32, 0, C.c_void_p(264), some, 4, 32, None),
        L.agpt_b200_act8_pack(some, 32, 3, some, some, 4, 32, None),
        L.agpt_b200_act8_unpack(some, None, some, 4, 32, None),
        L.agpt_b200_act8_relu_backward(some, 32, None, some, 4, 32, None),
        L.agpt_b200_act8_weight_grad(some, some, some, 7, 4, 32, 8, some, None, some, 1 << 30, None),
        L.agpt_b200_act8_weight_grad(some, some, some, 8, 100_000, 32, 8, some, None, some, 4, None),                     # workspace too small
        L.agpt_b200_act8_weight_grad(some, some, some, 8, 4, 0, 8, some, None, some, 1 << 30, None),
    ]
    assert bad == [-1] * len(bad)
    assert L.agpt_b200_qk_norm_rope(some, 1024, some, 1024, 0, None, None, some, some, some, 8, 4, 2, 2, 512, 1e-6, some, 1024, 0, some, 1024, 0, None) == -4
    assert L.agpt_b200_embedding_lookup(some, 8, 0, some, 0, some, 1 << 40, 8, 10, 1.0, None) == -4
    assert L.agpt_b200_embedding_grad_sorted_workspace_bytes(-1, 8, 10) == -1 and L.agpt_b200_act8_weight_grad_workspace_bytes(5, -1, 3) == -1
    assert L.agpt_b200_embedding_grad_sorted_workspace_bytes(1 << 20, 128, 1000) > 8 << 20


def test_no_rows_is_no_work():
    L, none = A.lib(), None
    assert L.agpt_b200_embedding_lookup(none, 8, 0, none, 0, none, 0, 8, 10, 1.0, None) == 0
    assert L.agpt_b200_qk_norm_rope(none, 64, none, 64, 0, none, none, none, none, none, 8, 0, 2, 2, 32, 1e-6, none, 64, 0, none, 64, 0, None) == 0
    assert L.agpt_b200_act8_pack(none, 32, 0, none, none, 0, 32, None) == 0 and L.agpt_b200_act8_unpack(none, none, none, 0, 32, None) == 0


def test_the_restated_checkpoint():
    """Known answers: a value on every code, ties to the even code, the scale's border, the smallest code."""
    x = np.zeros((1, 32), np.float32)
    x[0, :6] = [448, 17, 19, 2.0 ** -11, -2.0 ** -40, 1.0625]         # scale 1: 17 and 19 lie halfway between codes
    codes, scales, values = F.pack(x)
    assert scales[0, 0] == 127 and values[0, :6].tolist() == [448, 16, 20, 2.0 ** -9, -2.0 ** -9, 1.0] and not values[0, 6:].any() and codes[0, 4] == 129
    x[0, 0] = 448.5
    assert F.pack(x)[1][0, 0] == 128 and F.pack(x)[2][0, 0] == 448
    assert F.pack(np.zeros((1, 1), np.float32))[1][0, 0] == 17 and np.isnan(F.pack(np.full((1, 1), np.inf, np.float32))[2]).all()


def test_restated_gradients_against_differences():
    rng = np.random.default_rng(1)
    x, dy, g = rng.standard_normal((2, 12)), rng.standard_normal((2, 12)), rng.standard_normal(6)
    cos, sin = F.rope_table(9, 6)
    pos = np.array([2, 8])
    dx, _, dg, _ = F.norm_rope_backward(dy, x, g, pos, cos, sin, 1e-3)
    f = lambda x, g: float((F.norm_rope(x, g, pos, cos, sin, 1e-3)[0] * dy).sum())  # noqa: E731
    for a, got in ((x, dx), (g, dg)):
        for i in range(a.size):
            old = a.flat[i]
            a.flat[i] = old + 1e-6
            up = f(x, g)
            a.flat[i] = old - 1e-6
            down = f(x, g)
            a.flat[i] = old
            assert abs((up - down) / 2e-6 - got.flat[i]) < 1e-7 * max(1.0, np.abs(got).max())
