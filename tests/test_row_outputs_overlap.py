"""Outputs that lie on what other blocks of the kernel still read are refused; outputs on their own input, or between rows, are taken."""
import ctypes as C

import pytest

import agpt_b200 as A

AT = 1 << 24          # addresses that are never read: every call below is refused before a launch


def _forward(q, k, qo, ko, q_ld=64, k_ld=64, qo_ld=64, ko_ld=64, q_type=0, k_type=0, n=4, some=C.c_void_p(1 << 20)):
    p = C.c_void_p
    return A.lib().agpt_b200_qk_norm_rope(p(q), q_ld, p(k), k_ld, 0, None, None, some, some, some, 8, n, 2, 2, 32, 1e-6, p(qo), qo_ld, q_type, p(ko), ko_ld, k_type, None)


def _backward(dq, dk, q, k, qo, ko, ld=64, dq_ld=64, n=4, some=C.c_void_p(1 << 20)):
    p = C.c_void_p
    return A.lib().agpt_b200_qk_norm_rope_backward(p(dq), dq_ld, p(dk), ld, 0, p(q), ld, p(k), ld, 0, None, None, some, some, some, 8, n, 2, 2, 32, 1e-6, p(qo), ld, p(ko), ld,
                                                   None, None, None, 0, None)


def test_refused():
    a, b, c, d, e, f = [AT + (i << 20) for i in range(6)]
    assert _forward(a, b, b, c) == -1 and b"overlap" in A.lib().agpt_b200_last_error()      # queries over keys
    bad = [
        _forward(a, b, b, a), _forward(a, b, c, a), _forward(a, b, c, c),
        _forward(a, b, c, c + 63 * 4), _forward(a, b, c + 3 * 256 + 252, c),                # one element of one row
        _forward(a, b, a + 4, c), _forward(a, b, a - 256, c),                               # on its own input, shifted
        _forward(a, b, a, c, qo_ld=128), _forward(a, b, a, c, q_type=1),                    # of another stride, of another type
        _forward(a, b, c, c + 256, qo_ld=96, ko_ld=96),                                     # columns that run into the next row
        _backward(a, b, c, d, b, e), _backward(a, b, c, d, d, e), _backward(a, b, c, d, e, a), _backward(a, b, c, d, e, c), _backward(a, b, c, d, e, e),
        _backward(a, a, c, d, a, e), _backward(a, a, c, d, a, a),                           # one gradient for both, written over by one of them
        _backward(a, b, c, c, c, e), _backward(a, b, c, d, a, e, dq_ld=65), _backward(a, b, c, d, a + 8, e),
    ]
    assert bad == [-1] * len(bad)
    L, p = A.lib(), C.c_void_p
    for grad, ld, out in ((a, 33, a), (a, 32, a + 4), (a, 32, a + 3 * 128 + 124), (a + 128, 32, a)):
        assert L.agpt_b200_act8_relu_backward(p(grad), ld, p(b), p(out), 4, 32, None) == -1 and b"overlap" in L.agpt_b200_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_taken(cuda, dtype):
    """Every side on its own rows, and all four sets of rows as columns of one matrix."""
    import torch
    n, hd, h = 201, 32, 3
    w = h * hd
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    wide = torch.randn(n, 4 * w + 6, device=cuda).to(t)
    col = lambda m, i, at=0: m[:, at + i * w:at + (i + 1) * w]  # noqa: E731
    cos, sin = torch.randn(16, hd, device=cuda), torch.randn(16, hd, device=cuda)
    pos = torch.randint(0, 16, (n,), device=cuda, dtype=torch.int32)
    tab = (None, None, pos, cos, sin)
    apart = torch.zeros_like(wide)                                # what is right, in rows of the same alignment: other ones may add in another order
    for at in (0, 5):
        q, k, dq, dk = [col(wide, i, at) for i in range(4)]
        out = [col(apart, i, at) for i in range(4)]
        y = [v.clone() for v in A.qk_norm_rope(q, k, *tab, q_out=out[0], k_out=out[1])]
        dx = [v.clone() for v in A.qk_norm_rope_backward(dq, dk, q, k, *tab, q_out=out[0], k_out=out[1])]
        want = [v.clone() for v in A.qk_norm_rope(q, dq, *tab, q_out=out[0], k_out=out[1])]
        m = wide.clone()
        v = [col(m, i, at) for i in range(4)]
        A.qk_norm_rope(v[0], v[2], *tab, q_out=v[1], k_out=v[3])  # into the columns between
        assert torch.equal(v[1], want[0]) and torch.equal(v[3], want[1])
        assert torch.equal(v[0], q) and torch.equal(v[2], dq) and torch.equal(m[:, :at], wide[:, :at]) and torch.equal(m[:, at + 4 * w:], wide[:, at + 4 * w:])
        m = wide.clone()
        A.qk_norm_rope(col(m, 0, at), col(m, 1, at), *tab, q_out=col(m, 0, at), k_out=col(m, 1, at))
        assert torch.equal(col(m, 0, at), y[0]) and torch.equal(col(m, 1, at), y[1])
        for on_x in (False, True):                                # over the gradients, over the inputs
            m = wide.clone()
            v = [col(m, i, at) for i in range(4)]
            A.qk_norm_rope_backward(v[2], v[3], v[0], v[1], *tab, q_out=v[0 if on_x else 2], k_out=v[1 if on_x else 3])
            assert torch.equal(v[0 if on_x else 2], dx[0]) and torch.equal(v[1 if on_x else 3], dx[1])
            assert torch.equal(v[2 if on_x else 0], dq if on_x else q) and torch.equal(v[3 if on_x else 1], dk if on_x else k)
        m = wide[:1].clone()                                      # one row has no stride
        A.qk_norm_rope(col(m, 0, at), col(m, 1, at), None, None, pos[:1], cos, sin, q_out=col(m, 0, at), k_out=col(m, 1, at))
        one = A.qk_norm_rope(q[:1], k[:1], None, None, pos[:1], cos, sin, q_out=out[0][:1], k_out=out[1][:1])
        assert torch.equal(col(m, 0, at), one[0]) and torch.equal(col(m, 1, at), one[1])
    q, k = q.contiguous(), k.contiguous()
    with pytest.raises(A.AgptError, match="overlap"):
        A.qk_norm_rope(q, k, *tab, q_out=k, k_out=q)
    if dtype == "f32":
        a, g = A.act8_pack(q), torch.randn(2 * n, w, device=cuda)
        want = A.act8_relu_backward(g[:n].clone(), a)
        assert torch.equal(A.act8_relu_backward(g[:n], a, out=g[n:]), want) and torch.equal(A.act8_relu_backward(g[:n], a, out=g[:n]), want)
