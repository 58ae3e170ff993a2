"""Plain float64 forms of the row operators (token tables, query and key norms with the rotation, 8-bit checkpoints), with bounds for what float32 arithmetic
in any order of summation may be off: u = 2^-24 is the largest relative error of one rounding to nearest."""
import math

import numpy as np

U = 2.0 ** -24
BF16 = 2.0 ** -8          # half a step of bfloat16, relative


# ---- token tables ---------------------------------------------------------------------------------------------------------
def table_grad(grad, ids, vocab, scale):
    """(gradient, bound): m values of a token are added with at most m - 1 roundings of partial sums that the sum of magnitudes bounds, then scaled."""
    g = grad.astype(np.float64)
    out, mag, cnt = np.zeros((vocab, g.shape[1])), np.zeros((vocab, g.shape[1])), np.zeros(vocab)
    for i, t in enumerate(ids):
        if 0 <= t < vocab:
            out[t] += g[i]
            mag[t] += np.abs(g[i])
            cnt[t] += 1
    return out * scale, (cnt[:, None] + 1) * U * mag * abs(scale)


# ---- norms and rotation ---------------------------------------------------------------------------------------------------
def rope_table(positions, hd):
    a = np.arange(positions)[:, None] / 10000.0 ** (2 * np.arange(hd // 2) / hd)
    return [np.repeat(f(a).astype(np.float32), 2, axis=1) for f in (np.cos, np.sin)]


def norm_rope(x, gain, pos, cos, sin, eps):
    """(y, bound).  r has (hd + 1) roundings of the sum of squares, halved by the root, and four more; then x r g, two products, one sum."""
    n, hd = x.shape[0], cos.shape[1]
    v = x.astype(np.float64).reshape(n, -1, hd)
    g = np.ones(hd) if gain is None else gain.astype(np.float64)
    pos = np.clip(pos, 0, cos.shape[0] - 1)
    c, s = [t[pos].astype(np.float64)[:, None, 0::2] for t in (cos, sin)]
    a = v / np.sqrt((v * v).mean(2, keepdims=True) + eps) * g
    e, o = a[..., 0::2], a[..., 1::2]
    y, size = np.empty_like(a), np.empty_like(a)
    y[..., 0::2], y[..., 1::2] = e * c - o * s, e * s + o * c
    size[..., 0::2], size[..., 1::2] = np.abs(e * c) + np.abs(o * s), np.abs(e * s) + np.abs(o * c)
    return y.reshape(n, -1), ((hd / 2 + 10) * U * size).reshape(n, -1)


def norm_rope_backward(dy, x, gain, pos, cos, sin, eps):
    """(dx, bound, dgain, bound)."""
    n, hd = x.shape[0], cos.shape[1]
    v = x.astype(np.float64).reshape(n, -1, hd)
    d = dy.astype(np.float64).reshape(v.shape)
    g = np.ones(hd) if gain is None else gain.astype(np.float64)
    pos = np.clip(pos, 0, cos.shape[0] - 1)
    c, s = [t[pos].astype(np.float64)[:, None, 0::2] for t in (cos, sin)]
    r = 1 / np.sqrt((v * v).mean(2, keepdims=True) + eps)
    w, size = np.empty_like(v), np.empty_like(v)
    w[..., 0::2], w[..., 1::2] = d[..., 0::2] * c + d[..., 1::2] * s, d[..., 1::2] * c - d[..., 0::2] * s
    size[..., 0::2] = np.abs(d[..., 0::2] * c) + np.abs(d[..., 1::2] * s)
    size[..., 1::2] = np.abs(d[..., 1::2] * c) + np.abs(d[..., 0::2] * s)
    k, kn = w * g, size * np.abs(g)
    dx = r * (k - v * r * r * (k * v).mean(2, keepdims=True))
    dx_size = r * (kn + np.abs(v) * r * r * (kn * np.abs(v)).mean(2, keepdims=True))
    terms = n * v.shape[1]
    # each term of the mean: rotation (3), gain (1), product (1), at most hd additions; r twice or three times with (hd / 2 + 4) each; the last operations 4
    return (dx.reshape(n, -1), ((3 * hd + 30) * U * dx_size).reshape(n, -1),
            (w * v * r).sum((0, 1)), (terms + hd / 2 + 12) * U * (size * np.abs(v * r)).sum((0, 1)))


# ---- 8-bit checkpoints ------------------------------------------------------------------------------------------------------
def _e4m3_values():
    """The values of the codes 0 .. 126."""
    c = np.arange(127)
    e, f = c >> 3, c & 7
    return np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))


E4M3 = _e4m3_values()


def pack(x):
    """(codes, scales [blocks, n], values float64): nearest code by distance, a tie to the even code."""
    n, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((n, blocks * 32))
    v[:, :cols] = x.astype(np.float64)
    v = v.reshape(n, blocks, 32)
    codes, scales, values = np.zeros(v.shape, np.uint8), np.zeros((blocks, n), np.uint8), np.zeros(v.shape)
    for i in range(n):
        for b in range(blocks):
            w = v[i, b]
            if not np.isfinite(w).all():
                codes[i, b], scales[b, i], values[i, b] = 0x7f, 255, np.nan
                continue
            e = -110
            while np.abs(w).max() > 448.0 * 2.0 ** e:
                e += 1
            m = np.abs(w) / 2.0 ** e
            hi = np.clip(np.searchsorted(E4M3, m), 1, 126)
            up, down = E4M3[hi] - m, m - E4M3[hi - 1]
            code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
            code = np.where((code == 0) & (m > 0), 1, code)
            if e == 120:                      # 256 * 2^120 is beyond float32
                code = np.minimum(code, 0x77)
            codes[i, b] = code + 128 * np.signbit(w)
            scales[b, i] = e + 127
            values[i, b] = np.sign(w) * E4M3[code] * 2.0 ** e
    return codes.reshape(n, -1), scales, values.reshape(n, -1)[:, :cols]


def weight_grad(values, grad):
    """(X^T G, bound, column sums, bound): n products, the additions of a tensor core may cut instead of rounding (2 u each), and the slices' sums."""
    x, g = values.astype(np.float64), grad.astype(np.float64)
    n = x.shape[0]
    return x.T @ g, (2 * n + 200) * U * (np.abs(x).T @ np.abs(g)), g.sum(0), (n + 200) * U * np.abs(g).sum(0)
