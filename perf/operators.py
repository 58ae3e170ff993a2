"""What a training step runs in front of the attention and keeps for its backward, one operator a case:

  embedding   embedding_lookup, and with `gradient` embedding_grad_sorted: rows of the token table times a scale, and the gradient of the
              table summed over equal tokens
  qk          qk_norm_rope, and with `gradient` qk_norm_rope_backward: RMS norm of queries and keys per head with the rotation
  round_trip  act8_pack and act8_unpack: an activation to its 8-bit checkpoint and back
  backward    act8_relu_backward (with `relu`) and act8_weight_grad: the backward of a projection whose input, and output where a ReLU
              follows, were kept in 8 bits

A checkpoint is codes uint8 [rows, columns rounded up to 32] (e4m3) and scales uint8 [blocks of 32 columns, rows rounded up to 16]: the value of a code is
the e4m3 number times 2^(scale - 127).  The plain forms below are elementary torch operations in 32 bits.
"""
import math

import torch

own = False
EPS = 1e-6


def listed():
    return [
        # one sampled training unit of a model whose vocabulary is as large as the loss takes
        dict(name="embedding-sampled-unit", kind="embedding", n=301, vocab=1400, d=384, dtype="f32", scale=1.0, gradient=True),
        # every position of a depth-32 trie over a character set beyond the shared-memory table
        dict(name="embedding-trie-1000", kind="embedding", n=1_400_003, vocab=1000, d=128, dtype="f32", scale=1.0, gradient=True),
        # a batch over a subword vocabulary, bfloat16, the table scaled by sqrt(d)
        dict(name="embedding-subwords-bf16", kind="embedding", n=65_537, vocab=50_021, d=1024, dtype="bf16", scale=32.0, gradient=True),
        # the next token of seven sequences: what answering one position costs
        dict(name="qk-next-tokens-8x64", kind="qk", n=7, heads=8, kv_heads=8, head_dim=64, dtype="f32", store="bf16", fused=False, gradient=False),
        # a few sampled units, six heads of 64, keys straight into a bfloat16 store
        dict(name="qk-sampled-6x64", kind="qk", n=1_733, heads=6, kv_heads=6, head_dim=64, dtype="f32", store="bf16", fused=False, gradient=True),
        # every position of a depth-32 trie, 4 x 32
        dict(name="qk-trie-4x32", kind="qk", n=1_400_003, heads=4, kv_heads=4, head_dim=32, dtype="f32", store="same", fused=False, gradient=True),
        # grouped heads in bfloat16, queries and keys columns of one projection's output
        dict(name="qk-grouped-32x128-bf16", kind="qk", n=40_961, heads=32, kv_heads=8, head_dim=128, dtype="bf16", store="same", fused=True, gradient=True),
        # the normalised rows of a sampled unit
        dict(name="round-trip-sampled-unit", kind="round_trip", n=301, cols=384, dtype="f32"),
        # the feed-forward activation of a launch group, d_ff 512
        dict(name="round-trip-feed-forward", kind="round_trip", n=560_003, cols=512, dtype="f32"),
        # first feed-forward projection of a few sampled units, d_model 384
        dict(name="backward-sampled-384-1536", kind="backward", n=1_733, m=384, cols=1536, relu=True),
        # both feed-forward projections of a launch group, d_model 128
        dict(name="backward-group-128-512", kind="backward", n=400_003, m=128, cols=512, relu=True),
        dict(name="backward-group-512-128", kind="backward", n=400_003, m=512, cols=128, relu=False),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["embedding", "qk", "round_trip", "backward"])
    if kind == "embedding":
        d = rng.choice([64, 65, 96, 128, 130, 256, 384, 512, 768, 1024])
        return dict(kind=kind, n=size(1, 170_000_000 // d), vocab=size(401, 60_000), d=d, dtype=rng.choice(["f32", "bf16"]),
                    scale=rng.choice([1.0, math.sqrt(d)]), gradient=rng.random() < 0.8)
    if kind == "qk":
        hd, kv = rng.choice([16, 32, 48, 64, 96, 128]), rng.choice([1, 2, 3, 4, 6, 8])
        heads = kv * rng.choice([1, 1, 2, 4])
        return dict(kind=kind, n=size(1, 180_000_000 // ((heads + kv) * hd)), heads=heads, kv_heads=kv, head_dim=hd, dtype=rng.choice(["f32", "bf16"]),
                    store=rng.choice(["same", "bf16"]), fused=rng.random() < 0.5, gradient=rng.random() < 0.8)
    if kind == "round_trip":
        cols = size(4, 2048)
        return dict(kind=kind, n=size(1, 280_000_000 // cols), cols=cols, dtype=rng.choice(["f32", "f32", "bf16"]))
    m, cols = size(16, 1024), size(16, 1024)
    return dict(kind=kind, n=size(1, min(250_000_000 // (m + 4 * cols), 26_000_000_000 // (m * cols))), m=m, cols=cols, relu=rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _tokens(n, vocab, gen):
    """Zipf-distributed tokens (a token's rank is log-uniform, its id a fixed shuffle of the rank); one row in a hundred is padding (-1)."""
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    ids = torch.randperm(vocab, device="cuda", generator=gen)[rank]
    return torch.where(torch.rand(n, device="cuda", generator=gen) < 0.01, torch.full_like(ids, -1), ids).to(torch.int32)


def _table(positions, head_dim):
    """cos and sin of position / 10000^(2 i / head_dim), each at 2 i and 2 i + 1."""
    i = torch.arange(head_dim // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (2 * i / head_dim)
    return tuple(f(a).float().repeat_interleave(2, 1).contiguous() for f in (torch.cos, torch.sin))


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    kind, n = case["kind"], case["n"]
    s = dict(case=case)
    if kind == "embedding":
        s["ids"] = _tokens(n, case["vocab"], gen)
        s["table"] = (0.02 * randn(case["vocab"], case["d"])).to(_type(case))
        s["grad"] = randn(n, case["d"]).to(_type(case)) if case["gradient"] else None
    elif kind == "qk":
        hq, hk, hd = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"], case["head_dim"]
        if case["fused"]:
            both = randn(n, hq + 2 * hk).to(_type(case))
            s["q"], s["k"] = both[:, :hq], both[:, hq:hq + hk]
        else:
            s["q"], s["k"] = randn(n, hq).to(_type(case)), randn(n, hk).to(_type(case))
        s["gains"] = [1 + 0.1 * randn(hd) for _ in range(2)]
        s["cos"], s["sin"] = _table(4096, hd)
        s["pos"] = torch.randint(0, 4096, (n,), device="cuda", generator=gen, dtype=torch.int32)
        s["k_type"] = torch.bfloat16 if case["store"] == "bf16" else _type(case)
        s["dy"] = [randn(n, hq).to(_type(case)), randn(n, hk).to(_type(case))] if case["gradient"] else None
    elif kind == "round_trip":
        s["x"] = randn(n, case["cols"]).to(_type(case))
    else:
        s["grad"] = randn(n, case["cols"]) * 1e-3
        s["x"] = _pack(randn(n, case["m"]))
        s["y"] = _pack(torch.relu(randn(n, case["cols"]))) if case["relu"] else None
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _pack(x):
    """(codes, scales) of a float tensor.  The scale of a block is the smallest power of two with amax <= 448 of it (2^-110 at least); a value that
    is not zero keeps its sign and the smallest code at least."""
    n, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.nn.functional.pad(x.float(), (0, blocks * 32 - cols)).view(n, blocks, 32)
    amax = v.abs().amax(2)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8), torch.full_like(e, -110)).clamp(-110, 120)
    codes = (v * ((127 - e) << 23).view(torch.float32)[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    lost = (v != 0) & ((codes & 127) == 0)
    codes = torch.where(lost, (v < 0).to(torch.uint8) * 128 + 1, codes)
    scales = torch.full((blocks, (n + 15) // 16 * 16), 127, dtype=torch.uint8, device=x.device)
    scales[:, :n] = (e + 127).to(torch.uint8).t()
    return codes.reshape(n, blocks * 32), scales


def _values(packed, cols):
    codes, scales = packed
    n, blocks = codes.shape[0], scales.shape[0]
    f = (scales[:, :n].t().int() << 23).view(torch.float32)
    return (codes.view(torch.float8_e4m3fn).float().view(n, blocks, 32) * f[:, :, None]).reshape(n, blocks * 32)[:, :cols]


def _rotate(v, cos, sin):
    a, b = v[..., 0::2], v[..., 1::2]
    c, t = cos[..., 0::2], sin[..., 0::2]
    return torch.stack([a * c - b * t, a * t + b * c], -1).flatten(-2)


def _norm_rope(x, gain, cos, sin, out):
    v = x.float().view(x.shape[0], -1, gain.numel())
    r = 1.0 / torch.sqrt((v * v).mean(2, keepdim=True) + EPS)
    return _rotate(v * r * gain, cos[:, None], sin[:, None]).view(x.shape).to(out)


def _norm_rope_backward(dy, x, gain, cos, sin):
    v = x.float().view(x.shape[0], -1, gain.numel())
    r = 1.0 / torch.sqrt((v * v).mean(2, keepdim=True) + EPS)
    u = v * r
    w = _rotate(dy.float().view(v.shape), cos[:, None], -sin[:, None])
    dgain = (w * u).sum((0, 1))
    c = w * gain
    return (r * (c - u * (c * u).mean(2, keepdim=True))).view(x.shape).to(x.dtype), dgain


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s, case, kind)
    if kind == "embedding":
        ids, table = s["ids"].long(), s["table"]
        live = (ids >= 0) & (ids < case["vocab"])
        out = torch.where(live[:, None], table[ids.clamp(0, case["vocab"] - 1)].float() * case["scale"], 0.0).to(table.dtype)
        if not case["gradient"]:
            return dict(rows=out)
        grad = torch.zeros(case["vocab"] + 1, case["d"], device="cuda")
        grad.index_add_(0, torch.where(live, ids, torch.full_like(ids, case["vocab"])), s["grad"].float())
        return dict(rows=out, table=grad[:-1] * case["scale"])
    if kind == "qk":
        cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
        q, k, (gq, gk) = s["q"], s["k"], s["gains"]
        out = dict(q=_norm_rope(q, gq, cos, sin, q.dtype), k=_norm_rope(k, gk, cos, sin, s["k_type"]))
        if case["gradient"]:
            out["dq"], out["dq_gain"] = _norm_rope_backward(s["dy"][0], q, gq, cos, sin)
            out["dk"], out["dk_gain"] = _norm_rope_backward(s["dy"][1], k, gk, cos, sin)
        return out
    if kind == "round_trip":
        return dict(values=_values(_pack(s["x"]), case["cols"]))
    grad = s["grad"]
    if case["relu"]:
        grad = torch.where(_values(s["y"], case["cols"]) > 0, grad, 0.0)
    return dict(grad=grad, weight=_values(s["x"], case["m"]).t() @ grad, bias=grad.sum(0))


def _run_own(s, case, kind):
    import agpt_b200 as A
    if kind == "embedding":
        out = dict(rows=A.embedding_lookup(s["table"], s["ids"], case["scale"]))
        if case["gradient"]:
            out["table"] = A.embedding_grad_sorted(s["grad"], s["ids"], case["vocab"], case["scale"])
        return out
    if kind == "qk":
        (gq, gk), tab = s["gains"], (s["pos"], s["cos"], s["sin"])
        q, k = A.qk_norm_rope(s["q"], s["k"], gq, gk, *tab, eps=EPS, k_dtype=s["k_type"])
        if not case["gradient"]:
            return dict(q=q, k=k)
        dgq, dgk = torch.zeros_like(gq), torch.zeros_like(gk)
        dq, dk = A.qk_norm_rope_backward(*s["dy"], s["q"], s["k"], gq, gk, *tab, dgq, dgk, eps=EPS)
        return dict(q=q, k=k, dq=dq, dk=dk, dq_gain=dgq, dk_gain=dgk)
    if kind == "round_trip":
        return dict(values=A.act8_unpack(A.act8_pack(s["x"])))
    grad = s["grad"]
    if case["relu"]:
        grad = A.act8_relu_backward(grad, A.Act8(*s["y"], case["cols"]))
    weight, bias = A.act8_weight_grad(A.Act8(*s["x"], case["m"]), grad)
    return dict(grad=grad, weight=weight, bias=bias)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    kind, n = case["kind"], case["n"]
    if kind == "embedding":
        e, d, rows = (2 if case["dtype"] == "bf16" else 4), case["d"], min(case["n"], case["vocab"])
        b, f = 4.0 * n + rows * d * e + n * d * e, 1.0 * n * d
        if case["gradient"]:            # the tokens again, the rows' gradients, the table's gradient
            b, f = b + 4.0 * n + n * d * e + 4.0 * case["vocab"] * d, f + 2.0 * n * d
        return dict(bytes=b, flops=f)
    if kind == "qk":
        e = 2 if case["dtype"] == "bf16" else 4
        q, k = n * case["heads"] * case["head_dim"], n * case["kv_heads"] * case["head_dim"]
        b, f = 4.0 * n + (q + k) * e + q * e + k * (2 if case["store"] == "bf16" else e), 9.0 * (q + k)
        if case["gradient"]:            # x and dy in, dx out
            b, f = b + 4.0 * n + 3.0 * (q + k) * e, f + 20.0 * (q + k)
        return dict(bytes=b, flops=f)
    if kind == "round_trip":            # values in, codes and scales out and in, values out
        v, e = n * case["cols"], 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=v * (e + 2 * 33 / 32 + 4), flops=5.0 * v)
    m, c = case["m"], case["cols"]
    b = n * (m * 33 / 32 + 4.0 * c) + 4.0 * (m + 1) * c
    if case["relu"]:
        b += n * (c * 33 / 32 + 4.0 * c)
    return dict(bytes=b, flops=2.0 * n * m * c)


# ---- the operators in 64 bits -------------------------------------------------------------------------------------------
def _two(e):
    """2^e exactly, from the bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(packed, cols):
    """The numbers of a checkpoint from its bits: sign, four bits of exponent, three of fraction."""
    codes, scales = packed
    c, n = codes.long(), codes.shape[0]
    exponent, fraction = (c >> 3) & 15, (c & 7).double()
    size = torch.where(exponent == 0, fraction / 8 * 2.0 ** -6, (1 + fraction / 8) * _two(exponent - 7))
    size = torch.where(c >= 128, -size, size)
    up = _two(scales[:, :n].t().long() - 127)
    return (size * up.repeat_interleave(32, 1))[:, :cols]


def _exact_round_trip(x):
    """Values at eight bits: the step of a binade is an eighth of its power of two, below the smallest normal number it stays what it is there."""
    n, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(n, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.view(n, blocks, 32)
    top = v.abs().amax(2, keepdim=True).clamp_min(2.0 ** -140)
    base = _two(torch.ceil(torch.log2(top / 448.0) - 1e-13).clamp(-110, 120))
    base = torch.where((top > 448.0 * base) & (base < 2.0 ** 120), base * 2, base)
    size = v.abs() / base
    binade = torch.floor(torch.log2(size.clamp_min(2.0 ** -6)) + 1e-14)
    step = _two(binade - 3)
    got = torch.round(size / step) * step
    got = torch.where((size > 0) & (got == 0), 2.0 ** -9, got) * base * torch.sign(v)
    return got.reshape(n, blocks * 32)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    kind, n = case["kind"], case["n"]
    if kind == "embedding":
        ids, vocab = s["ids"].long(), case["vocab"]
        inside = (ids >= 0) & (ids < vocab)
        grown = torch.cat([s["table"].double() * case["scale"], torch.zeros(1, case["d"], dtype=torch.float64, device="cuda")])
        ids = torch.where(inside, ids, torch.full_like(ids, vocab))
        out = dict(rows=grown[ids])
        if case["gradient"]:            # differences of a running sum over the rows in the order of their tokens
            order = torch.sort(ids, stable=True)
            run_sum = torch.cumsum(torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device="cuda"), s["grad"].double()[order.indices]]), 0)
            edge = torch.searchsorted(order.values, torch.arange(vocab + 1, device="cuda"))
            out["table"] = (run_sum[edge[1:]] - run_sum[edge[:-1]]) * case["scale"]
        return out
    if kind == "qk":
        angle = torch.complex(s["cos"].double()[:, 0::2], s["sin"].double()[:, 0::2])[s["pos"].long()][:, None]
        out = {}
        for name, x, gain, i in (("q", s["q"], s["gains"][0], 0), ("k", s["k"], s["gains"][1], 1)):
            v = x.double().reshape(n, -1, case["head_dim"])
            g, r = gain.double(), torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
            turned = torch.view_as_complex((v * g * r).reshape(*v.shape[:2], -1, 2)) * angle
            out[name] = torch.view_as_real(turned).reshape(x.shape)
            if case["gradient"]:
                back = torch.view_as_complex(s["dy"][i].double().reshape(*v.shape[:2], -1, 2)) * angle.conj()
                back = torch.view_as_real(back).reshape(v.shape)
                out["d%s_gain" % name] = (back * v * r).sum((0, 1))
                back = back * g
                out["d" + name] = (r * back - r ** 3 * v * (back * v).mean(-1, keepdim=True)).reshape(x.shape)
        return out
    if kind == "round_trip":
        return dict(values=_exact_round_trip(s["x"]))
    grad = s["grad"].double()
    if case["relu"]:
        grad = grad * (_exact_values(s["y"], case["cols"]) > 0)
    return dict(grad=grad, weight=torch.mm(grad.t(), _exact_values(s["x"], case["m"])).t(), bias=grad.t().mv(torch.ones(n, dtype=torch.float64, device="cuda")))
