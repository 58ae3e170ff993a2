"""The row operators as the trainer uses them: a vocabulary beyond the shared-memory table with a scaled embedding, normalised queries and keys, 8-bit
activations, alone and together, against a dense float64 model; and from the command line."""
import os

import numpy as np
import pytest

import agpt_b200 as A
from agpt_b200 import model_file as MF
from agpt_b200 import trainer as T
from tests import row_forms as F
from tests.helpers import TOL_BF16, TOL_F32, rel_err
from tests.test_train_step_gpu import _group

pytestmark = pytest.mark.gpu


def _part(name):
    return (name.split(".") + [""])[1]


def _model(d, heads, layers, vocab, seed=3):
    mf = MF.random_init(d, heads, layers, vocab, 64, seed=seed, std=0.1)
    rng = np.random.default_rng(7)
    mf.mats = [(k, (a + 0.1 * rng.standard_normal(a.shape)).astype(np.float32)) for k, a in mf.mats]
    # feed-forward units well away from the kink of the ReLU (the same float32 sum in another order may fall on its other side)
    mf.mats = [(k, a * 0.1 if k.endswith("l1.w") else (np.where(np.arange(a.size) % 3, 0.5, -0.5).astype(np.float32)[None] if k.endswith("l1.b") else a))
               for k, a in mf.mats]
    return mf


def _dense(model, g, cotangent, qk_norm, scale, bf16=False):
    """float64 logits and gradients of sum(logits * cotangent): every row attends its ancestors and itself."""
    import torch
    m, P = model.cfg, {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.params.items()}
    parent, n, H, hd = g.plan.parent_dfs, g.n, m.n_heads, m.d_model // m.n_heads
    mask = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        a = i
        while a >= 0:
            mask[i, a] = True
            a = int(parent[a])
    pos = g.pos.cpu().long()
    cos, sin = [t.cpu().double()[pos][:, None, 0::2] for t in (model.cos, model.sin)]

    def ln(x, gain, shift):
        return (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5) * gain + shift

    def rope(x):
        e, o = x[..., 0::2], x[..., 1::2]
        return torch.stack([e * cos - o * sin, e * sin + o * cos], -1).flatten(-2)

    def rms(x, gain):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain

    def stored(x):          # the store's rounding, with the gradient of the unrounded value
        return x + (x.float().bfloat16().double() - x).detach() if bf16 else x

    x = P["token_emb"][g.tokens.cpu().long()] * scale
    for l in range(m.n_layers):
        w = lambda k: P[f"layer{l}.{k}"]  # noqa: E731
        y = ln(x, w("ln1.gamma"), w("ln1.beta"))
        q, k, v = [(y @ w(f"w{c}.w") + w(f"w{c}.b")).view(n, H, hd) for c in "qkv"]
        if qk_norm:
            q, k = rms(q, w("qn.gain")), rms(k, w("kn.gain"))
        q, k, v = rope(q), stored(rope(k)), stored(v)
        s = torch.einsum("ihc,jhc->hij", q, k) / np.sqrt(hd)
        p = torch.softmax(s.masked_fill(~mask, -np.inf), -1)
        x = x + torch.einsum("hij,jhc->ihc", p, v).reshape(n, -1) @ w("wo.w") + w("wo.b")
        y = ln(x, w("ln2.gamma"), w("ln2.beta"))
        x = x + torch.relu(y @ w("l1.w") + w("l1.b")) @ w("l2.w") + w("l2.b")
    logits = ln(x, P["final.gamma"], P["final.beta"]) @ P["out.w"] + P["out.b"]
    (logits * cotangent.cpu().double()).sum().backward()
    return logits.detach().numpy(), {k: v.grad.numpy() for k, v in P.items()}


def _run(model, g, cotangent, **kw):
    model.flat_grad.zero_()
    logits = model.logits(g, **kw)[:, :model.cfg.vocab]
    logits.backward(cotangent)
    return logits.detach().cpu().numpy(), {k: v.grad.cpu().numpy().copy() for k, v in model.params.items()}


@pytest.mark.parametrize("n,depth,d,heads,vocab,qk_norm,scale,bf16", [
    (1, 1, 32, 2, 401, True, 2.0, False),
    (300, 20, 64, 4, 1000, False, 8.0, False),
    (300, 20, 64, 2, 65, True, 1.0, False),
    (257, 40, 128, 2, 1397, True, 11.3, False),
    (300, 20, 64, 4, 500, True, 1.0, True),
])
def test_gradients_match_a_dense_model(cuda, n, depth, d, heads, vocab, qk_norm, scale, bf16):
    import torch
    g, _ = _group(n, depth, vocab, n + d, 64, cuda)
    model = T.TrieWalkModel(_model(d, heads, 2, vocab), cuda, qk_norm, scale)
    if qk_norm:
        rng = np.random.default_rng(5)
        model.set_qk_gains({k: (a + 0.3 * rng.standard_normal(a.shape)).astype(np.float32) for k, a in model.qk_gains().items()})
    cotangent = torch.randn(n, vocab, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)) / n
    want_y, want = _dense(model, g, cotangent, qk_norm, scale, bf16)
    got_y, got = _run(model, g, cotangent, bf16_store=bf16)
    tol = TOL_BF16 if bf16 else TOL_F32
    assert rel_err(got_y, want_y) < tol
    for k in want:
        if n == 1 and _part(k) in ("wq", "wk", "qn", "kn"):
            # One key: the probability is 1 and these gradients are 0.  dS = dP - delta is the difference of two equal sums of hd products, each off by (hd + 1) u
            # |v| |dout| at most; dq = dS k / sqrt(hd), times r g of the norm.  Next to dWv = x dout that is 2 (hd + 1) u |v| |k| r g / sqrt(hd), with |k| <= sqrt(hd)
            # max g, |v| < 8 and r max g^2 < 6 here less than 100 (hd + 1) u of its largest entry, whatever the entries' places.
            hd, dv = d // heads, np.abs(want[k.split(".")[0] + ".wv.w"]).max()
            assert np.abs(want[k]).max() < 1e-12 and np.abs(got[k]).max() <= 100 * (hd + 1) * F.U * max(dv, np.abs(want[k.split(".")[0] + ".wv.b"]).max()), k
            continue
        assert rel_err(got[k].astype(np.float64), want[k], floor=1e-6) < tol, k
    # together with 8-bit activations the forward is the same, and so is every gradient that no kept activation enters
    model.activations_8bit = True
    y8, g8 = _run(model, g, cotangent, bf16_store=bf16)
    assert np.array_equal(y8, got_y)
    for k in got:
        if _part(k) in ("wq", "wk", "wv", "l1", "l2"):
            assert np.isfinite(g8[k]).all() and (k.endswith(".b") or n == 1 or not np.array_equal(g8[k], got[k]))
        else:
            assert np.array_equal(g8[k], got[k]), k
    again = _run(model, g, cotangent, bf16_store=bf16)
    assert all(np.array_equal(again[1][k], g8[k]) for k in g8)                    # repeatable bit for bit


@pytest.mark.parametrize("n,d,ff", [(1, 32, 64), (333, 64, 256), (1500, 96, 388)])
def test_projections_over_8_bit_activations(cuda, n, d, ff):
    """The feed-forward and q/k/v functions against float64 with the kept inputs in the weight gradients and the exact ones elsewhere."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(n)
    randn = lambda *s: torch.randn(*s, device=cuda, generator=gen)  # noqa: E731
    x, res, w1, b1, w2, b2 = randn(n, d), randn(n, d), 0.2 * randn(d, ff), 0.2 * randn(ff), 0.2 * randn(ff, d), 0.2 * randn(d)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, b1, w2, b2, res)]
    dy = randn(n, d)
    T._ffn8_function().apply(*leaves).backward(dy)
    D = lambda t: t.detach().cpu().double().numpy()  # noqa: E731
    h = A.gemm_f32(x, w1, bias=b1, relu=True)
    x8, h8 = [D(A.act8_unpack(A.act8_pack(t))) for t in (x, h)]
    dh = np.where(D(h) > 0, D(dy) @ D(w2).T, 0.0)
    got = [D(t.grad) for t in leaves]
    for a, b in zip(got, (dh @ D(w1).T, x8.T @ dh, dh.sum(0), h8.T @ D(dy), D(dy).sum(0), D(dy))):
        assert rel_err(a, b) < TOL_F32
    # and against the exact inputs: a kept value is off by 2^-4 of itself, or half a step of its block, at most
    step = np.repeat(np.abs(np.pad(D(x), ((0, 0), (0, -d % 32)))).reshape(n, -1, 32).max(2), 32, 1)[:, :d] / 224 * 2.0 ** -9
    assert (np.abs(got[1] - D(x).T @ dh) <= np.maximum(np.abs(D(x)) / 16, step).T @ np.abs(dh) + 1e-4 * np.abs(D(x)).T @ np.abs(dh)).all()
    ws = [0.2 * randn(d, d) for _ in range(3)]
    args = [x.clone().requires_grad_(True)] + [t.clone().requires_grad_(True) for w in ws for t in (w, randn(d))]
    cot = [randn(n, d) for _ in range(3)]
    torch.autograd.backward(T._qkv8_function().apply(*args), cot)
    want = [sum(D(c) @ D(w).T for c, w in zip(cot, ws))] + [t for c in cot for t in (x8.T @ D(c), D(c).sum(0))]
    for a, b in zip(args, want):
        assert rel_err(D(a.grad), b) < TOL_F32


def test_8_bit_activations_take_less_memory(cuda):
    import torch
    n, d, layers = 20_000, 128, 4
    g, _ = _group(n, 12, 65, 3, 64, cuda)
    model = T.TrieWalkModel(_model(d, 4, layers, 65), cuda)
    peak = {}
    for eight in (False, True):
        model.activations_8bit = eight
        for _ in range(2):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = model.logits(g)
            peak[eight] = torch.cuda.memory_allocated() - before
            del y
    # a layer keeps two inputs of d and one of 4 d columns in 1 + 1/32 bytes an element instead of 4 (the ReLU's output once)
    saved = layers * n * 6 * d * (4 - 33 / 32)
    assert peak[False] - peak[True] >= 0.95 * saved


def test_combinations_that_are_refused(cuda):
    g, _ = _group(30, 6, 65, 3, 64, cuda)
    model = T.TrieWalkModel(_model(32, 2, 1, 65), cuda)
    model.activations_8bit = True
    for attribute, value in (("ffn_recompute", True), ("dense_impl", "torch")):
        old = getattr(model, attribute)
        setattr(model, attribute, value)
        with pytest.raises(A.AgptError, match="8-bit"):
            model.logits(g)
        setattr(model, attribute, old)
    assert not model.native_step_available()
    model.activations_8bit = False
    assert model.native_step_available()


def test_epochs_with_everything_on(cuda):
    """Two epochs over a trie of 700 symbols, both kinds of units, repeat bit for bit."""
    import torch
    trie = A.RadixTrie.build(A.synth_markov_corpus(3000, 700, 1, 4), 5)
    counts = [torch.tensor(np.asarray(c), dtype=torch.int32, device=cuda) for c in (trie.cnt_off, trie.cnt_tok, trie.cnt_val)]
    groups, _ = T.build_groups(trie, 0, 1, 4000, "linear", 64, cuda)

    def run():
        model = T.TrieWalkModel(MF.random_init(64, 4, 2, 700, 64, seed=2), cuda, qk_norm=True, embed_scale=8.0)
        model.activations_8bit = True
        opt = T.make_optimizer("adam", model, 1e-3)
        out = [T.train_epoch(model, groups, counts, opt, bf16_store=b) for b in (False, True)]
        out.append(T.train_lightning_epoch(model, T.SampleSpace(trie), counts, opt, 3, 4, 9)[:3])
        return out, model.flat.clone(), model
    a, flat_a, model = run()
    b, flat_b, _ = run()
    assert a == b and torch.equal(flat_a, flat_b) and torch.isfinite(flat_a).all()
    assert all(np.abs(v - 1).max() > 0 for v in model.qk_gains().values())                     # the gains are trained
    assert A.device_status() == 0


def test_from_the_command_line(cuda, tmp_path):
    trie = A.RadixTrie.build(A.synth_markov_corpus(2000, 500, 1, 5), 4)
    trie.save_dir(str(tmp_path / "trie"), 2000, 500, 1)
    mf = MF.random_init(32, 2, 1, 500, 64, seed=1)
    MF.save(str(tmp_path / "m.model"), mf)
    common = ["--model", str(tmp_path / "m.model"), "--trie-dir", str(tmp_path / "trie"), "--embed-scale", "5.6"]
    T.main(common + ["--qk-norm", "--activations-8bit", "--save", str(tmp_path / "o.model")])
    gains = MF.load_gains(str(tmp_path / "o.model") + MF.GAINS_SUFFIX, 1, 16)
    assert list(gains) == MF.gain_names(1) and all(np.abs(g - 1).max() > 0 for g in gains.values())
    common[1] = str(tmp_path / "o.model")
    T.main(common + ["--qk-norm"])                                                             # read back, trained on, saved in place
    again = MF.load_gains(str(tmp_path / "o.model") + MF.GAINS_SUFFIX, 1, 16)
    assert any(not np.array_equal(again[k], gains[k]) for k in gains)
    with pytest.raises(SystemExit):
        T.main(common)                                                                         # trained with the norms, asked for without
    with pytest.raises(SystemExit):
        T.main(common + ["--qk-norm", "--activations-8bit", "--ffn-recompute"])
    os.remove(str(tmp_path / "o.model") + MF.GAINS_SUFFIX)
    T.main(common)
