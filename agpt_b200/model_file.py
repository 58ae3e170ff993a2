"""MGPT model file: the checkpoint format of the reference trainer, read and written unchanged.

Layout (src/cuda/agpt_train.cu:1209-1296): u32 magic 0x4D475054, i32 d_model, n_heads, n_layers, d_ff,
vocab, seq_len, then 1 + 16*n_layers + 4 matrices, each i32 rows, i32 cols, f32[rows*cols] row-major
([d_in, d_out], y = x W + b), in the order token_emb; per layer wq.w, wq.b, wk.w, wk.b, wv.w, wv.b, wo.w,
wo.b, ln1.gamma, ln1.beta, l1.w, l1.b, l2.w, l2.b, ln2.gamma, ln2.beta; final gamma, beta; out.w, out.b.
"""
from __future__ import annotations

import os
import struct
from dataclasses import dataclass, field

import numpy as np

MAGIC = 0x4D475054
LAYER_NAMES = ("wq.w", "wq.b", "wk.w", "wk.b", "wv.w", "wv.b", "wo.w", "wo.b", "ln1.gamma", "ln1.beta",
               "l1.w", "l1.b", "l2.w", "l2.b", "ln2.gamma", "ln2.beta")


@dataclass
class Model:
    d_model: int
    n_heads: int
    n_layers: int
    d_ff: int
    vocab: int
    seq_len: int
    mats: list = field(default_factory=list)     # [(name, float32 array [rows, cols])] in file order

    def names(self):
        out = ["token_emb"]
        for l in range(self.n_layers):
            out += [f"layer{l}.{n}" for n in LAYER_NAMES]
        return out + ["final.gamma", "final.beta", "out.w", "out.b"]

    def expected_shapes(self):
        D, F, V = self.d_model, self.d_ff, self.vocab
        per = [(D, D), (1, D)] * 4 + [(1, D), (1, D), (D, F), (1, F), (F, D), (1, D), (1, D), (1, D)]
        return [(V, D)] + per * self.n_layers + [(1, D), (1, D), (D, V), (1, V)]

    def get(self, name):
        return dict(self.mats)[name]


def load(path: str) -> Model:
    with open(path, "rb") as f:
        raw = f.read()
    if len(raw) < 28 or struct.unpack_from("<I", raw, 0)[0] != MAGIC:
        raise ValueError(f"{path}: bad model magic")
    d_model, n_heads, n_layers, d_ff, vocab, seq_len = struct.unpack_from("<6i", raw, 4)
    m = Model(d_model, n_heads, n_layers, d_ff, vocab, seq_len)
    off = 28
    for name, shape in zip(m.names(), m.expected_shapes()):
        rows, cols = struct.unpack_from("<2i", raw, off)
        off += 8
        if (rows, cols) != shape:
            raise ValueError(f"{path}: matrix {name} is {rows}x{cols}, expected {shape[0]}x{shape[1]}")
        cnt = rows * cols
        m.mats.append((name, np.frombuffer(raw, dtype="<f4", count=cnt, offset=off).reshape(rows, cols).copy()))
        off += cnt * 4
    if off != len(raw):
        raise ValueError(f"{path}: {len(raw) - off} trailing bytes")
    return m


def save(path: str, m: Model) -> None:
    with open(path, "wb") as f:
        f.write(struct.pack("<I6i", MAGIC, m.d_model, m.n_heads, m.n_layers, m.d_ff, m.vocab, m.seq_len))
        for (name, a), shape in zip(m.mats, m.expected_shapes()):
            a = np.ascontiguousarray(a, dtype="<f4")
            if a.shape != shape:
                raise ValueError(f"matrix {name} has shape {a.shape}, expected {shape}")
            f.write(struct.pack("<2i", *shape))
            f.write(a.tobytes())


# Gains of the query and key norms, which the model file has no place for: a file beside it, u32 magic, i32 count, then
# matrices [1, head_dim] as in the model file, per layer those of the queries and of the keys.
GAINS_MAGIC, GAINS_SUFFIX = 0x4E474B51, ".qk_gains"


def load_gains(path: str, n_layers: int, head_dim: int):
    """{name: float32 [1, head_dim]} of a gains file."""
    with open(path, "rb") as f:
        raw = f.read()
    if len(raw) != 8 + 2 * n_layers * (8 + 4 * head_dim) or struct.unpack_from("<Ii", raw, 0) != (GAINS_MAGIC, 2 * n_layers):
        raise ValueError(f"{path}: not the query and key gains of {n_layers} layers with heads of {head_dim}")
    out, off = {}, 8
    for name in gain_names(n_layers):
        if struct.unpack_from("<2i", raw, off) != (1, head_dim):
            raise ValueError(f"{path}: {name} is not 1x{head_dim}")
        out[name] = np.frombuffer(raw, dtype="<f4", count=head_dim, offset=off + 8).reshape(1, head_dim).copy()
        off += 8 + 4 * head_dim
    return out


def save_gains(path: str, gains) -> None:
    with open(path, "wb") as f:
        f.write(struct.pack("<Ii", GAINS_MAGIC, len(gains)))
        for a in gains.values():
            a = np.ascontiguousarray(a, dtype="<f4")
            f.write(struct.pack("<2i", 1, a.size))
            f.write(a.tobytes())


# The factor on the embedding, which is part of the function that the weights were trained for: a file beside the model, u32 magic, f64 factor; no file: 1.
SCALE_MAGIC, SCALE_SUFFIX = 0x4C435345, ".embed_scale"


def load_embed_scale(model_path: str) -> float:
    """The factor on the embedding that the model was saved with."""
    path = model_path + SCALE_SUFFIX
    if not os.path.exists(path):
        return 1.0
    with open(path, "rb") as f:
        raw = f.read()
    if len(raw) != 12 or struct.unpack_from("<I", raw, 0)[0] != SCALE_MAGIC:
        raise ValueError(f"{path}: not the embedding factor of a model")
    return struct.unpack_from("<d", raw, 4)[0]


def same_embed_scale(a: float, b: float) -> bool:
    """Equal as the float32 numbers that the rows are multiplied with."""
    return np.float32(a) == np.float32(b)


def save_with_gains(path: str, m: Model, gains, embed_scale: float = 1.0) -> None:
    """The model file and, beside it, its gains file and its embedding factor.  Without gains, or with a factor of 1, a file that an earlier model left there
    goes: it would be read as this model's."""
    save(path, m)
    if gains:
        save_gains(path + GAINS_SUFFIX, gains)
    elif os.path.exists(path + GAINS_SUFFIX):
        os.remove(path + GAINS_SUFFIX)
    if not same_embed_scale(embed_scale, 1.0):
        with open(path + SCALE_SUFFIX, "wb") as f:
            f.write(struct.pack("<Id", SCALE_MAGIC, embed_scale))
    elif os.path.exists(path + SCALE_SUFFIX):
        os.remove(path + SCALE_SUFFIX)


def gain_names(n_layers: int):
    return [f"layer{l}.{n}.gain" for l in range(n_layers) for n in ("qn", "kn")]


def random_init(d_model, n_heads, n_layers, vocab, seq_len, d_ff=None, seed=0, std=0.02) -> Model:
    """Seeded N(0, std) weights, gamma 1, beta and biases 0, in file order."""
    d_ff = 4 * d_model if d_ff is None else d_ff
    m = Model(d_model, n_heads, n_layers, d_ff, vocab, seq_len)
    rng = np.random.default_rng(seed)
    for name, shape in zip(m.names(), m.expected_shapes()):
        if name.endswith("gamma"):
            a = np.ones(shape, np.float32)
        elif name.endswith(".b") or name.endswith("beta"):
            a = np.zeros(shape, np.float32)
        else:
            a = (rng.standard_normal(shape) * std).astype(np.float32)
        m.mats.append((name, a))
    return m
