"""The file of query and key gains beside a model."""
import numpy as np
import pytest

from agpt_b200 import model_file as MF


def test_round_trip_and_refusals(tmp_path):
    path = str(tmp_path / "m.model") + MF.GAINS_SUFFIX
    gains = {k: np.random.default_rng(i).standard_normal((1, 16)).astype(np.float32) for i, k in enumerate(MF.gain_names(3))}
    MF.save_gains(path, gains)
    got = MF.load_gains(path, 3, 16)
    assert list(got) == ["layer0.qn.gain", "layer0.kn.gain", "layer1.qn.gain", "layer1.kn.gain", "layer2.qn.gain", "layer2.kn.gain"]
    assert all(np.array_equal(got[k], gains[k]) for k in gains)
    for layers, hd in ((2, 16), (3, 32), (4, 16)):
        with pytest.raises(ValueError):
            MF.load_gains(path, layers, hd)
    raw = open(path, "rb").read()
    for bad in (raw[:-4], raw + b"\0", b"XXXX" + raw[4:], raw[:8] + b"\2\0\0\0" + raw[12:], b""):
        open(path, "wb").write(bad)
        with pytest.raises(ValueError):
            MF.load_gains(path, 3, 16)
