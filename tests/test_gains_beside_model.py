"""The gains file beside a model file is that model's, or is not there."""
import os

import numpy as np

from agpt_b200 import model_file as MF


def test_gains_go_with_the_model(tmp_path):
    path = str(tmp_path / "m.model")
    m = MF.random_init(32, 2, 2, 11, 16, seed=1)
    gains = {name: np.full((1, 16), i + 1, np.float32) for i, name in enumerate(MF.gain_names(2))}
    MF.save_with_gains(path, m, gains)
    back = MF.load_gains(path + MF.GAINS_SUFFIX, 2, 16)
    assert list(back) == list(gains) and all(np.array_equal(back[k], gains[k]) for k in gains)
    MF.save_with_gains(path, m, {})
    assert os.listdir(tmp_path) == ["m.model"]
    MF.save_with_gains(path, m, {})                              # nothing beside it: nothing to take away
    assert [n for n, _ in MF.load(path).mats] == [n for n, _ in m.mats]
