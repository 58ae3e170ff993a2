"""The factor on the embedding goes with the model: kept beside the model file, and another one is refused."""
import os

import pytest

from agpt_b200 import model_file as MF
from agpt_b200 import trainer as T


def test_kept_beside_the_model(tmp_path):
    path = str(tmp_path / "m.model")
    m = MF.random_init(32, 2, 1, 11, 16, seed=1)
    MF.save_with_gains(path, m, {})
    assert MF.load_embed_scale(path) == 1.0 and os.listdir(tmp_path) == ["m.model"]
    MF.save_with_gains(path, m, {}, 11.3)
    assert MF.load_embed_scale(path) == 11.3 and sorted(os.listdir(tmp_path)) == ["m.model", "m.model.embed_scale"]
    MF.save_with_gains(path, m, {}, 1.0)                         # saved over it: the factor of the earlier model goes
    assert os.listdir(tmp_path) == ["m.model"]
    MF.save_with_gains(path, m, {}, 2.0)
    raw = open(path + MF.SCALE_SUFFIX, "rb").read()
    for bad in (b"", raw[:-1], raw + b"\0", b"XXXX" + raw[4:]):
        open(path + MF.SCALE_SUFFIX, "wb").write(bad)
        with pytest.raises(ValueError):
            MF.load_embed_scale(path)


def test_the_trainer_refuses_another_factor(tmp_path):
    """Before it looks for a device or a trie."""
    path = str(tmp_path / "m.model")
    MF.save_with_gains(path, MF.random_init(32, 2, 1, 11, 16, seed=1), {}, 5.6)
    args = ["--model", path, "--trie-dir", str(tmp_path / "none")]
    for more in ([], ["--embed-scale", "1"], ["--embed-scale", "5.7"]):
        with pytest.raises(SystemExit, match="5.6"):
            T.main(args + more)


@pytest.mark.gpu
def test_from_the_command_line(cuda, tmp_path):
    import agpt_b200 as A
    trie = A.RadixTrie.build(A.synth_markov_corpus(2000, 65, 1, 5), 4)
    trie.save_dir(str(tmp_path / "trie"), 2000, 65, 1)
    MF.save(str(tmp_path / "m.model"), MF.random_init(32, 2, 1, 65, 64, seed=1))
    args = ["--model", str(tmp_path / "m.model"), "--trie-dir", str(tmp_path / "trie"), "--save", str(tmp_path / "o.model"), "--save-every", "1"]
    T.main(args + ["--embed-scale", "5.6"])
    assert MF.load_embed_scale(str(tmp_path / "o.model")) == 5.6 == MF.load_embed_scale(str(tmp_path / "o.model.ep1"))
    args[1] = str(tmp_path / "o.model")
    with pytest.raises(SystemExit):
        T.main(args)
    T.main(args + ["--embed-scale", "5.6"])
    T.main(["--model", str(tmp_path / "m.model")] + args[2:])    # trained without a factor, saved in its place
    assert MF.load_embed_scale(str(tmp_path / "o.model")) == 1.0
