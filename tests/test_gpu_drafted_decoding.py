"""Drafted greedy decoding gives the tokens of one-token greedy decoding, which reproduces the reference's (tests/golden/
greedy_7m_golden.npz), near-ties of the router among them: at the 16th generated token two experts are 9.5e-5 apart, which queries or
weights of 8 bits do not resolve."""
from pathlib import Path

import numpy as np
import pytest

from gptoss_b200 import binfmt, synth

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

GREEDY = Path(__file__).parent / "golden" / "greedy_7m_golden.npz"
SURE = 32  # up to here no gap between the two largest logits is small (test_gpu_model.py)


@pytest.fixture(scope="module")
def greedy():
    return np.load(GREEDY)


@pytest.fixture(scope="module")
def checkpoint(greedy, tmp_path_factory):
    p = tmp_path_factory.mktemp("ckpt") / "gpt-oss-7m-greedy.bin"
    binfmt.write_synthetic(str(p), binfmt.config_7m(), int(greedy["seed"]))
    return p


@pytest.mark.parametrize("drafter", ["none", "right", "some_wrong"])
@pytest.mark.parametrize("others", [0, 2])
def test_drafted_decoding_follows_one_token_decoding(greedy, checkpoint, drafter, others):
    """The reference's continuation from its first token on, alone and with other sequences in the step."""
    from gptoss_b200 import model
    cfg = binfmt.config_7m()
    m = model.Model(cfg, max_batch=64, max_seq=128)
    m.load_bin(checkpoint)
    prompt, want = greedy["prompt"].tolist(), greedy["generated"].tolist()
    truth = prompt + want

    def draft(history):
        n = len(history)
        right = truth[n:n + 5] if history == truth[:n] else []
        if drafter == "none":
            return [], []
        if drafter == "right":
            return right, list(range(-1, len(right) - 1))
        toks, pars, last = [], [], -1   # a wrong sibling before each right token
        for t in right:
            toks += [(t + 1) % cfg.vocab_size, t]
            pars += [last, last]
            last = len(toks) - 1
        return toks, pars

    out = m.generate_drafted([prompt] + [synth.uniform_ids(i, 9, 11 + i, cfg.vocab_size).tolist() for i in range(others)], SURE, draft)
    assert out[0].tolist() == want[:SURE]
    m.close()
