"""Adapters that nothing was loaded into are zero from the first step on."""
import numpy as np
import pytest

from gptoss_b200 import binfmt, synth

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n_adapters,rank", [(3, 8), (8192, 128)])  # the second: arrays that take a while to clear
def test_unloaded_adapters_change_nothing(tmp_path, n_adapters, rank):
    """Room for adapters, rows bound to them, a step at once: the bits of the model without adapters, in every row."""
    from gptoss_b200 import model
    cfg, B = binfmt.config_7m(), 24
    ckpt = tmp_path / "7m.bin"
    binfmt.write_synthetic(str(ckpt), cfg, 3)
    plain = model.Model(cfg, max_batch=B, max_seq=16)
    plain.load_bin(ckpt)
    ids = synth.uniform_ids(4, 5, 3 * B, cfg.vocab_size).reshape(3, B).astype(np.int32)
    want = []
    for pos in range(3):
        plain.step(ids[pos], pos)
        want.append([plain.logits(row) for row in range(B)])
    plain.close()
    m = model.Model(cfg, max_batch=B, max_seq=16)
    m.load_bin(ckpt)
    # what the arrays will be made of has held something else: NaN in every type
    junk = torch.full((1 << 30,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    del junk
    torch.cuda.empty_cache()
    m.lora_create(n_adapters, rank)
    for row in range(0, B, 2):
        m.lora_bind(row, (row * 977) % n_adapters)
    for pos in range(3):
        m.step(ids[pos], pos)
        for row in range(B):
            assert np.array_equal(m.logits(row), want[pos][row]), (pos, row)
    m.close()
