"""A prompt whose workspaces find no memory: the call says so, and the handle's next prompts answer what they did before."""
import numpy as np
import pytest

import crane_b200
from crane_b200 import CraneB200Error, synth

pytestmark = pytest.mark.gpu
ROWS = 3_000_000          # x 4 bytes of the inner width below: more than a GPU has


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_a_prompt_that_finds_no_memory(kind):
    cfg = dict(synth.TINY_QWEN3, num_hidden_layers=1, intermediate_size=16384, max_position_embeddings=1 << 22)
    cfg = synth.fp8_config(cfg) if kind == "fp8" else cfg
    m = crane_b200.Qwen3Model(cfg, device=0, max_seq_len=ROWS + 64)
    m.load_checkpoint(synth.fp8_checkpoint(cfg) if kind == "fp8" else synth.synth_checkpoint(cfg))
    ids = synth.synth_token_ids(90, cfg["vocab_size"], "growth")

    def answers():
        m.clear_kv_cache()
        return [m.forward_step(ids[:20], 0), m.forward_step([3], 20)]
    want = answers()
    for _ in range(2):
        m.clear_kv_cache()
        with pytest.raises(CraneB200Error) as e:
            m.forward_step(np.resize(ids, ROWS), 0)
        assert e.value.code == crane_b200.OOM
        for a, b in zip(want, answers()):
            assert np.array_equal(a, b)
    m.clear_kv_cache()
    assert np.isfinite(m.forward_step(ids, 0)).all()
    m.close()
