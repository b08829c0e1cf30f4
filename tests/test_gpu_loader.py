"""What a context sets up on the device is there before anything reads it: the
context's stream does not wait for the legacy default stream, nor the other
way round."""
import numpy as np
import pytest

from helpers import lcg_ids, mini_config, rdet, write_model

pytestmark = pytest.mark.gpu


def test_synthetic_scalars_behind_a_long_queue():
    # The embedding's generator (2 GB) is still running when the first layer's
    # scalar is generated and read back.  Generated values depend on their
    # index alone, so the rows of the first 97 tokens, and with them all layer
    # outputs, are those of the small model, whose scalars come from its file.
    over = dict(hidden_size=256, hidden_size_per_layer_input=None)
    small, big = mini_config(**over), mini_config(vocab_size=1 << 22, **over)
    for cfg in (small, big):
        cfg["text_config"] = {k: v for k, v in cfg["text_config"].items() if v is not None}
    ids = lcg_ids(9, 97, 5)
    m = rdet.Model.open(write_model(small, seed=31), max_prefill=16, layer_commitments=True)
    s = m.new_sequence(16)
    s.prefill(ids)
    want = [s.commitment(rdet.BUF_LAYER_OUTPUT, l) for l in range(m.L)]
    hidden = s.read(rdet.BUF_HIDDEN)
    for _ in range(3):
        b = rdet.Model.synthetic(big, seed=31, max_prefill=16, layer_commitments=True)
        t = b.new_sequence(16)
        t.prefill(ids)
        assert [t.commitment(rdet.BUF_LAYER_OUTPUT, l) for l in range(b.L)] == want
        assert np.array_equal(t.read(rdet.BUF_HIDDEN), hidden)
        b.close()
