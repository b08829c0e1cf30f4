"""A generation that fails half way (a selected token without a per-layer
embedding) leaves a sequence that has to be prefilled again: its position on
the device and its rows have moved, its position on the host has not."""
import numpy as np
import pytest

from helpers import mini_config, rdet

pytestmark = pytest.mark.gpu


def refused(code, call, *args):
    with pytest.raises(rdet.RdetError) as e:
        call(*args)
    assert e.value.code == code and e.value.msg


def test_a_failed_generation_asks_for_a_new_prefill():
    m = rdet.Model.synthetic(mini_config(vocab_size_per_layer_input=5, tie_word_embeddings=False), seed=4, width=16, max_prefill=16)
    s, r = m.new_sequence(43), m.new_sequence(43)
    for x in (s, r):
        x.prefill([1, 2, 3])
    rdet.tree_decode(m, [s], [[1, 2]], [[-1, 0]])
    assert s.generate(0) == []                      # nothing happens to the sequence or its tree
    assert rdet.tree_select(m, [s])[0]
    refused(-6, s.generate, 40)
    assert s.position == 3
    refused(-5, rdet.tree_accept, m, [s], [[0]])
    refused(-5, s.decode, 1)
    refused(-5, s.generate, 1)
    refused(-5, rdet.tree_decode, m, [s], [[1]], [[-1]])
    s.prefill([1, 2, 3])
    for x in (s, r):
        for _ in range(40):                         # to the end of its cache
            x.decode(2)
    assert np.array_equal(s.read(rdet.BUF_LOGITS), r.read(rdet.BUF_LOGITS))
    assert s.commitment(rdet.BUF_KV) == r.commitment(rdet.BUF_KV)


def test_counts_past_the_cache_are_refused():
    # counts of 2^31 and more are negative as an int, so they must not be compared as one
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=16)
    s = m.new_sequence(10)
    s.prefill([1, 2, 3])
    out = np.zeros(16, dtype=np.uint32)
    for n in (8, 1 << 31, (1 << 32) - 4, (1 << 32) - 1):
        assert rdet.lib().rdet_generate(m._h, s._h, n, out.ctypes.data) == -6
    assert s.position == 3 and len(s.generate(7)) == 7
