"""Calls that are refused for want of device memory leave everything else as
it was."""
import numpy as np
import pytest

from helpers import mini_config, rdet

pytestmark = pytest.mark.gpu

RDET_E_OOM = -7


def test_a_refused_sequence_leaves_the_context_usable():
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=16)
    a, b = m.new_sequence(16), m.new_sequence(16)
    for s in (a, b):
        s.prefill([1, 2, 3])
    with pytest.raises(rdet.RdetError) as e:
        m.new_sequence(2_000_000_000)  # 256 GB of keys in the first layer
    assert e.value.code == RDET_E_OOM
    a.decode(5)
    b.decode(5)
    assert np.array_equal(a.read(rdet.BUF_LOGITS), b.read(rdet.BUF_LOGITS))
    with pytest.raises(rdet.RdetError):
        m.new_sequence(2_000_000_000)
    rdet.decode_batch(m, [a, b], [6, 6])
    assert a.select() == b.select()
