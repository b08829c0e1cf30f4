"""Calls that are refused for want of device memory leave everything else as
it was."""
import numpy as np
import pytest

from helpers import mini_config, rdet

torch = pytest.importorskip("torch")
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


def test_a_refused_tree_decode_keeps_the_trees_before_it():
    # 8192 rows of 4 million logits: the batch tables take 137 GB, and the trees'
    # rows, as large again, are not to be had
    cfg = mini_config(vocab_size=1 << 22, hidden_size_per_layer_input=None)
    cfg["text_config"] = {k: v for k, v in cfg["text_config"].items() if v is not None}
    m = rdet.Model.synthetic(cfg, seed=4, width=16, max_prefill=8192)
    a, r = m.new_sequence(12), m.new_sequence(12)
    for s in (a, r):
        s.prefill([1, 2, 3])
    rdet.tree_decode(m, [a], [[5, 6, 7]], [[-1, 0, 0]])
    many = [m.new_sequence(68) for _ in range(128)]
    for s in many:
        s.prefill([1])
    for _ in range(2):
        with pytest.raises(rdet.RdetError) as e:
            rdet.tree_decode(m, many, [[1] * 64] * 128, [[-1] * 64] * 128)
        assert e.value.code == RDET_E_OOM
    picked = rdet.tree_select(m, [a])
    rdet.tree_accept(m, [a], [[0, 2]])
    for t, p in ((5, picked[0][0]), (7, picked[0][2])):
        r.decode(t)
        assert r.select() == p
    assert np.array_equal(a.read(rdet.BUF_LOGITS), r.read(rdet.BUF_LOGITS))
    for l in range(m.L):
        assert a.commitment(rdet.BUF_LAYER_OUTPUT, l) == r.commitment(rdet.BUF_LAYER_OUTPUT, l)
    assert a.commitment(rdet.BUF_KV) == r.commitment(rdet.BUF_KV)
    rdet.tree_decode(m, [a], [[5, 6]], [[-1, 0]])  # and the context goes on
    assert rdet.tree_select(m, [a])[0]
    m.close()


def test_growing_trees_and_rules_keep_no_superseded_buffers():
    # every call needs more rows than any before it; a row of a million logits is
    # 4 MB in the batch tables and 4 MB among the trees' outputs
    vocab, nseq = 1 << 20, 8
    cfg = mini_config(vocab_size=vocab, hidden_size_per_layer_input=None)
    cfg["text_config"] = {k: v for k, v in cfg["text_config"].items() if v is not None}
    m = rdet.Model.synthetic(cfg, seed=4, width=16, max_prefill=512)
    seqs = [m.new_sequence(600) for _ in range(nseq)]
    ref = m.new_sequence(600)
    for s in (*seqs, ref):
        s.prefill([1, 2, 3])
    rdet.tree_decode(m, seqs, [[1]] * nseq, [[-1]] * nseq)  # loads the kernels
    rdet.tree_select(m, seqs, [dict(history=[1])] * nseq)
    torch.cuda.synchronize()
    before, rows, at = torch.cuda.mem_get_info()[0], 0, 3
    for n in range(9, 26):
        rdet.tree_decode(m, seqs, [[(7 * n + j) % vocab for j in range(n)]] * nseq, [list(range(-1, n - 1))] * nseq)
        picked = rdet.tree_select(m, seqs, [dict(history=list(range(40 * n)))] * nseq)
        assert all(p == picked[0] for p in picked)
        rdet.tree_accept(m, seqs, [[0, 1]] * nseq)
        for j in range(2):
            ref.decode((7 * n + j) % vocab)
        rows = n * nseq
    used = before - torch.cuda.mem_get_info()[0]
    assert used <= 2 * rows * 2 * (vocab + 4096) * 4 + (256 << 20), used
    for s in seqs:
        assert np.array_equal(s.read(rdet.BUF_LOGITS), ref.read(rdet.BUF_LOGITS))
        assert s.commitment(rdet.BUF_KV) == ref.commitment(rdet.BUF_KV)
    m.close()
