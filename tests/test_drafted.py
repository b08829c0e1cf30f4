"""The drafts and the walk of greedy decode through a drafted tree, and what
the wrappers refuse before they reach the library (no GPU)."""
import importlib

import numpy as np
import pytest

from helpers import rdet

drafted = importlib.import_module("raster-inference_b200.drafted")


def paths(tokens, parents):
    out = []
    for t, p in zip(tokens, parents):
        out.append((out[p] if p >= 0 else []) + [t])
    return out


@pytest.mark.parametrize("nodes", [1, 2, 5, 16, 64])
def test_ngram_trees_are_text_that_followed(nodes):
    rng = np.random.default_rng(nodes)
    text = [int(t) for t in rng.integers(0, 4, 200)]
    d = drafted.NgramDraft(text[:150])
    d.extend(text[150:])
    assert d.tokens == text
    for root in range(4):
        tokens, parents = d.tree(root, nodes)
        assert 1 <= len(tokens) <= nodes and tokens[0] == root and parents[0] == -1
        assert all(0 <= p < j for j, p in enumerate(parents) if j)
        all_paths = paths(tokens, parents)
        assert len({tuple(p) for p in all_paths}) == len(tokens)  # no node twice
        joined = ",".join(map(str, text + [root])) + ","
        for p in all_paths:
            assert ",".join(map(str, p)) + "," in joined


def test_ngram_tree_prefers_the_longest_and_latest():
    d = drafted.NgramDraft([1, 2, 3, 9, 2, 3, 8, 1, 2])
    tokens, parents = d.tree(3, 4)
    assert (tokens, parents) == ([3, 9, 2, 3], [-1, 0, 1, 2])   # behind 1 2 3
    assert drafted.NgramDraft([]).tree(7, 8) == ([7], [-1])
    assert drafted.NgramDraft([7, 7]).tree(7, 8)[0] == [7, 7, 7]
    assert drafted.NgramDraft([1, 2]).tree(9, 8) == ([9], [-1])  # never seen


def test_accepted_path():
    tokens, parents = [1, 2, 3, 5], [-1, 0, 0, 2]
    assert drafted.accepted_path(tokens, parents, [3, 0, 5, 9], 4) == [0, 2, 3]
    assert drafted.accepted_path(tokens, parents, [3, 0, 5, 9], 2) == [0, 2]
    assert drafted.accepted_path(tokens, parents, [4, 0, 5, 9], 4) == [0]
    assert drafted.accepted_path([1], [-1], [rdet.NO_TOKEN], 4) == [0]


def test_wrappers_refuse():
    class M:
        V, _h, max_prefill = 97, None, 8
    with pytest.raises(ValueError):
        rdet.tree_decode(M, [], [[1]], [[-1]])
    with pytest.raises(ValueError):
        rdet.tree_accept(M, [], [[1]])
    with pytest.raises(ValueError):
        rdet.select_rules(M, [], [{}])
    with pytest.raises(ValueError):
        rdet._rules(M, [dict(allow=[1, 2, 3])], [1])
    with pytest.raises(TypeError):
        rdet._rules(M, [dict(temperature=1)], [1])
    with pytest.raises(ValueError):
        drafted.run_output_decode(M, [], [], 4, nodes=65)
    with pytest.raises(ValueError):
        drafted.run_output_decode(M, [], [[1]], 4)
    assert drafted.run_output_decode(M, [], [], 0) == []


@pytest.mark.parametrize("name,args", [
    ("rdet_select_rules", (None, None, 1, None, None)), ("rdet_tree_decode", (None, None, 1, None, None, None)),
    ("rdet_tree_select", (None, None, 1, None, None)), ("rdet_tree_accept", (None, None, 1, None, None))])
def test_null_arguments(name, args):
    assert getattr(rdet.lib(), name)(*args) == -1
