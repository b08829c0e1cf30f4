"""Arguments that the draft-verification entry points refuse.  Every check
runs on the host before anything is launched, so no GPU is needed and the
addresses stand for device memory that nothing reads."""
import pytest

from helpers import rdet

A = 1 << 20  # an address nothing reads


def seq(**over):
    s = dict(k_cache=A, v_cache=A, k_tree=A, v_tree=A, cap=64, context=8, tree_cap=16, parents=[-1, 0, 0])
    s.update(over)
    return s


def tree(s, heads=4, kv=2, d=16, window=0, q=A, out=A, ws=A, ws_bytes=1 << 40, n=1):
    rdet.det_attention_tree(rdet.tree_seqs([s] * n), q, heads, kv, d, window, out, ws, ws_bytes)


@pytest.mark.parametrize("over,code", [
    (dict(parents=[]), -6), (dict(parents=[-1] * 65, tree_cap=65), -6), (dict(parents=[-1, 1]), -1),
    (dict(parents=[-2]), -1), (dict(context=65), -6), (dict(tree_cap=2), -6), (dict(k_tree=0), -1),
    (dict(v_cache=0), -1), (dict(context=1 << 24, cap=1 << 25), -6), (dict(context=523262, cap=1 << 20), -6)])
def test_tree_refuses_sequences(over, code):
    with pytest.raises(rdet.RdetError) as e:
        tree(seq(**over))
    assert e.value.code == code and e.value.msg


@pytest.mark.parametrize("over,code", [
    (dict(heads=3), -1), (dict(kv=0), -1), (dict(d=0), -6), (dict(d=513), -6), (dict(q=0), -1), (dict(out=0), -1),
    (dict(ws=0), -1), (dict(ws=A + 8), -1), (dict(ws_bytes=16), -6), (dict(heads=2048), -6)])
def test_tree_refuses_shapes(over, code):
    with pytest.raises(rdet.RdetError) as e:
        tree(seq(), **over)
    assert e.value.code == code and e.value.msg


def test_tree_workspace_grows_with_the_work():
    def need(**over):
        return rdet.det_attention_tree_workspace(rdet.tree_seqs([seq(**over)]), 4, 2, 16, over.pop("window", 0))
    assert 0 < need() < need(cap=4096, context=4000)
    assert rdet.det_attention_tree_workspace(rdet.tree_seqs([]), 4, 2, 16, 0) == 0


def row(**over):
    r = dict(logits=A)
    r.update(over)
    return r


@pytest.mark.parametrize("rows,vocab,code", [
    ([row(logits=0)], 32, -1), ([row(history_len=3)], 32, -1), ([row(n_bias=1, bias_ids=A)], 32, -1),
    ([row(repetition=0)], 32, -1), ([row(repetition=-5)], 32, -1), ([row(parent=0)], 32, -1),
    ([row(), row(parent=1)], 32, -1), ([row(parent=-2)], 32, -1), ([row()], 0, -6), ([row()], (1 << 30) + 1, -6),
    ([row()] + [row()] * 192 + [row(parent=0)], 32, -6)])
def test_rules_refuse(rows, vocab, code):
    with pytest.raises(rdet.RdetError) as e:
        rdet.det_logits_rules(rdet.logit_rows(rows), vocab, A)
    assert e.value.code == code and e.value.msg


def test_rules_refuse_null_tokens():
    with pytest.raises(rdet.RdetError) as e:
        rdet.det_logits_rules(rdet.logit_rows([row()]), 32, 0)
    assert e.value.code == -1


def move(**over):
    m = dict(cache=A, draft=A, cap=32, draft_cap=8, kv_heads=2, head_dim=16, context=10, path=0)
    m.update(over)
    return m


@pytest.mark.parametrize("over,paths,code", [
    (dict(cache=0), [[0, 1]], -1), (dict(draft=0), [[0, 1]], -1), (dict(path=1), [[0, 1]], -1),
    (dict(), [[1, 1]], -1), (dict(), [[2, 1]], -1), (dict(), [[0, 64]], -1), (dict(), [[0, 8]], -6),
    (dict(context=31), [[0, 1]], -6), (dict(context=0xffffffff), [[0, 1]], -6), (dict(kv_heads=0), [[0]], -6),
    (dict(head_dim=0), [[0]], -6), (dict(head_dim=1025), [[0]], -6)])
def test_commit_refuses(over, paths, code):
    with pytest.raises(rdet.RdetError) as e:
        rdet.det_tree_commit(rdet.tree_moves([move(**over)], paths))
    assert e.value.code == code and e.value.msg


def test_descriptor_layouts():
    import ctypes as C
    assert (C.sizeof(rdet.TreeSeq), C.sizeof(rdet.LogitRow), C.sizeof(rdet.TreeMove)) == (56, 80, 40)
