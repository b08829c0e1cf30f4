"""Drafted decoding end to end: what a tree decode selects and what an
accepted path leaves (tokens, logits, layer outputs, caches, commitments) equal
decoding the same tokens one by one.  All arithmetic is exact: no tolerance."""
import importlib

import numpy as np
import pytest

import draft_ref as R
from helpers import lcg_ids, mini_config, rdet, write_model
from test_gpu_models import VARIANTS

drafted = importlib.import_module("raster-inference_b200.drafted")
pytestmark = pytest.mark.gpu

# (tokens' ranks among the greedy choices are irrelevant: any tokens are a draft)
PARENTS = [-1, -1, 1, 0, 2, 2, 3, 5, 7, 4]   # two roots; 1-2-5-7-8 is a path that skips nodes


def state_of(seq, layers):
    return dict(pos=seq.position, logits=seq.read(rdet.BUF_LOGITS).tolist(), kv=seq.commitment(rdet.BUF_KV),
                hidden=seq.commitment(rdet.BUF_HIDDEN),
                layers=[seq.commitment(rdet.BUF_LAYER_OUTPUT, l) for l in range(layers)])


def argmax(row):
    return int(np.argmax(row))


def check_tree(cfg, width, n_prompt, parents, path, seed, extra=(), **opts):
    """One sequence's tree (with other sequences `extra` = (prompt, parents, path)
    beside it) against sequences that decode the nodes one by one."""
    cfg = {"text_config": {k: v for k, v in cfg["text_config"].items() if v is not None}}
    vocab = cfg["text_config"]["vocab_size"]
    jobs = [(n_prompt, parents, path), *extra]
    longest = max(n for n, _, _ in jobs)
    m = rdet.Model.synthetic(cfg, seed=seed, width=width, max_prefill=max(longest, sum(len(p) for _, p, _ in jobs)),
                             layer_commitments=True, **opts)
    trees, tokens = [], []
    for i, (n, par, _) in enumerate(jobs):
        s = m.new_sequence(n + len(par) + 4)
        s.prefill(lcg_ids(n, vocab, seed + i))
        trees.append(s)
        tokens.append([int(t) for t in lcg_ids(len(par), vocab, seed + 50 + i)])
    before = [state_of(s, m.L) for s in trees]
    rdet.tree_decode(m, trees, tokens, [p for _, p, _ in jobs])
    assert [state_of(s, m.L) for s in trees] == before  # nothing moves until a path is accepted
    picked = rdet.tree_select(m, trees)
    rdet.tree_accept(m, trees, [pa for _, _, pa in jobs])
    for i, (n, par, pa) in enumerate(jobs):
        leaves = [j for j in range(len(par)) if j not in par]
        ref_state = None
        for leaf in {*leaves, *(pa[-1:])}:
            ref = m.new_sequence(n + len(par) + 4)
            ref.prefill(lcg_ids(n, vocab, seed + i))
            chain = R.path_of(par, leaf)
            for j in chain:
                ref.decode(tokens[i][j])
                assert picked[i][j] == ref.select() == argmax(ref.read(rdet.BUF_LOGITS)), (i, j)
            if pa and leaf == pa[-1]:
                assert chain == pa
                ref_state = state_of(ref, m.L)
                for _ in range(3):  # and the sequences go on alike
                    t = ref.select()
                    ref.decode(t)
                keep = ref
        if pa:
            assert state_of(trees[i], m.L) == ref_state, i
            for _ in range(3):
                trees[i].decode(trees[i].select())
            assert state_of(trees[i], m.L) == state_of(keep, m.L), i
        else:
            assert state_of(trees[i], m.L) == before[i], i


@pytest.mark.parametrize("variant", sorted(VARIANTS))
def test_tree_equals_stepwise_decode(variant):
    cfg, width = VARIANTS[variant]
    check_tree(cfg, width, 21, PARENTS, [1, 2, 5, 7, 8], seed=61)


@pytest.mark.parametrize("n_prompt,parents,path", [
    (1, [-1], [0]),                       # one token behind one token
    (1, [-1], []),                        # nothing accepted
    (8, [-1, 0, 1, 2], [0, 1, 2, 3]),     # a chain whose rows are in place; the window's edge
    (7, [-1] * 12, [11]),                 # only roots
    (9, PARENTS, [0, 3, 6]),
    (5, list(range(-1, 63)), list(range(40))),  # the deepest tree, cut short
])
def test_tree_shapes(n_prompt, parents, path):
    check_tree(mini_config(), 16, n_prompt, parents, path, seed=71)


def test_ragged_batch_of_trees():
    rng = np.random.default_rng(5)
    extra = []
    for i in range(36):  # more sequences than one attention launch takes
        n = 1 + int(rng.integers(0, 17))
        par = [int(rng.integers(-1, j)) if j else -1 for j in range(n)]
        leaf = int(rng.integers(0, n))
        extra.append((1 + int(rng.integers(0, 30)), par, R.path_of(par, leaf) if i % 5 else []))
    check_tree(mini_config(), 16, 21, PARENTS, [1, 2, 5, 7, 8], seed=81, extra=extra)


def test_without_tensor_cores():
    check_tree(mini_config(), 16, 21, PARENTS, [1, 2, 5, 7, 8], seed=91, extra=[(3, [-1, 0, 0], [0, 2])],
               tensor_cores=False)


def test_wide_heads_and_window_over_several_tiles():
    cfg = mini_config(hidden_size=256, intermediate_size=512, num_attention_heads=8, num_key_value_heads=2,
                      head_dim=256, global_head_dim=512, sliding_window=512, hidden_size_per_layer_input=32,
                      num_hidden_layers=4, num_kv_shared_layers=1, vocab_size=300,
                      layer_types=["sliding_attention", "full_attention", "sliding_attention", "sliding_attention"])
    check_tree(cfg, 16, 640, PARENTS, [1, 2, 5, 7, 8], seed=101, extra=[(200, [-1, 0, 0, 1], [0, 1, 3])])


# ---- the output loop ------------------------------------------------------------------
def greedy_loop(m, ids, n, rules=None):
    """One token at a time through the entry points that were there."""
    s = m.new_sequence(len(ids) + n + 70)
    s.prefill(ids)
    out = []
    for _ in range(n):
        if rules is None:
            t = s.select()
        else:
            t = reference_token(m, s.read(rdet.BUF_LOGITS), list(ids) + out, rules, out)
        if t == rdet.NO_TOKEN:
            break
        out.append(t)
        s.decode(t)
    return out, s


def reference_token(m, logits, text, rules, out):
    counts = {}
    for t in text:
        counts[t] = counts.get(t, 0) + 1
    mask = rules["allow"](out) if "allow" in rules else None
    allow = None if mask is None else np.unpackbits(mask.view(np.uint8), bitorder="little")[:m.V].astype(bool)
    return R.rules_row(logits, counts, rules.get("repetition", 1 << 16), rules.get("frequency", 0),
                       rules.get("presence", 0), list(rules.get("bias", {}).items()), allow)[1]


@pytest.mark.parametrize("nodes", [1, 5, 16])
def test_output_equals_greedy(nodes):
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=48, 
                             layer_commitments=True)  # several chunks of sequences
    prompts = [[int(t) for t in lcg_ids(n, 97, n)] for n in (1, 10, 23, 12, 5)]
    prompts[2] = prompts[2][:6] * 4  # repeats itself
    seqs = [m.new_sequence(len(p) + 110) for p in prompts]
    for s, p in zip(seqs, prompts):
        s.prefill(p)
    stats = {}
    out = drafted.run_output_decode(m, seqs, prompts, 40, nodes=nodes, stats=stats)
    for s, p, o in zip(seqs, prompts, out):
        ref, r = greedy_loop(m, p, 40)
        assert o == ref == m_generate(m, p, 40)
        assert state_of(s, m.L) == state_of(r, m.L)
    assert stats["passes"] >= 1


def m_generate(m, ids, n):
    s = m.new_sequence(len(ids) + n)
    s.prefill(ids)
    return s.generate(n)


def test_right_drafts_save_passes():
    """A draft that knows the output: every step takes a whole tree."""
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=48, layer_commitments=True)
    ids = [int(t) for t in lcg_ids(10, 97, 4)]
    ref = m_generate(m, ids, 33)

    class Known:
        def __init__(self, tokens):
            self.at = 0

        def extend(self, tokens):
            self.at += len(tokens)

        def tree(self, root, nodes):
            assert root == ref[self.at]
            part = ref[self.at:self.at + nodes]
            return part, list(range(-1, len(part) - 1))

    s = m.new_sequence(len(ids) + 50)
    s.prefill(ids)
    stats = {}
    assert drafted.run_output_decode(m, [s], [ids], 33, nodes=11, draft=Known, stats=stats) == [ref]
    assert stats["passes"] == 3


def test_output_under_rules_equals_stepwise_reference():
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=64, layer_commitments=True)
    words = (97 + 31) // 32

    def odd_even(output):  # what is allowed changes with the position
        bits = np.zeros(words * 32, dtype=np.uint8)
        bits[len(output) % 2:97:2] = 1
        return np.packbits(bits, bitorder="little").view(np.uint32)

    def three_only(output):  # ends after three tokens
        bits = np.zeros(words * 32, dtype=np.uint8)
        if len(output) < 3:
            bits[:97] = 1
        return np.packbits(bits, bitorder="little").view(np.uint32)

    rules = [dict(repetition=90000, frequency=3000, presence=9000, bias={5: 1 << 15, 96: -(1 << 20), 7: 70000}),
             dict(allow=odd_even, repetition=70000), dict(), dict(allow=three_only, bias={3: 1 << 21})]
    prompts = [[int(t) for t in lcg_ids(n, 97, n)] for n in (10, 14, 6, 9)]
    seqs = [m.new_sequence(len(p) + 60) for p in prompts]
    for s, p in zip(seqs, prompts):
        s.prefill(p)
    out = drafted.run_output_decode(m, seqs, prompts, 24, nodes=12, rules=rules)
    for s, p, o, r in zip(seqs, prompts, out, rules):
        ref, rs = greedy_loop(m, p, 24, r)
        assert o == ref
        assert state_of(s, m.L) == state_of(rs, m.L)
    assert len(out[3]) == 3 and len(out[0]) == 24


@pytest.mark.parametrize("nodes", [1, 8])
def test_one_sequence_under_rules(nodes):
    # alone and without a draft it decodes one token at a time
    m = rdet.Model.synthetic(mini_config(), seed=6, width=16, max_prefill=32, layer_commitments=True)
    words = (97 + 31) // 32

    def low(output):
        bits = np.zeros(words * 32, dtype=np.uint8)
        bits[:40 + len(output)] = 1
        return np.packbits(bits, bitorder="little").view(np.uint32)

    rules = dict(repetition=80000, presence=4000, bias={2: 1 << 14}, allow=low)
    ids = [int(t) for t in lcg_ids(9, 97, 9)]
    s = m.new_sequence(60)
    s.prefill(ids)
    stats = {}
    out = drafted.run_output_decode(m, [s], [ids], 20, nodes=nodes, rules=[rules], stats=stats)[0]
    ref, r = greedy_loop(m, ids, 20, rules)
    assert out == ref and state_of(s, m.L) == state_of(r, m.L)
    assert nodes > 1 or stats["passes"] == 20


def test_select_without_rules_and_empty_lists():
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=16)
    s = m.new_sequence(20)
    s.prefill([1, 2, 3])
    assert rdet.select_rules(m, [s], None) == rdet.select_rules(m, [s], [{}]) == [s.select()]
    assert rdet.select_rules(m, [], None) == []
    rdet.tree_decode(m, [], [], [])
    assert rdet.tree_select(m, []) == []
    rdet.tree_accept(m, [], [])


# ---- refusals -------------------------------------------------------------------------
def refused(code, call, *args, **kw):
    with pytest.raises(rdet.RdetError) as e:
        call(*args, **kw)
    assert e.value.code == code and e.value.msg


def test_refusals_leave_the_sequence_as_it_is():
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=8, layer_commitments=True)
    other = rdet.Model.synthetic(mini_config(), seed=5, width=16, max_prefill=8)
    s, fresh, foreign = m.new_sequence(12), m.new_sequence(12), other.new_sequence(12)
    foreign.prefill([1])
    s.prefill([1, 2, 3])
    before = state_of(s, m.L)
    ok = ([5, 6, 7], [-1, 0, 0])
    refused(-5, rdet.tree_decode, m, [fresh], [[1]], [[-1]])             # no prefill
    refused(-1, rdet.tree_decode, m, [foreign], [[1]], [[-1]])
    refused(-1, rdet.tree_decode, m, [s, s], [[1]] * 2, [[-1]] * 2)
    refused(-6, rdet.tree_decode, m, [s], [[]], [[]])
    refused(-6, rdet.tree_decode, m, [s], [[1] * 9], [[-1] * 9])         # above max_prefill
    refused(-6, rdet.tree_decode, m, [s], [[1] * 10], [[-1] * 10])       # above the cache
    refused(-6, rdet.tree_decode, m, [s], [[97]], [[-1]])                # not a token
    refused(-1, rdet.tree_decode, m, [s], [[1, 2]], [[-1, 1]])
    refused(-1, rdet.tree_decode, m, [s], [[1, 2]], [[-1, -2]])
    refused(-5, rdet.tree_select, m, [s])                                # no tree
    refused(-5, rdet.tree_accept, m, [s], [[]])
    rdet.tree_decode(m, [s], [ok[0]], [ok[1]])
    refused(-1, rdet.tree_accept, m, [s], [[1]])                         # not a root
    refused(-1, rdet.tree_accept, m, [s], [[0, 1, 2]])                   # 2 does not follow 1
    refused(-1, rdet.tree_accept, m, [s], [[0, 3]])
    refused(-1, rdet.tree_accept, m, [s, s], [[0], [0]])
    refused(-1, rdet.tree_select, m, [s], [dict(repetition=0)])
    assert state_of(s, m.L) == before
    rdet.tree_accept(m, [s], [[0, 2]])
    assert s.position == 5
    refused(-5, rdet.tree_accept, m, [s], [[]])                          # accepted once
    rdet.tree_decode(m, [s], [ok[0]], [ok[1]])
    s.decode(4)
    refused(-5, rdet.tree_select, m, [s])                                # a decode dropped it
    rdet.tree_decode(m, [s], [ok[0]], [ok[1]])
    s.decode_begin(4)
    refused(-5, rdet.tree_accept, m, [s], [[0]])
    refused(-5, rdet.tree_decode, m, [s], [ok[0]], [ok[1]])              # a decode is in flight
    s.decode_range(0, m.L)
    s.decode_finalize()
    t = m.new_sequence(12)
    t.prefill([1, 2])
    rdet.tree_decode(m, [s], [ok[0]], [ok[1]])
    rdet.tree_decode(m, [t], [ok[0]], [ok[1]])                           # a later tree decode drops it
    refused(-5, rdet.tree_select, m, [s])
    t.prefill([1, 2])
    refused(-5, rdet.tree_select, m, [t])
    refused(-5, rdet.select_rules, m, [fresh], [{}])


def test_a_refused_call_keeps_the_tree():
    m = rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=8, layer_commitments=True)
    s, r = m.new_sequence(12), m.new_sequence(12)
    for x in (s, r):
        x.prefill([1, 2, 3])
    rdet.tree_decode(m, [s], [[5, 6, 7]], [[-1, 0, 0]])
    refused(-6, rdet.tree_decode, m, [s], [[97]], [[-1]])
    rdet.tree_accept(m, [s], [[0, 2]])
    r.decode(5)
    r.decode(7)
    assert state_of(s, m.L) == state_of(r, m.L)
