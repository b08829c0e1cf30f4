"""The output loop under masks that depend on the output, over a toy model on
the host: what the callback is asked, and that the output is that of one token
a step."""
import importlib

import numpy as np
import pytest

from helpers import rdet

drafted = importlib.import_module("raster-inference_b200.drafted")

V = 70
WORDS = (V + 31) // 32


def scores(text):
    """Logits after a text: any function of it that repeats itself now and then."""
    h = sum((k + 1) * t for k, t in enumerate(text[-3:])) * 2654435761 % 2**32
    return np.random.default_rng(h % 11).permutation(V)


def pick(text, mask):
    bits = np.unpackbits(np.ascontiguousarray(mask, np.uint32).view(np.uint8), bitorder="little")[:V]
    s = np.where(bits > 0, scores(text), -1)
    return int(np.argmax(s)) if bits.any() else rdet.NO_TOKEN


class Toy:
    """The calls of the loop on host lists."""
    max_prefill, max_ctx = 64, 10**6

    def __init__(self):
        self.V = V

    def install(self, monkeypatch):
        for name in ("select_rules", "tree_decode", "tree_select", "tree_accept"):
            monkeypatch.setattr(rdet, name, getattr(self, name))

    def select_rules(self, model, seqs, rules):
        return [pick(s.text, r["allow"]) for s, r in zip(seqs, rules)]

    def tree_decode(self, model, seqs, tokens, parents):
        for s, t, p in zip(seqs, tokens, parents):
            assert 1 <= len(t) == len(p) and all(-1 <= q < j for j, q in enumerate(p)) and p[0] == -1
            s.tree = (list(t), list(p))

    def tree_select(self, model, seqs, rules):
        out = []
        for s, r in zip(seqs, rules):
            tokens, parents = s.tree
            masks = np.asarray(r["allow"]).reshape(len(tokens), WORDS)
            paths = []
            for t, p in zip(tokens, parents):
                paths.append((paths[p] if p >= 0 else s.text) + [t])
            out.append([pick(p, m) for p, m in zip(paths, masks)])
        return out

    def tree_accept(self, model, seqs, paths):
        for s, p in zip(seqs, paths):
            s.text = s.text + [s.tree[0][j] for j in p]


class Seq:
    max_ctx = 10**6

    def __init__(self, text):
        self.text = list(text)

    @property
    def position(self):
        return len(self.text)

    def decode(self, t):
        self.text.append(t)


def grammar(limit, asked):
    """Two thirds of the tokens follow a token; raises when it is asked about an
    output that its own masks do not allow, or a complete one."""
    def bits(last):
        return np.array([(3 * t + 5 * last) % 7 < 4 for t in range(V)])

    def allow(output):
        assert len(output) < limit, "asked about a complete output"
        for a, b in zip([0] + output[:-1], output):
            if not bits(a)[b]:
                raise ValueError("not a prefix of the language")
        asked.append(list(output))
        m = np.zeros(WORDS * 32, np.uint8)
        m[:V] = bits(output[-1] if output else 0)
        return np.packbits(m, bitorder="little").view(np.uint32)
    return allow


class Wild:
    """Drafts that know nothing: forbidden tokens, a second root, ids past the vocabulary."""

    def __init__(self, tokens):
        self.rng = np.random.default_rng(len(tokens))

    def extend(self, tokens):
        pass

    def tree(self, root, nodes):
        par = [-1] + [int(self.rng.integers(-1, j)) for j in range(1, nodes)]
        return [root] + [int(t) for t in self.rng.integers(0, V + 9, nodes - 1)], par


@pytest.mark.parametrize("draft", [drafted.NgramDraft, Wild])
@pytest.mark.parametrize("nodes", [1, 4, 16, 64])
@pytest.mark.parametrize("nseq", [1, 3])
def test_the_callback_is_asked_about_admissible_outputs_alone(monkeypatch, draft, nodes, nseq):
    toy, n = Toy(), 60
    toy.install(monkeypatch)
    prompts = [[1 + k, 2, 3 + k, 2, 3] for k in range(nseq)]
    asked = [[] for _ in range(nseq)]
    rules = [dict(allow=grammar(n, a)) for a in asked]
    out = drafted.run_output_decode(toy, [Seq(p) for p in prompts], prompts, n, nodes=nodes, rules=rules, draft=draft)
    for p, o in zip(prompts, out):
        want, mask = [], grammar(n, [])
        while len(want) < n:
            want.append(pick(p + want, mask(want)))
        assert o == want


def test_admissible_nodes():
    none = np.zeros(WORDS, np.uint32)
    even = np.full(WORDS, 0x55555555, np.uint32)

    def allow(output):
        return none if output[-1] == 4 else even

    # 0: 7; children 4, 5 (odd), 8; 4 ends; behind 8: 6, 70 (no token); a second root
    tokens, parents = [7, 4, 5, 8, 2, 6, 70, 2, 9], [-1, 0, 0, 0, 1, 3, 3, -1, 2]
    (t, p), m = drafted._admissible(allow, [1], 10, V, tokens, parents)
    assert (t, p) == ([7, 4, 8, 6], [-1, 0, 0, 2])
    assert [x.tolist() for x in m] == [even.tolist(), none.tolist(), even.tolist(), even.tolist()]
    (t, p), m = drafted._admissible(allow, [1], 3, V, tokens, parents)
    assert (t, p) == ([7, 4, 8], [-1, 0, 0])        # the third token completes the output
    assert [x.tolist() for x in m[1:]] == [[0xFFFFFFFF] * WORDS] * 2


def test_a_mask_of_another_size_is_refused():
    for words in (WORDS - 1, WORDS + 1):
        with pytest.raises(ValueError):
            drafted._admissible(lambda output: np.ones(words, np.uint32), [1], 10, V, [7, 4], [-1, 0])
