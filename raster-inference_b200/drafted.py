"""Greedy output decode with drafted tokens.

Deterministic decode is exact: the token after a prefix, its logits and its
K/V rows are one fixed sequence of bits.  So several guessed tokens can be
checked in one pass over the weights (tree_decode), and the accepted ones leave
the sequence exactly as decoding them one at a time does: same tokens, caches,
logits and commitments.  The guesses come from the sequence's own text
(NgramDraft); any other source of token trees works with the same loop.
"""
from __future__ import annotations

import importlib

import numpy as np

rdet = importlib.import_module(__package__)


class NgramDraft:
    """Drafts from earlier occurrences of a sequence's last tokens.

    Every n-gram of 1 to `longest` tokens remembers where it ended; the text
    behind the latest occurrences of the last tokens, longest n-gram first,
    fills the tree."""

    def __init__(self, tokens, longest: int = 3, occurrences: int = 4):
        self.longest, self.occurrences = longest, occurrences
        self.tokens: list[int] = []
        self.ends: dict[tuple, list[int]] = {}
        self.extend(tokens)

    def extend(self, tokens):
        for t in tokens:
            # an n-gram is entered once it has a successor
            for n in range(1, min(self.longest, len(self.tokens)) + 1):
                self.ends.setdefault(tuple(self.tokens[-n:]), []).append(len(self.tokens))
            self.tokens.append(int(t))

    def tree(self, root: int, nodes: int):
        """(tokens, parents) of at most `nodes` nodes; node 0 is `root`, the
        token that follows the text."""
        text = self.tokens + [int(root)]
        tokens, parents = [int(root)], [-1]
        children: dict[tuple, int] = {}
        for n in range(min(self.longest, len(text)), 0, -1):
            gram = tuple(text[-n:])
            for end in reversed(self.ends.get(gram, [])[-self.occurrences:]):
                at = 0
                for t in text[end:end + nodes]:
                    node = children.get((at, t))
                    if node is None:
                        if len(tokens) >= nodes:
                            return tokens, parents
                        node = children[(at, t)] = len(tokens)
                        tokens.append(t)
                        parents.append(at)
                    at = node
        return tokens, parents


def accepted_path(tokens, parents, selected, limit: int):
    """The nodes, from node 0 on, that greedy decode takes: behind a node comes
    the child that holds the token selected after it.  At most `limit` nodes."""
    path = [0]
    while len(path) < limit:
        nxt = [j for j in range(path[-1] + 1, len(tokens))
               if parents[j] == path[-1] and tokens[j] == selected[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


def _rules_of(rules, text, allow):
    if rules is None:
        return None
    out = {k: v for k, v in rules.items() if k != "allow"}
    out["history"] = text
    if allow is not None:
        out["allow"] = np.stack(allow)
    return out


def run_output_decode(model, seqs, prompts, max_new_tokens: int, nodes: int = 16, rules=None, draft=NgramDraft,
                      stats=None) -> list[list[int]]:
    """The greedy tokens of every prefilled sequence, as
    rdet.run_output_decode gives them one sequence at a time, with up to
    `nodes` drafted tokens per sequence and step.  It drafts whenever the draft
    offers a tree and does not measure what is accepted: drafts that are never
    right cost a lone sequence up to twice the time of one token a step (E4B
    shape, 128 tokens: 0.96 s against 0.48; without a draft to offer 0.49).

    prompts[i] are the tokens behind sequence i's cache.  rules[i] (or None for
    all): bias, repetition, frequency and presence as rdet.select_rules takes
    them, the prompt and the output being the history, and allow, a function
    from the output so far to the mask of the next token.  It is asked about
    outputs shorter than max_new_tokens whose every token its own masks allow,
    and about no others, as in a loop of one token a step: drafted nodes that a
    mask forbids are dropped.  A sequence ends early where its mask allows no
    token.  stats, a dict, receives the number of passes over the weights."""
    if not 1 <= nodes <= rdet.MAX_TREE_NODES:
        raise ValueError(f"nodes: 1 to {rdet.MAX_TREE_NODES}")
    if len(prompts) != len(seqs) or (rules is not None and len(rules) != len(seqs)):
        raise ValueError("one prompt, and one dict of rules, per sequence")
    drafts = [draft(p) for p in prompts]
    out: list[list[int]] = [[] for _ in seqs]
    text = [list(p) for p in prompts]
    if max_new_tokens <= 0:
        return out
    allow = [None if rules is None else r.get("allow") for r in (rules or [{}] * len(seqs))]
    first = rdet.select_batch(model, seqs) if rules is None else rdet.select_rules(
        model, seqs, [_rules_of(r, t, a and [a([])]) for r, t, a in zip(rules, text, allow)])
    nxt = list(first)
    chunk = max(1, model.max_prefill // nodes)  # sequences of one pass
    while True:
        live = [i for i in range(len(seqs)) if len(out[i]) < max_new_tokens and nxt[i] != rdet.NO_TOKEN]
        if not live:
            return out
        for at in range(0, len(live), chunk):
            part = live[at:at + chunk]
            s = [seqs[i] for i in part]
            trees = [drafts[i].tree(nxt[i], min(nodes if len(out[i]) + 1 < max_new_tokens else 1, model.max_prefill,
                                                seqs[i].max_ctx - seqs[i].position)) for i in part]
            masks = [None] * len(part)
            for k, i in enumerate(part):
                if allow[i]:
                    trees[k], masks[k] = _admissible(allow[i], out[i], max_new_tokens, model.V, *trees[k])
            if stats is not None:
                stats["passes"] = stats.get("passes", 0) + 1
            if len(part) == 1 and len(trees[0][0]) == 1:
                # nothing drafted: the one-token decode (4.0 ms against 7.2 of a
                # tree's batched pass, E4B shape at context 4096)
                i = part[0]
                seqs[i].decode(nxt[i])
                for t in (out[i], text[i]):
                    t.append(nxt[i])
                drafts[i].extend([nxt[i]])
                if len(out[i]) < max_new_tokens:
                    nxt[i] = seqs[i].select() if rules is None else rdet.select_rules(
                        model, s, [_rules_of(rules[i], text[i], masks[0])])[0]
                continue
            rdet.tree_decode(model, s, [t for t, _ in trees], [p for _, p in trees])
            lists = None if rules is None else [_rules_of(rules[i], text[i], m) for i, m in zip(part, masks)]
            picked = rdet.tree_select(model, s, lists)
            paths = [accepted_path(*t, sel, max_new_tokens - len(out[i])) for i, t, sel in zip(part, trees, picked)]
            rdet.tree_accept(model, s, paths)
            for i, (tokens, _), sel, path in zip(part, trees, picked, paths):
                new = [tokens[j] for j in path]
                out[i] += new
                text[i] += new
                drafts[i].extend(new)
                nxt[i] = sel[path[-1]]


def _admissible(allow, output, limit, vocab, tokens, parents):
    """The nodes of a drafted tree that the masks allow behind `output`, as
    (tokens, parents), and the mask after each.  Node 0 is the token that was
    selected, so it is allowed.  An output of `limit` tokens is complete: no
    node follows it, and its mask, which nothing selects under, allows all."""
    kept: list[int] = []   # old numbers
    new: dict[int, int] = {}
    masks, paths, words = [], [], (vocab + 31) // 32
    for j, (t, p) in enumerate(zip(tokens, parents)):
        if j:
            if p not in new or t >= vocab or len(paths[new[p]]) >= limit:
                continue
            if not int(masks[new[p]][t >> 5]) >> (t & 31) & 1:
                continue
        new[j] = len(kept)
        kept.append(j)
        paths.append((list(output) if j == 0 else paths[new[p]]) + [t])
        mask = np.full(words, 0xFFFFFFFF, dtype=np.uint32)
        if len(paths[-1]) < limit:
            mask = np.ascontiguousarray(allow(paths[-1]), dtype=np.uint32)
            if mask.shape != (words,):
                raise ValueError(f"allow: a mask of {words} words")
        masks.append(mask)
    return ([tokens[j] for j in kept], [new[parents[j]] if j else -1 for j in kept]), masks
