"""Plain whole-number implementations of the draft-verification operators,
from their definitions, over the oracle's scalar arithmetic."""
import numpy as np

import oracle as O

I32_MIN, I32_MAX = -2**31, 2**31 - 1
ONE = 1 << 16
NO_TOKEN = 0xFFFFFFFF


def path_of(parents, node):
    """The nodes from the root to `node`."""
    out = []
    while node >= 0:
        out.insert(0, node)
        node = parents[node]
    return out


def attention_tree(q, k, v, kt, vt, context, parents, window):
    """q [n, Hq, d]; k, v [Hkv, >= context, d]; kt, vt [Hkv, >= n, d]."""
    n, hq, d = q.shape
    g = hq // k.shape[0]
    out = np.empty_like(q)
    for i in range(n):
        path = path_of(parents, i)
        for h in range(hq):
            keys = np.concatenate([k[h // g, :context], kt[h // g, path]])
            vals = np.concatenate([v[h // g, :context], vt[h // g, path]])
            if window:
                keys, vals = keys[-window:], vals[-window:]
            out[i, h] = O.attention_one(q[i, h], np.ascontiguousarray(keys), np.ascontiguousarray(vals))
    return out


def sat(x):
    return max(I32_MIN, min(I32_MAX, x))


def rules_row(logits, counts, rep, freq, pres, bias, allow):
    """(processed row, token): logits i32 [V], counts {token: count}, bias a
    list of (token, value), allow a bool [V] or None."""
    L = O.lib()
    row = [int(x) for x in logits]
    vocab = len(row)
    for t, c in counts.items():
        if c and t < vocab:
            l = row[t]
            l = L.dor_div_act(l, rep) if l > 0 else L.dor_mul_sat(l, rep)
            l = L.dor_sub_sat(l, sat(freq * c))
            row[t] = L.dor_sub_sat(l, pres)
    total = {}
    for t, b in bias:
        total[t] = total.get(t, 0) + b
    for t, b in total.items():
        if t < vocab:
            row[t] = L.dor_add_sat(row[t], sat(b))
    best = NO_TOKEN
    for t in range(vocab):
        if allow is None or allow[t]:
            if best == NO_TOKEN or row[t] > row[best]:
                best = t
        else:
            row[t] = I32_MIN
    return np.array(row, dtype=np.int64).astype(np.int32), best
