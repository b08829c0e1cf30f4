"""Measured cases of the operators that verify drafted tokens, with their plain forms.

Three operators of the det path (Q16.16 activations, exact integer arithmetic,
every result a whole number that has one right value):

tree    attention of a tree of drafted tokens over a KV cache: node i of a
        sequence's tree stands at position context + depth(i) and attends to
        the cache rows of its window, to its ancestors and to itself.
rules   rules on logits rows and the greedy token: repetition, frequency and
        presence penalties over a token history, biases, a mask of allowed
        tokens, then the first maximum.
commit  the K and V rows of an accepted path move from the drafted rows into
        the caches of every layer.

`run` is the plain form (elementary torch operations) while `own` is false
and the framework's call while it is true.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
ONE = 1 << 16
LN2 = 2977044472  # ln 2 in Q32.32
I32_MIN, I32_MAX = -(1 << 31), (1 << 31) - 1
NO_TOKEN = -1     # 0xffffffff as i32: no token of the row is allowed


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    """Head shapes, windows, vocabulary and layer counts are those of
    raster-inference_b200/configs/e4b_text_standin.json (8 query heads on 2 KV
    heads; sliding layers of 256 dims and window 512, full layers of 512 dims;
    24 layers with caches of their own, 4 of them full) and of the tests'
    small configuration."""
    return [
        # the smallest call: a short draft on the tests' small model, where launch latency counts
        dict(name="tree_small", op="tree", seqs=1, nodes=4, lo=37, hi=37, heads=4, kv_heads=2, dim=16, window=8),
        # one conversation, one token per step: the form without a draft
        dict(name="tree_one_token", op="tree", seqs=1, nodes=1, lo=4095, hi=4095, heads=8, kv_heads=2, dim=512, window=0),
        # one conversation, a sliding layer: a draft of 8 over the last 512 positions
        dict(name="tree_sliding", op="tree", seqs=1, nodes=8, lo=4096, hi=4096, heads=8, kv_heads=2, dim=256, window=512),
        # one conversation, a full layer at the benchmark's context
        dict(name="tree_full", op="tree", seqs=1, nodes=16, lo=4096, hi=4096, heads=8, kv_heads=2, dim=512, window=0),
        # a ragged batch of conversations, full layer
        dict(name="tree_batch", op="tree", seqs=16, nodes=11, lo=128, hi=4097, heads=8, kv_heads=2, dim=512, window=0),
        # a long document with the widest tree: the largest call
        dict(name="tree_long", op="tree", seqs=1, nodes=64, lo=32768, hi=32768, heads=8, kv_heads=2, dim=512, window=0),
        # one conversation: only its greedy token under a history's penalties
        dict(name="rules_token", op="rules", seqs=1, nodes=1, vocab=262144, history=513, bias=0, mask=0, write=False),
        # a small odd vocabulary under a grammar that allows few tokens (and for one row none)
        dict(name="rules_odd", op="rules", seqs=3, nodes=5, vocab=32003, history=97, bias=19, mask=2, write=True),
        # every node of a batch of drafts: all rules, the processed rows kept
        dict(name="rules_tree", op="rules", seqs=4, nodes=16, vocab=262144, history=4096, bias=300, mask=1, write=True),
        # one conversation accepts 3 drafted tokens
        dict(name="commit_one", op="commit", seqs=1, nodes=16, accepted=3, sliding=20, full=4, kv_heads=2, cap=160),
        # a batch accepts about 7 of 64 each
        dict(name="commit_batch", op="commit", seqs=16, nodes=64, accepted=7, sliding=20, full=4, kv_heads=2, cap=251),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["tree", "tree", "rules", "commit"])
    if op == "tree":
        dim, window = rng.choice([(16, 8), (64, 0), (128, 256), (256, 512), (512, 0), (80, 0)])
        kv = rng.choice([1, 2, 4])
        group = rng.choice([1, 2, 4])
        nodes = log(1, 64)
        seqs = log(1, 24)
        hi = log(16, 32768)
        # rows x context x dim at most that of the largest listed case, cache memory within 4 GB
        while seqs > 1 and (seqs * nodes * kv * group * hi * dim > 64 * 8 * 32768 * 512 // 4 or seqs * kv * hi * dim * 8 > 4e9):
            seqs = max(1, seqs // 2)
        while nodes * kv * group * hi * dim > 64 * 8 * 32768 * 512:
            hi //= 2
        return dict(op="tree", seqs=seqs, nodes=nodes, lo=max(0, hi // rng.choice([1, 2, 16])), hi=hi, heads=kv * group,
                    kv_heads=kv, dim=dim, window=window)
    if op == "rules":
        vocab = rng.choice([97, 1000, 32003, 65537, 128256, 262144])
        nodes, seqs = log(1, 32), log(1, 8)
        while seqs * nodes > 64:
            nodes -= 1
        return dict(op="rules", seqs=seqs, nodes=nodes, vocab=vocab, history=log(1, 8192), bias=rng.choice([0, 1, 33, 300]),
                    mask=rng.choice([0, 1, 2]), write=rng.random() < 0.7)
    nodes = log(1, 64)
    return dict(op="commit", seqs=log(1, 16), nodes=nodes, accepted=min(nodes, log(1, 12)), sliding=rng.choice([2, 5, 20]),
                full=rng.choice([1, 4]), kv_heads=rng.choice([1, 2, 4]), cap=rng.choice([96, 160, 251]))


def contexts(case):
    """The committed lengths of the case's sequences, spread over [lo, hi]."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi if n == 1 else lo + (hi - lo) * ((i * 7 + 3) % n) // (n - 1) for i in range(n)]


def counts(case):
    """Nodes of each sequence's tree: ragged, at most case["nodes"]."""
    return [max(1, case["nodes"] - i % 3) for i in range(case["seqs"])]


def work(case):
    if case["op"] == "tree":
        heads, kv, d, w = case["heads"], case["kv_heads"], case["dim"], case["window"]
        byts = flops = 0
        for c, t in zip(contexts(case), counts(case)):
            rows = min(c, w - 1) if w else c
            byts += 2 * kv * (rows + t) * d * 4 + 2 * t * heads * d * 4
            flops += t * heads * (rows + 1) * d * 2 * 2
        return {"bytes": byts, "flops": flops}
    if case["op"] == "rules":
        rows, v = sum(counts(case)), case["vocab"]
        byts = rows * v * 4 * (2 if case["write"] else 1) + rows * 4
        byts += rows * ((v + 31) // 32) * 4 if case["mask"] else 0
        byts += case["seqs"] * (case["history"] * 4 + case["bias"] * 8)
        return {"bytes": byts, "flops": rows * v}
    rows = case["seqs"] * accepted(case) * 2 * case["kv_heads"]
    return {"bytes": 2 * 4 * rows * (case["sliding"] * 256 + case["full"] * 512), "flops": 0}


def accepted(case):
    return min(case["accepted"], case["nodes"])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def trees(rnd, case):
    """A draft as a drafter makes it: one likely chain with alternatives on
    the way (parents come before their children, -1 is the last committed token)."""
    out = []
    for n in counts(case):
        par = [-1]
        for i in range(1, n):
            par.append(i - 1 if rnd.random() < 0.5 else rnd.randrange(max(0, i - 6), i))
        out.append(par)
    return out


def normal(gen, shape, std):
    """Q16.16 values of a normal distribution (activations after their norms)."""
    return (torch.randn(shape, generator=gen, device=DEV) * (std * ONE)).round().to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = random.Random(seed)
    st = {"tree": prepare_tree, "rules": prepare_rules, "commit": prepare_commit}[case["op"]](case, gen, rnd)
    st["case"] = case
    if own:
        plan(st)
    return st


def prepare_tree(case, gen, rnd):
    s, t, kv, d = case["seqs"], case["nodes"], case["kv_heads"], case["dim"]
    cap = max(contexts(case)) + t
    par = trees(rnd, case)
    total = sum(len(p) for p in par)
    pad = torch.tensor([p + [-1] * (t - len(p)) for p in par], device=DEV)
    first = np.cumsum([0] + [len(p) for p in par])
    # row of every (sequence, node) in the packed queries, 0 where a tree is shorter
    at = torch.tensor([[first[i] + min(j, len(p) - 1) for j in range(t)] for i, p in enumerate(par)], device=DEV)
    real = torch.tensor([[j < len(p) for j in range(t)] for p in par], device=DEV)
    return dict(k=normal(gen, (s, kv, cap, d), 1.0), v=normal(gen, (s, kv, cap, d), 1.0),
                q=normal(gen, (total, case["heads"], d), 0.2), parents=par, pad=pad, at=at, real=real,
                ctx=torch.tensor(contexts(case), device=DEV),
                out=torch.empty((total, case["heads"], d), dtype=torch.int32, device=DEV))


def prepare_rules(case, gen, rnd):
    s, t, v = case["seqs"], case["nodes"], case["vocab"]
    par = trees(rnd, case)
    n = [len(p) for p in par]
    total = sum(n)
    logits = normal(gen, (total, v), 4.0).clamp_(-30 * ONE, 30 * ONE)
    # token ids as text has them: few are frequent
    def ids(shape):
        return (torch.rand(shape, generator=gen, device=DEV).pow(3) * v).to(torch.int32).clamp_(max=v - 1)
    st = dict(logits=logits, history=ids((s, case["history"])), tokens=ids((total,)), parents=par,
              bias_ids=ids((s, case["bias"])), bias=normal(gen, (s, case["bias"]), 2.0),
              out=torch.empty_like(logits) if case["write"] else None,
              chosen=torch.empty((total,), dtype=torch.int32, device=DEV), allow=None)
    if case["mask"]:
        words = (v + 31) // 32
        if case["mask"] == 1:    # a mask that forbids a part
            m = torch.randint(I32_MIN, I32_MAX, (total, words), generator=gen, device=DEV, dtype=torch.int64)
            m |= torch.randint(I32_MIN, I32_MAX, (total, words), generator=gen, device=DEV, dtype=torch.int64)
        else:                    # a grammar's: few tokens left, for the last row none
            keep = torch.rand((total, words), generator=gen, device=DEV) < 8.0 / words
            m = torch.where(keep, torch.randint(I32_MIN, I32_MAX, (total, words), generator=gen, device=DEV, dtype=torch.int64), 0)
            m[-1] = 0
        st["allow"] = m.to(torch.int32).contiguous()
    # one conversation's penalties: Q16.16 repetition, frequency, presence
    st["penalty"] = [(ONE + rnd.randrange(1, 30000), rnd.randrange(0, 40000), rnd.randrange(0, 40000)) for _ in range(s)]
    first = np.cumsum([0] + n)
    st["seq_of"] = torch.tensor([i for i in range(s) for _ in range(n[i])], device=DEV)
    # parents as rows of the call, -1 for a root
    st["row_parent"] = torch.tensor([int(first[i]) + q if q >= 0 else -1 for i, p in enumerate(par) for q in p], device=DEV)
    st["pen"] = torch.tensor(st["penalty"], device=DEV)
    return st


def prepare_commit(case, gen, rnd):
    s, kv, cap, n = case["seqs"], case["kv_heads"], case["cap"], case["nodes"]
    a = accepted(case)
    st = dict(path=[sorted(rnd.sample(range(n), a)) for _ in range(s)], ctx=[cap - a - rnd.randrange(0, 20) for _ in range(s)])
    for name, layers, d in (("sliding", case["sliding"], 256), ("full", case["full"], 512)):
        st[name] = normal(gen, (s, layers, 2, kv, cap, d), 1.0)        # the caches, K and V
        st[name + "_draft"] = normal(gen, (s, layers, 2, kv, n, d), 1.0)  # the drafted rows
    st["path_dev"] = torch.tensor(st["path"], device=DEV)
    st["ctx_dev"] = torch.tensor(st["ctx"], device=DEV)
    return st


def plan(st):
    """The call's descriptors, as a program keeps them beside its buffers."""
    lib = importlib.import_module("raster-inference_b200")
    st["lib"], case = lib, st["case"]
    if case["op"] == "tree":
        k, v, d = st["k"], st["v"], case["dim"]
        st["seqs"] = lib.tree_seqs([
            dict(k_cache=k[i].data_ptr(), v_cache=v[i].data_ptr(), cap=k.shape[2], context=c,
                 k_tree=k[i].data_ptr() + c * d * 4, v_tree=v[i].data_ptr() + c * d * 4, tree_cap=k.shape[2], parents=p)
            for i, (c, p) in enumerate(zip(contexts(case), st["parents"]))])
        n = lib.det_attention_tree_workspace(st["seqs"], case["heads"], case["kv_heads"], d, case["window"])
        st["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    elif case["op"] == "rules":
        rows, r, tok = [], 0, st["tokens"].tolist()
        for i, par in enumerate(st["parents"]):
            rep, freq, pres = st["penalty"][i]
            for j, p in enumerate(par):
                rows.append(dict(logits=st["logits"][r].data_ptr(), out=st["out"][r].data_ptr() if case["write"] else 0,
                                 allow=st["allow"][r].data_ptr() if st["allow"] is not None else 0,
                                 history=st["history"][i].data_ptr(), history_len=case["history"],
                                 bias_ids=st["bias_ids"][i].data_ptr() if case["bias"] else 0,
                                 bias_values=st["bias"][i].data_ptr() if case["bias"] else 0, n_bias=case["bias"],
                                 repetition=rep, frequency=freq, presence=pres,
                                 parent=r - j + p if p >= 0 else -1, token=tok[r]))
                r += 1
        st["rows"] = lib.logit_rows(rows)
    else:
        moves = []
        for i in range(case["seqs"]):
            for name in ("sliding", "full"):
                for x, y in zip(st[name][i].flatten(0, 1), st[name + "_draft"][i].flatten(0, 1)):
                    moves.append(dict(cache=x.data_ptr(), cap=x.shape[1], kv_heads=x.shape[0], head_dim=x.shape[2],
                                      draft=y.data_ptr(), draft_cap=y.shape[1], context=st["ctx"][i], path=i))
        st["moves"] = lib.tree_moves(moves, st["path"])


# ---------------------------------------------------------------------------
# the pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if case["op"] == "tree":
            st["lib"].det_attention_tree(st["seqs"], st["q"].data_ptr(), case["heads"], case["kv_heads"], case["dim"],
                                         case["window"], st["out"].data_ptr(), st["ws"].data_ptr(), st["ws"].numel(), stream)
            return st["out"]
        if case["op"] == "rules":
            st["lib"].det_logits_rules(st["rows"], case["vocab"], st["chosen"].data_ptr(), stream)
            return [st["out"], st["chosen"]] if case["write"] else st["chosen"]
        st["lib"].det_tree_commit(st["moves"], stream)
        return [st["sliding"], st["full"]]
    return {"tree": plain_tree, "rules": plain_rules, "commit": plain_commit}[case["op"]](st)


def half_even(q, r, d):
    """q + 1 where the remainder r of a division by d (both >= 0) is over half, or half and q odd."""
    return q + ((2 * r > d) | ((2 * r == d) & (q % 2 == 1))).to(torch.int64)


def requantize(x):
    """i64 Q32.32 to i32 Q16.16, half to even, saturated (in an i64 tensor)."""
    return half_even(x >> 16, x & 0xFFFF, torch.full_like(x, 1 << 16)).clamp_(I32_MIN, I32_MAX)


def dots(a, b):
    """Exact sums of products of whole numbers, mod 2^64: a [..., m, k] (33 bits) with b [..., n, k] (32 bits).
    16-bit halves make every product and sum of the f64 matrix products exact."""
    ah, al = (a >> 16).double(), (a & 0xFFFF).double()
    bh, bl = (b >> 16).double().transpose(-1, -2), (b & 0xFFFF).double().transpose(-1, -2)
    mid = (ah @ bl).to(torch.int64) + (al @ bh).to(torch.int64)
    return ((ah @ bh).to(torch.int64) << 32) + (mid << 16) + (al @ bl).to(torch.int64)


def exp_q32(delta):
    """exp(delta) in Q32.32 for Q16.16 delta <= 0: halvings and a fifth-order series, 0 from -16 down."""
    pos = (-delta).clamp(max=16 << 16) << 16
    shift = pos // LN2
    r = pos - shift * LN2

    def mul(x, y):
        p = x * y
        return half_even(p >> 32, p & 0xFFFFFFFF, torch.full_like(p, 1 << 32))

    def div(x, k):
        return half_even(x // k, x % k, torch.full_like(x, k))

    r2 = mul(r, r)
    r3 = mul(r2, r)
    r4 = mul(r3, r)
    r5 = mul(r4, r)
    e = (1 << 32) - r + div(r2, 2) - div(r3, 6) + div(r4, 24) - div(r5, 120)
    one = torch.ones_like(e)
    e = torch.where(shift > 0, half_even(e >> shift, e & ((one << shift) - 1), one << shift), e)
    return torch.where(delta <= -(16 << 16), torch.zeros_like(e), e)


def weight_q16(e, total):
    """requantize(e / total in Q32.32), both roundings half to even; the quotient's 32 bits in four steps of 8."""
    q, r = e // total, e % total
    r = r << 8
    q, r = (q << 8) + r // total, (r % total) << 8
    q, r = (q << 8) + r // total, (r % total) << 8
    q, r = (q << 8) + r // total, (r % total) << 8
    q, r = (q << 8) + r // total, r % total
    return requantize(half_even(q, r, total))


def ancestors(parent):
    """[.., t] parents (-1: none) -> [.., t, t] whether column j is row i itself or one of its ancestors."""
    t = parent.shape[-1]
    step = torch.eye(t, device=parent.device) + torch.nn.functional.one_hot(parent + 1, t + 1)[..., 1:].float()
    reach = (step @ step).clamp(max=1)
    reach = (reach @ reach).clamp(max=1)
    reach = (reach @ reach).clamp(max=1)
    reach = (reach @ reach).clamp(max=1)
    reach = (reach @ reach).clamp(max=1)
    return (reach @ reach) > 0


def plain_tree(st):
    case = st["case"]
    s, t, heads, kv, d, w = (case[x] for x in ("seqs", "nodes", "heads", "kv_heads", "dim", "window"))
    g, ctx = heads // kv, st["ctx"].view(-1, 1, 1)
    anc = ancestors(st["pad"])
    depth = anc.sum(-1) - 1                                             # [s, t]
    pos = ctx[..., 0] + depth
    start = (pos + 1 - w).clamp(min=0) if w else torch.zeros_like(pos)
    n = st["k"].shape[2]
    row = torch.arange(n, device=DEV).view(1, 1, -1)
    node = (row - ctx).clamp(0, t - 1).expand(s, t, n)
    seen = torch.where(row < ctx, row >= start.unsqueeze(-1), anc.gather(2, node) & (row - ctx < t))
    key_pos = torch.where(row < ctx, row.expand(s, t, n), ctx + depth.unsqueeze(1).expand(s, t, t).gather(2, node))
    seen = seen & (key_pos >= start.unsqueeze(-1))                      # [s, t, n]
    q = st["q"].long()[st["at"]].view(s, t, kv, g, d).permute(0, 2, 3, 1, 4).reshape(s, kv, g * t, d)
    score = requantize(dots(q, st["k"].long())).view(s, kv, g, t, n)
    seen = seen[:, None, None].expand_as(score)
    top = score.masked_fill(~seen, I32_MIN - 1).amax(-1, keepdim=True)
    first = torch.where(seen & (score == top), row.view(1, 1, 1, 1, -1), n).amin(-1, keepdim=True)
    e = torch.where(seen, exp_q32((score - top).clamp(min=I32_MIN, max=0)), 0)
    wgt = weight_q16(e, e.sum(-1, keepdim=True))
    left = ONE - wgt.sum(-1, keepdim=True)                              # what rounding left goes to the first maximum
    wgt = wgt.scatter_add(-1, first, left).view(s, kv, g * t, n)
    o = requantize(dots(wgt, st["v"].long().transpose(-1, -2)))
    o = o.view(s, kv, g, t, d).permute(0, 3, 1, 2, 4).reshape(s, t, heads, d).to(torch.int32)
    return o[st["real"]]


def plain_rules(st):
    case = st["case"]
    v, x = case["vocab"], st["logits"].long()
    seq = st["seq_of"]
    rep, freq, pres = (c.unsqueeze(-1) for c in st["pen"][seq].unbind(-1))
    count = torch.zeros((case["seqs"], v), dtype=torch.int64, device=DEV)
    count = count.scatter_add(1, st["history"].long(), torch.ones_like(st["history"], dtype=torch.int64))[seq]
    path = ancestors(st["row_parent"]).long()                           # a node's own token and its ancestors'
    count = count.scatter_add(1, st["tokens"].long().expand(path.shape), path)
    # repetition: divided where positive, multiplied otherwise
    num = (x << 16).clamp(min=0)
    down = half_even(num // rep, num % rep, rep.expand_as(x)).clamp(max=I32_MAX)
    y = torch.where(x > 0, down, requantize(x * rep))
    y = (y - (freq * count).clamp(max=I32_MAX)).clamp(I32_MIN, I32_MAX)
    y = (y - pres).clamp(I32_MIN, I32_MAX)
    y = torch.where(count > 0, y, x)
    if case["bias"]:
        b = torch.zeros((case["seqs"], v), dtype=torch.int64, device=DEV)
        b = b.scatter_add(1, st["bias_ids"].long(), st["bias"].long()).clamp_(I32_MIN, I32_MAX)
        y = (y + b[seq]).clamp(I32_MIN, I32_MAX)
    ids = torch.arange(v, device=DEV)
    ok = torch.ones_like(y, dtype=torch.bool)
    if st["allow"] is not None:
        ok = (st["allow"][:, ids // 32] >> (ids % 32).to(torch.int32)) & 1 == 1
    top = y.masked_fill(~ok, I32_MIN - 1).amax(-1, keepdim=True)
    best = torch.where(ok & (y == top), ids, v).amin(-1)
    chosen = torch.where(best < v, best, NO_TOKEN).to(torch.int32)
    return [y.masked_fill(~ok, I32_MIN).to(torch.int32), chosen] if case["write"] else chosen


def plain_commit(st):
    s, a = st["path_dev"].shape
    seq = torch.arange(s, device=DEV).view(-1, 1)
    row = st["ctx_dev"].view(-1, 1) + torch.arange(a, device=DEV)
    st["sliding"].permute(0, 4, 1, 2, 3, 5)[seq, row] = st["sliding_draft"].permute(0, 4, 1, 2, 3, 5)[seq, st["path_dev"]]
    st["full"].permute(0, 4, 1, 2, 3, 5)[seq, row] = st["full_draft"].permute(0, 4, 1, 2, 3, 5)[seq, st["path_dev"]]
    return [st["sliding"], st["full"]]


# ---------------------------------------------------------------------------
# from the definitions, row by row, in wrapping i64 and Python's whole numbers
# ---------------------------------------------------------------------------
def rte(n, d):
    """round half to even of n / d, d > 0 (Python's whole numbers)."""
    q, r = divmod(n, d)
    return q + (1 if 2 * r > d or (2 * r == d and q & 1) else 0)


def sat(x):
    return max(I32_MIN, min(I32_MAX, x))


def exp_exact(d):
    if d <= -(16 << 16):
        return 0
    shift, r = divmod(-d << 16, LN2)
    powers = [r]
    for _ in range(4):
        powers.append(rte(powers[-1] * r, 1 << 32))
    e = (1 << 32) - r + rte(powers[1], 2) - rte(powers[2], 6) + rte(powers[3], 24) - rte(powers[4], 120)
    return rte(e, 1 << shift)


def exact(case, seed):
    if case["op"] == "tree":
        if work(case)["flops"] > 3e9 or sum(counts(case)) * case["heads"] * max(contexts(case)) > 1.5e6:
            return None
        return exact_tree(case, prepare(case, seed))
    if case["op"] == "rules":
        if sum(counts(case)) * case["vocab"] > 3e7:
            return None
        return exact_rules(case, prepare(case, seed))
    if work(case)["bytes"] > 1e8:
        return None
    st = prepare(case, seed)
    res = []
    for name in ("sliding", "full"):
        x, y = st[name].cpu().numpy(), st[name + "_draft"].cpu().numpy()
        for i, path in enumerate(st["path"]):
            for j, n in enumerate(path):
                x[i, :, :, :, st["ctx"][i] + j] = y[i, :, :, :, n]
        res.append(torch.from_numpy(x))
    return res


def exact_tree(case, st):
    g, w = case["heads"] // case["kv_heads"], case["window"]
    q, res, at = st["q"].cpu().numpy().astype(np.int64), np.empty(st["q"].shape, np.int32), 0
    for i, (c, par) in enumerate(zip(contexts(case), st["parents"])):
        k, v = (st[x][i].cpu().numpy().astype(np.int64) for x in "kv")
        for j in range(len(par)):
            path, n = [], j
            while n >= 0:
                path.insert(0, n)
                n = par[n]
            rows = list(range(c)) + [c + n for n in path]       # in the order of their positions
            rows = np.array(rows[-w:] if w else rows)
            for h in range(case["heads"]):
                acc = (k[h // g][rows] * q[at + j, h]).sum(-1)
                s = [sat(rte(int(x), 1 << 16)) for x in acc]
                top = max(s)
                e = [exp_exact(x - top) for x in s]
                total = sum(e)
                wt = [sat(rte(rte(x << 32, total), 1 << 16)) if x else 0 for x in e]
                wt[s.index(top)] += ONE - sum(wt)
                o = (v[h // g][rows] * np.array(wt, np.int64)[:, None]).sum(0)
                res[at + j, h] = [sat(rte(int(x), 1 << 16)) for x in o]
        at += len(par)
    return torch.from_numpy(res)


def exact_rules(case, st):
    x, tok = st["logits"].cpu().numpy().astype(np.int64), st["tokens"].tolist()
    chosen, at = [], 0
    for i, par in enumerate(st["parents"]):
        rep, freq, pres = st["penalty"][i]
        hist, bias = st["history"][i].tolist(), {}
        for t, b in zip(st["bias_ids"][i].tolist(), st["bias"][i].tolist()):
            bias[t] = bias.get(t, 0) + b
        for j in range(len(par)):
            seen, n = list(hist), j
            while n >= 0:
                seen.append(tok[at + n])
                n = par[n]
            count, row = {}, x[at + j]
            for t in seen:
                count[t] = count.get(t, 0) + 1
            for t, c in count.items():
                l = int(row[t])
                l = sat(rte(l << 16, rep)) if l > 0 else sat(rte(l * rep, 1 << 16))
                row[t] = sat(sat(l - sat(freq * c)) - pres)
            for t, b in bias.items():
                row[t] = sat(int(row[t]) + sat(b))
            if st["allow"] is not None:
                words = st["allow"][at + j].cpu().numpy().view(np.uint32)
                ok = np.unpackbits(words.view(np.uint8), bitorder="little")[:case["vocab"]].astype(bool)
            else:
                ok = np.ones(case["vocab"], bool)
            live = np.flatnonzero(ok)
            chosen.append(int(live[np.argmax(row[live])]) if len(live) else NO_TOKEN)
            row[~ok] = I32_MIN
        at += len(par)
    chosen = torch.tensor(chosen, dtype=torch.int32)
    return [torch.from_numpy(x.astype(np.int32)), chosen] if case["write"] else chosen
