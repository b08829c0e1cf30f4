"""The draft-verification operators against plain whole-number
implementations, through the C ABI on device buffers (torch holds the
memory).  Every result is a whole number with one right value, so the
tolerance is zero throughout."""
import numpy as np
import pytest

import draft_ref as R
from helpers import rdet

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

I32_MIN, I32_MAX = -2**31, 2**31 - 1


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def random_tree(rng, n, roots=False):
    par = [-1]
    for i in range(1, n):
        par.append(int(rng.integers(-1 if roots else 0, i)) if rng.random() < 0.5 else i - 1)
    return par


def values(rng, shape, kind):
    """Activations after a norm, values of any size, or the type's limits and
    their neighbours (every digit and carry of a limb decomposition)."""
    if kind == "norm":
        return np.round(rng.normal(0, 40000, shape)).astype(np.int32)
    if kind == "wide":
        return rng.integers(I32_MIN, I32_MAX + 1, shape, dtype=np.int64).astype(np.int32)
    edge = np.array([I32_MIN, I32_MIN + 1, I32_MAX, I32_MAX - 1, 0, 1, -1, 0x7F7F7F7F, 0x7F7F7F80, 0x7F7F7FFF,
                     -0x7F7F7F80, -0x7F808080, 127, 128, -128, -129, 32767, 32768,
                     -32768, -32769, 0x7FFFFF, 0x800000, -0x800000, 65536], dtype=np.int64)
    return edge[rng.integers(0, edge.size, shape)].astype(np.int32)


class Case:
    """Device buffers of a batch of trees; `own` puts the drafted rows into
    buffers of their own, else they follow the context in the cache."""

    def __init__(self, rng, ctxs, trees, heads, kv, d, kind, own=False, qscale=None, shift=0, cap_extra=0):
        n = sum(len(t) for t in trees)
        q = values(rng, (n, heads, d), kind)
        self.q = q if qscale is None else (q // qscale).astype(np.int32)
        self.parts, self.keep, items = [], [], []
        for c, par in zip(ctxs, trees):
            cap = c + (0 if own else len(par)) + cap_extra
            k, v = values(rng, (kv, max(cap, 1), d), kind), values(rng, (kv, max(cap, 1), d), kind)
            kd, vd = self.put(k, shift), self.put(v, shift)
            if own:
                tc = len(par) + 2
                kt, vt = values(rng, (kv, tc, d), kind), values(rng, (kv, tc, d), kind)
                ktd, vtd = self.put(kt, shift), self.put(vt, shift)
                it = dict(k_tree=ktd, v_tree=vtd, tree_cap=tc)
            else:
                kt, vt = k[:, c:], v[:, c:]
                it = dict(k_tree=kd + c * d * 4, v_tree=vd + c * d * 4, tree_cap=cap)
            items.append(dict(k_cache=kd, v_cache=vd, cap=cap, context=c, parents=par, **it))
            self.parts.append((k, v, kt, vt, c, par))
        self.heads, self.kv, self.d = heads, kv, d
        self.seqs = rdet.tree_seqs(items)

    def put(self, a, shift):
        t = torch.zeros(a.size + shift, dtype=torch.int32, device="cuda")
        t[shift:] = dev(a.reshape(-1))
        self.keep.append(t)
        return t.data_ptr() + 4 * shift

    def run(self, window, shift=0, stream=None):
        s = stream.cuda_stream if stream else 0
        qd = torch.zeros(self.q.size + shift, dtype=torch.int32, device="cuda")
        qd[shift:] = dev(self.q.reshape(-1))
        out = torch.full((self.q.size + shift,), 77, dtype=torch.int32, device="cuda")
        need = rdet.det_attention_tree_workspace(self.seqs, self.heads, self.kv, self.d, window)
        ws = torch.randint(0, 255, (need,), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        rdet.det_attention_tree(self.seqs, qd.data_ptr() + 4 * shift, self.heads, self.kv, self.d, window,
                                out.data_ptr() + 4 * shift, ws.data_ptr(), need, s)
        torch.cuda.synchronize()
        assert (out[:shift] == 77).all()
        return out[shift:].cpu().numpy().reshape(self.q.shape)

    def want(self, window):
        res, at = [], 0
        for k, v, kt, vt, c, par in self.parts:
            res.append(R.attention_tree(self.q[at:at + len(par)], k, v, kt, vt, c, par, window))
            at += len(par)
        return np.concatenate(res)


@pytest.mark.parametrize("ctx,nodes,heads,kv,d,window", [
    (0, 1, 1, 1, 1, 0), (0, 7, 4, 2, 16, 0), (1, 1, 2, 1, 2, 0), (5, 3, 4, 2, 16, 8), (37, 4, 4, 2, 16, 8),
    (20, 12, 2, 2, 6, 3), (40, 30, 4, 1, 10, 5), (63, 1, 8, 2, 64, 0), (64, 2, 8, 2, 64, 0), (127, 8, 8, 2, 64, 0),
    (130, 64, 4, 2, 32, 0), (200, 17, 3, 3, 80, 64), (700, 9, 8, 1, 128, 512), (511, 5, 8, 2, 256, 512),
    (1000, 16, 8, 2, 256, 512), (300, 5, 8, 2, 512, 0), (90, 3, 12, 2, 100, 1), (33, 8, 10, 2, 5, 0),
    (70, 6, 16, 1, 24, 0), (2049, 3, 2, 1, 33, 0)])
@pytest.mark.parametrize("kind", ["norm", "wide", "edge"])
def test_tree_attention(ctx, nodes, heads, kv, d, window, kind):
    rng = np.random.default_rng(ctx * 131 + nodes * 7 + d)
    c = Case(rng, [ctx], [random_tree(rng, nodes, roots=nodes % 2 == 1)], heads, kv, d, kind,
             qscale=8 if kind == "norm" else None, own=nodes % 3 == 0)
    assert np.array_equal(c.run(window), c.want(window))


@pytest.mark.parametrize("window", [0, 8, 100])
@pytest.mark.parametrize("own", [False, True])
def test_tree_attention_ragged_batch(window, own):
    # more sequences than one launch group takes, a context of every kind
    rng = np.random.default_rng(5 + window)
    ctxs = [0, 1, 7, 8, 9, 63, 64, 65, 127, 128, 129, 300] * 3
    trees = [random_tree(rng, int(rng.integers(1, 20))) for _ in ctxs]
    c = Case(rng, ctxs, trees, 4, 2, 64, "norm", own=own, qscale=8, cap_extra=3)
    assert np.array_equal(c.run(window), c.want(window))


@pytest.mark.parametrize("ctx,nodes,heads,kv,d,window", [
    (5000, 20, 8, 2, 16, 0),      # blocks of 64 rows, the last one short, several tiles a CTA
    (9001, 40, 8, 2, 80, 0),      # two chunks of dims, the second short
    (5003, 33, 4, 2, 7, 0),       # rows that are not 16-byte aligned
    (5000, 64, 4, 2, 16, 4500),   # windows that begin inside the tiles
    (6000, 16, 4, 1, 130, 0),     # two blocks of dims
    (40000, 1, 2, 1, 64, 0),      # few rows, many tiles a CTA
    (40000, 8, 4, 1, 36, 0),
    (1500, 64, 32, 4, 8, 0)])     # more rows than softmax CTAs are resident
@pytest.mark.parametrize("kind", ["norm", "wide", "edge"])
def test_tree_attention_long(ctx, nodes, heads, kv, d, window, kind):
    rng = np.random.default_rng(ctx + nodes + d)
    c = Case(rng, [ctx], [random_tree(rng, nodes, roots=nodes % 2 == 1)], heads, kv, d, kind,
             qscale=8 if kind == "norm" else None, own=nodes % 3 == 0)
    assert np.array_equal(c.run(window), c.want(window))


def test_tree_attention_ragged_batch_of_wide_blocks():
    rng = np.random.default_rng(77)
    ctxs = [900, 0, 2500, 64, 1300, 4001, 127, 3000]
    trees = [random_tree(rng, n) for n in (20, 64, 17, 33, 1, 40, 16, 64)]
    c = Case(rng, ctxs, trees, 8, 2, 32, "norm", own=True, qscale=8, cap_extra=5)
    assert np.array_equal(c.run(0), c.want(0))


@pytest.mark.parametrize("ctx", [200000, 300000])
def test_tree_attention_of_the_longest_rows(ctx):
    # rows of eight and of sixteen softmax CTAs
    rng = np.random.default_rng(ctx)
    c = Case(rng, [ctx], [[-1, 0]], 2, 1, 4, "norm", qscale=8)
    assert np.array_equal(c.run(0), c.want(0))


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_tree_attention_unaligned(shift):
    # rows that start off a 16-byte boundary
    rng = np.random.default_rng(shift)
    c = Case(rng, [150], [random_tree(rng, 6)], 4, 2, 64, "norm", qscale=8, shift=shift)
    assert np.array_equal(c.run(0, shift=shift), c.want(0))


def test_tree_attention_chain_is_the_decode():
    # a chain's last node gives what the decode attention gives with the chain committed
    rng = np.random.default_rng(11)
    n, ctx, heads, kv, d = 6, 90, 8, 2, 64
    for window in (0, 32):
        c = Case(rng, [ctx], [[i - 1 for i in range(n)]], heads, kv, d, "norm", qscale=8)
        got = c.run(window)
        k, v = dev(c.parts[0][0]), dev(c.parts[0][1])
        for i in range(n):
            qd, out = dev(c.q[i]), torch.zeros((heads, d), dtype=torch.int32, device="cuda")
            rdet.det_attention_decode(qd.data_ptr(), k.data_ptr(), v.data_ptr(), ctx + n, heads, kv, d, ctx + i,
                                      window, out.data_ptr())
            torch.cuda.synchronize()
            assert np.array_equal(got[i], out.cpu().numpy())


def test_tree_attention_saturated_scores():
    # every score at one end of the type: the first key of the row takes the residual
    rng = np.random.default_rng(3)
    for sign in (1, -1):
        c = Case(rng, [70], [random_tree(rng, 5)], 2, 1, 32, "norm")
        c.q[:] = I32_MAX
        for i in (0,):
            k, v, kt, vt, ctx, par = c.parts[i]
            k[:] = sign * (I32_MAX - 5)
            c.keep[0][:] = dev(k.reshape(-1))
        assert np.array_equal(c.run(0), c.want(0))


def test_tree_attention_many_small_weights():
    # equal scores over more keys than 2^16: each weight rounds by itself and
    # the first key's residual is negative
    n, d = 100000, 2
    q = np.zeros((1, 1, d), np.int32)
    k = np.zeros((1, n + 1, d), np.int32)
    v = np.random.default_rng(1).integers(-2**20, 2**20, (1, n + 1, d)).astype(np.int32)
    kd, vd, qd = dev(k), dev(v), dev(q)
    out = torch.zeros((1, 1, d), dtype=torch.int32, device="cuda")
    s = rdet.tree_seqs([dict(k_cache=kd.data_ptr(), v_cache=vd.data_ptr(), cap=n + 1, context=n,
                             k_tree=kd.data_ptr() + n * d * 4, v_tree=vd.data_ptr() + n * d * 4, tree_cap=n + 1,
                             parents=[-1])])
    need = rdet.det_attention_tree_workspace(s, 1, 1, d, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    rdet.det_attention_tree(s, qd.data_ptr(), 1, 1, d, 0, out.data_ptr(), ws.data_ptr(), need)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), R.attention_tree(q, k[:, :n], v[:, :n], k[:, n:], v[:, n:], n, [-1], 0))


def test_tree_attention_rows_past_2_31_elements():
    # a cache whose second KV head starts past 2^31 elements: only the rows in reach are written
    d, cap = 512, (1 << 22) + 64
    rng = np.random.default_rng(2)
    base = torch.zeros(2 * cap * d, dtype=torch.int32, device="cuda").view(2, cap, d)
    ctx, par = 40, [-1, 0, 0]
    k = values(rng, (2, ctx + 3, d), "norm")
    base[:, :ctx + 3] = dev(k)
    q = values(rng, (3, 4, d), "norm") // 8
    qd, out = dev(q), torch.zeros((3, 4, d), dtype=torch.int32, device="cuda")
    p = base.data_ptr()
    s = rdet.tree_seqs([dict(k_cache=p, v_cache=p, cap=cap, context=ctx, k_tree=p + ctx * d * 4,
                             v_tree=p + ctx * d * 4, tree_cap=cap, parents=par)])
    need = rdet.det_attention_tree_workspace(s, 4, 2, d, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    rdet.det_attention_tree(s, qd.data_ptr(), 4, 2, d, 0, out.data_ptr(), ws.data_ptr(), need)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), R.attention_tree(q, k[:, :ctx], k[:, :ctx], k[:, ctx:], k[:, ctx:], ctx, par, 0))


def test_tree_attention_streams_and_repeats():
    # two calls on streams of their own with workspaces of their own, and the same call again
    rng = np.random.default_rng(8)
    a = Case(rng, [600, 20], [random_tree(rng, 9), random_tree(rng, 3)], 8, 2, 64, "norm", qscale=8)
    b = Case(rng, [333], [random_tree(rng, 16)], 8, 2, 128, "norm", qscale=8)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    first = a.run(0, stream=sa), b.run(64, stream=sb)
    again = b.run(64, stream=sa), a.run(0, stream=sb)
    assert np.array_equal(first[0], again[1]) and np.array_equal(first[1], again[0])
    assert np.array_equal(first[0], a.want(0)) and np.array_equal(first[1], b.want(64))


def test_tree_attention_in_a_graph():
    rng = np.random.default_rng(9)
    c = Case(rng, [257], [random_tree(rng, 8)], 8, 2, 64, "norm", qscale=8)
    want = c.run(0)
    qd, out = dev(c.q), torch.zeros(c.q.shape, dtype=torch.int32, device="cuda")
    need = rdet.det_attention_tree_workspace(c.seqs, 8, 2, 64, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rdet.det_attention_tree(c.seqs, qd.data_ptr(), 8, 2, 64, 0, out.data_ptr(), ws.data_ptr(), need,
                                torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)


def test_tree_attention_no_sequences():
    rdet.det_attention_tree(rdet.tree_seqs([]), 0, 4, 2, 16, 0, 0, 0, 0)


# ---------------------------------------------------------------------------
# rules on logits
# ---------------------------------------------------------------------------
def rules_case(rng, vocab, trees, hist, nbias, mask, write, inplace=False, shift=0, extreme=False):
    rows = sum(len(t) for t in trees)
    logits = rng.integers(I32_MIN, I32_MAX + 1, (rows, vocab), dtype=np.int64).astype(np.int32) if extreme else \
        np.clip(np.round(rng.normal(0, 300000, (rows, vocab))), -30 * 65536, 30 * 65536).astype(np.int32)
    ld = vocab + shift
    lg = torch.zeros(rows * ld + shift, dtype=torch.int32, device="cuda")
    view = lg[shift:shift + rows * ld].view(rows, ld)
    view[:, :vocab] = dev(logits)
    out = lg.view(-1) if inplace else torch.full_like(lg, 55)
    words = (vocab + 31) // 32
    allow = None
    if mask:
        allow = rng.random((rows, vocab)) < (0.6 if mask == 1 else 3.0 / vocab)
        if mask == 3:
            allow[:] = False
        allow[-1] = False
        bits = np.zeros((rows, words * 32), np.uint8)
        bits[:, :vocab] = allow
        bits[:, vocab:] = 1  # past the vocabulary: never a token
        ad = dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(rows, words))
    items, want, keep, r = [], [], [], 0
    for par in trees:
        h = (rng.random(hist) ** 3 * (vocab + 2)).astype(np.int64)  # some ids past the vocabulary
        bi = (rng.random(nbias) * (vocab + 2)).astype(np.int64)
        if nbias > 3:
            bi[1] = bi[0]
        bv = rng.integers(-2**20, 2**20, nbias)
        if nbias > 5:
            bv[:2] = I32_MAX
        rep, freq, pres = int(rng.integers(1, 3 * 65536)), int(rng.integers(-2**17, 2**17)), int(rng.integers(-2**17, 2**17))
        if extreme:
            freq, pres = I32_MAX, I32_MIN
        hd, bid, bvd = dev(h.astype(np.int32)), dev(bi.astype(np.int32)), dev(bv.astype(np.int32))
        keep += [hd, bid, bvd]
        tok = [int(rng.integers(0, vocab + 1)) if rng.random() < 0.9 else R.NO_TOKEN for _ in par]
        for j, p in enumerate(par):
            items.append(dict(logits=lg.data_ptr() + 4 * (shift + r * ld),
                              out=out.data_ptr() + 4 * (shift + r * ld) if write else 0,
                              allow=ad[r].data_ptr() if mask else 0, history=hd.data_ptr(), history_len=hist,
                              bias_ids=bid.data_ptr(), bias_values=bvd.data_ptr(), n_bias=nbias, repetition=rep,
                              frequency=freq, presence=pres, parent=r - j + p if p >= 0 else -1, token=tok[j]))
            count = {}
            for t in list(h) + [tok[x] for x in R.path_of(par, j)]:
                count[int(t)] = count.get(int(t), 0) + 1
            want.append(R.rules_row(logits[r], count, rep, freq, pres, [(int(a), int(b)) for a, b in zip(bi, bv)],
                                    allow[r] if mask else None))
            r += 1
    tokens = torch.full((rows,), 9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rdet.det_logits_rules(rdet.logit_rows(items), vocab, tokens.data_ptr())
    torch.cuda.synchronize()
    got = tokens.cpu().numpy().view(np.uint32)
    assert [int(t) for t in got] == [w[1] for w in want]
    if write:
        o = out[shift:shift + rows * ld].view(rows, ld).cpu().numpy()
        for x, w in zip(o, want):
            assert np.array_equal(x[:vocab], w[0])
            assert (x[vocab:] == (0 if inplace else 55)).all()
    elif not inplace:
        assert (out == 55).all()


@pytest.mark.parametrize("vocab", [1, 31, 33, 97, 4099, 16384, 16385, 40000])
@pytest.mark.parametrize("hist,nbias,mask,write", [
    (0, 0, 0, True), (0, 0, 0, False), (50, 0, 0, True), (50, 9, 1, True), (0, 7, 2, True), (300, 20, 2, False),
    (5, 3, 3, True)])
def test_logit_rules(vocab, hist, nbias, mask, write):
    rng = np.random.default_rng(vocab * 3 + hist + nbias)
    rules_case(rng, vocab, [random_tree(rng, 4), [-1], random_tree(rng, 3, roots=True)], hist, nbias, mask, write)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("inplace", [False, True])
def test_logit_rules_unaligned_and_in_place(shift, inplace):
    rng = np.random.default_rng(shift)
    rules_case(rng, 5003, [random_tree(rng, 3)], 40, 6, 1, True, inplace=inplace, shift=shift)


def test_logit_rules_in_place_aligned():
    rules_case(np.random.default_rng(4), 4096, [random_tree(np.random.default_rng(4), 5)], 60, 8, 1, True, inplace=True)


def test_logit_rules_extremes():
    # values and penalties at the type's limits: every saturation
    for seed in range(4):
        rng = np.random.default_rng(seed)
        rules_case(rng, 700, [random_tree(rng, 4)], 900, 12, seed % 3, True, extreme=True)


def test_logit_rules_many_rows_and_trees():
    # more rows than one launch takes; a tree is never split
    rng = np.random.default_rng(6)
    trees = [random_tree(rng, int(rng.integers(1, 65))) for _ in range(14)]
    rules_case(rng, 97, trees, 10, 2, 1, True)


@pytest.mark.parametrize("vocab,hist,nbias,mask,write,inplace,extreme", [
    (70004, 500, 30, 1, True, False, False), (70004, 500, 30, 1, True, True, False), (66000, 0, 0, 2, False, False, False),
    (70001, 300, 40, 3, True, False, False), (131072, 40000, 20, 0, True, True, False), (70004, 900, 12, 2, True, False, True)])
def test_logit_rules_wide_vocabularies(vocab, hist, nbias, mask, write, inplace, extreme):
    # rows whose CTAs stream and compute side by side; 40000 ids are more than a table holds
    rng = np.random.default_rng(vocab + hist)
    rules_case(rng, vocab, [random_tree(rng, 7), random_tree(rng, 4, roots=True)], hist, nbias, mask, write, inplace=inplace,
               extreme=extreme)


def test_logit_rules_ties_and_lowest_value():
    # all equal: the lowest allowed index; all at the type's lowest value: still a token
    for value in (0, I32_MIN, I32_MAX):
        v = 70000
        lg = torch.full((v,), value, dtype=torch.int32, device="cuda")
        allow = np.zeros((v + 31) // 32 * 32, np.uint8)
        allow[[40001, 69999, 50]] = 1
        ad = dev(np.packbits(allow, bitorder="little").view(np.int32))
        tok = torch.zeros(2, dtype=torch.int32, device="cuda")
        rdet.det_logits_rules(rdet.logit_rows([dict(logits=lg.data_ptr()), dict(logits=lg.data_ptr(), allow=ad.data_ptr())]),
                              v, tok.data_ptr())
        torch.cuda.synchronize()
        assert tok.tolist() == [0, 50]


def test_logit_rules_no_rows():
    rdet.det_logits_rules(rdet.logit_rows([]), 10, 0)


# ---------------------------------------------------------------------------
# accepted rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("d", [1, 2, 16, 30, 256, 512])
def test_tree_commit(d, own, shift):
    rng = np.random.default_rng(d + own)
    kept, moves, paths, want = [], [], [], []
    for s in range(3):
        n = int(rng.integers(1, 65))
        path = sorted(rng.choice(n, size=int(rng.integers(0, min(n, 9) + 1)), replace=False).tolist())
        paths.append(path)
        for layer in range(3):
            kv = 1 + layer
            ctx = int(rng.integers(0, 20))
            cap = ctx + n + 2
            a = rng.integers(I32_MIN, I32_MAX + 1, (kv, cap, d), dtype=np.int64).astype(np.int32)
            t = torch.zeros(a.size + shift, dtype=torch.int32, device="cuda")
            t[shift:] = dev(a.reshape(-1))
            p = t.data_ptr() + 4 * shift
            if own:
                b = rng.integers(I32_MIN, I32_MAX + 1, (kv, n + 1, d), dtype=np.int64).astype(np.int32)
                bt = torch.zeros(b.size + shift, dtype=torch.int32, device="cuda")
                bt[shift:] = dev(b.reshape(-1))
                kept.append(bt)
                it = dict(draft=bt.data_ptr() + 4 * shift, draft_cap=n + 1)
            else:
                b = a[:, ctx:].copy()
                it = dict(draft=p + ctx * d * 4, draft_cap=cap)
            w = a.copy()
            for i, x in enumerate(path):
                w[:, ctx + i] = b[:, x]
            kept.append(t)
            want.append((t, w))
            moves.append(dict(cache=p, cap=cap, kv_heads=kv, head_dim=d, context=ctx, path=s, **it))
    rdet.det_tree_commit(rdet.tree_moves(moves, paths))
    torch.cuda.synchronize()
    for t, w in want:
        assert np.array_equal(t[shift:].cpu().numpy().reshape(w.shape), w)
        assert (t[:shift] == 0).all()


def test_tree_commit_many_moves():
    # more moves and paths than one launch takes
    rng = np.random.default_rng(1)
    n, moves = 700, []
    a = rng.integers(-9999, 9999, (n, 2, 12, 4)).astype(np.int32)
    b = rng.integers(-9999, 9999, (n, 2, 5, 4)).astype(np.int32)
    ad, bd = dev(a), dev(b)
    paths = [sorted(rng.choice(5, size=i % 4, replace=False).tolist()) for i in range(n)]
    for i in range(n):
        moves.append(dict(cache=ad[i].data_ptr(), draft=bd[i].data_ptr(), cap=12, draft_cap=5, kv_heads=2, head_dim=4,
                          context=i % 8, path=i))
        for j, x in enumerate(paths[i]):
            a[i, :, i % 8 + j] = b[i, :, x]
    rdet.det_tree_commit(rdet.tree_moves(moves, paths))
    torch.cuda.synchronize()
    assert np.array_equal(ad.cpu().numpy(), a)


def test_tree_attention_many_tiles_back_to_back():
    # many key tiles per block and calls that overlap at their ends: a block
    # whose warps drift apart must not miss a barrier's phase (it would wait
    # out its bound of a second)
    import time
    n, ctx, d = 64, 12000, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    k = (torch.randn((8, ctx + n, d), generator=gen, device="cuda") * 65536).to(torch.int32)
    q = (torch.randn((n, 32, d), generator=gen, device="cuda") * 9000).to(torch.int32)
    s = rdet.tree_seqs([dict(k_cache=k.data_ptr(), v_cache=k.data_ptr(), cap=ctx + n, context=ctx,
                             k_tree=k.data_ptr() + ctx * d * 4, v_tree=k.data_ptr() + ctx * d * 4, tree_cap=ctx + n,
                             parents=[i - 1 for i in range(n)])])
    need = rdet.det_attention_tree_workspace(s, 32, 8, d, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    outs = [torch.zeros((n, 32, d), dtype=torch.int32, device="cuda") for _ in range(2)]
    rdet.det_attention_tree(s, q.data_ptr(), 32, 8, d, 0, outs[0].data_ptr(), ws.data_ptr(), need)
    torch.cuda.synchronize()
    t = time.monotonic()
    for _ in range(150):
        rdet.det_attention_tree(s, q.data_ptr(), 32, 8, d, 0, outs[1].data_ptr(), ws.data_ptr(), need)
    torch.cuda.synchronize()
    assert time.monotonic() - t < 0.9
    assert torch.equal(outs[0], outs[1])


def test_logit_rules_every_token_special():
    # more special and biased tokens in a tile than its lists hold
    rng = np.random.default_rng(12)
    vocab = 9000
    lg = rng.integers(-2**20, 2**20, vocab).astype(np.int32)
    hist = np.concatenate([rng.permutation(vocab)[:6000], rng.integers(0, vocab, 9000)]).astype(np.int32)
    ids = np.concatenate([rng.permutation(vocab)[:5000], rng.integers(0, vocab, 300)]).astype(np.int32)
    val = rng.integers(-2**20, 2**20, ids.size).astype(np.int32)
    ld, hd, idd, vd = dev(lg), dev(hist), dev(ids), dev(val)
    out = torch.zeros(vocab, dtype=torch.int32, device="cuda")
    tok = torch.zeros(1, dtype=torch.int32, device="cuda")
    rdet.det_logits_rules(rdet.logit_rows([dict(
        logits=ld.data_ptr(), out=out.data_ptr(), history=hd.data_ptr(), history_len=hist.size, bias_ids=idd.data_ptr(),
        bias_values=vd.data_ptr(), n_bias=ids.size, repetition=80000, frequency=1234, presence=777, token=3)]),
        vocab, tok.data_ptr())
    torch.cuda.synchronize()
    count = {}
    for t in list(hist) + [3]:
        count[int(t)] = count.get(int(t), 0) + 1
    want, best = R.rules_row(lg, count, 80000, 1234, 777, [(int(a), int(b)) for a, b in zip(ids, val)], None)
    assert np.array_equal(out.cpu().numpy(), want) and tok.item() == best
