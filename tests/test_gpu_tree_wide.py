"""The tree attention's wide forms against the oracle: blocks of 64 query rows
with many chunks of dims, many key tiles a CTA and values split over CTAs; and
calls that overlap on two streams.  The oracle checks a sample of the nodes.
Whole numbers: no tolerance."""
import numpy as np
import pytest

import draft_ref as R
import oracle as O
from helpers import rdet
from test_gpu_draft_ops import Case, random_tree
from tree_shapes import WIDE

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def sample(rng, n, most):
    return sorted({0, n - 1, *(int(x) for x in rng.integers(0, n, most))})


def check(case, got, window, rng, most=4):
    """Some nodes of every tree, all heads, against the oracle."""
    at, g = 0, case.heads // case.kv
    for k, v, kt, vt, c, par in case.parts:
        for i in sample(rng, len(par), most):
            path = R.path_of(par, i)
            for kvh in range(case.kv):
                keys = np.concatenate([k[kvh, :c], kt[kvh, path]])
                vals = np.concatenate([v[kvh, :c], vt[kvh, path]])
                if window:
                    keys, vals = keys[-window:], vals[-window:]
                keys, vals = np.ascontiguousarray(keys), np.ascontiguousarray(vals)
                for h in range(kvh * g, (kvh + 1) * g):
                    assert np.array_equal(got[at + i, h], O.attention_one(case.q[at + i, h], keys, vals)), (c, i, h)
        at += len(par)


@pytest.mark.parametrize("name", sorted(WIDE))
@pytest.mark.parametrize("kind", ["norm", "wide", "edge"])
def test_wide_blocks(name, kind):
    ctxs, nodes, heads, kv, d, window = WIDE[name]
    rng = np.random.default_rng(sum(ctxs) + d + len(kind))
    c = Case(rng, ctxs, [random_tree(rng, n, roots=n % 2 == 1) for n in nodes], heads, kv, d, kind,
             qscale=8 if kind == "norm" else None, own=d % 3 == 0)
    got = c.run(window)
    rdet.det_status()
    check(c, got, window, rng, most=3 if len(ctxs) == 1 else 1)


class Call:
    """A case's buffers on the device, prepared before any launch."""

    def __init__(self, case, window):
        self.case, self.window = case, window
        self.q = torch.from_numpy(case.q).cuda()
        self.need = rdet.det_attention_tree_workspace(case.seqs, case.heads, case.kv, case.d, window)

    def launch(self, ws, stream):
        c = self.case
        out = torch.empty(c.q.shape, dtype=torch.int32, device="cuda")
        rdet.det_attention_tree(c.seqs, self.q.data_ptr(), c.heads, c.kv, c.d, self.window, out.data_ptr(), ws.data_ptr(),
                                ws.numel(), stream.cuda_stream)
        return out


def test_calls_that_overlap_on_two_streams():
    """Calls of many shapes on two streams without a wait between them, each
    stream's calls sharing one workspace: every one of them is right."""
    rng = np.random.default_rng(21)
    shapes = [([700, 20], [9, 3], 8, 2, 64, 0), ([9000], [64], 8, 2, 512, 0), ([4096], [16], 8, 2, 512, 0),
              ([37], [4], 4, 2, 16, 8), ([4096], [8], 8, 2, 256, 512), ([3000], [64], 8, 2, 128, 0), ([511], [1], 8, 2, 256, 512),
              ([2001], [12], 4, 1, 33, 0)]
    calls = []
    for ctxs, nodes, heads, kv, d, window in shapes:
        c = Case(rng, ctxs, [random_tree(rng, n) for n in nodes], heads, kv, d, "norm", qscale=8)
        calls.append(Call(c, window))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    need = max(c.need for c in calls)
    spaces = [torch.full((need,), 201, dtype=torch.uint8, device="cuda") for _ in streams]
    calls[0].launch(spaces[0], streams[0])  # loads the library's kernels
    torch.cuda.synchronize()
    outs = []
    for r in range(6):
        for i in range(len(calls)):
            for s in range(2):
                k = (i + s * (3 + r)) % len(calls)
                with torch.cuda.stream(streams[s]):
                    outs.append((k, calls[k].launch(spaces[s], streams[s])))
    torch.cuda.synchronize()
    rdet.det_status()
    first = {}
    for k, out in outs:
        got = out.cpu().numpy()
        assert np.array_equal(first.setdefault(k, got), got), shapes[k]
    for k, got in first.items():
        check(calls[k].case, got, calls[k].window, rng, most=2)


def test_many_calls_back_to_back_end_without_a_lost_wait():
    # a warp that misses a barrier's phase waits out its bound and says so
    rng = np.random.default_rng(4)
    c = Case(rng, [12000], [[i - 1 for i in range(64)]], 8, 2, 128, "norm", qscale=8)
    call = Call(c, 0)
    ws = torch.zeros(call.need, dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream()
    outs = [call.launch(ws, s) for _ in range(100)]
    rdet.det_status()
    assert all(torch.equal(outs[0], o) for o in outs)
    check(c, outs[0].cpu().numpy(), 0, rng)


