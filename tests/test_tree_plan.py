"""What the tree attention launches for the shapes that its tests name, from the
library's own plan (no GPU): a rule that changes must not take a form out of
the tests' sight."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from helpers import ROOT, rdet
from tree_shapes import WIDE

HERE = os.path.dirname(os.path.abspath(__file__))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def plan():
    out = os.path.join(tempfile.mkdtemp(prefix="tree-plan-"), "plan.so")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "raster-inference_b200", "csrc"),
                        "-I", os.path.join(CUDA, "include"), os.path.join(HERE, "plan_host.cpp"), rdet.LIB_PATH,
                        "-Wl,-rpath," + os.path.dirname(rdet.LIB_PATH), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    f = C.CDLL(out).plan
    f.restype = C.c_longlong

    def call(ctxs, nodes, heads, kv, d, window):
        res = (C.c_int * 6)()
        n = len(ctxs)
        assert f(n, (C.c_int * n)(*ctxs), (C.c_int * n)(*nodes), heads, kv, d, window, res) > 0
        return dict(zip(("rows", "tiles", "splits", "chunks", "qk", "pv"), res))
    return call


@pytest.mark.parametrize("name", sorted(WIDE))
def test_wide_shapes_take_64_rows_many_tiles_and_splits(plan, name):
    ctxs, nodes, heads, kv, d, window = WIDE[name]
    p = plan(*WIDE[name])
    assert p["rows"] == 64 and p["tiles"] >= 2 and p["splits"] >= 2
    assert (d + 63) // 64 >= 4 and (d + 127) // 128 >= 2


def test_the_rule_of_64_rows(plan):
    # 148 score tiles of 64-row blocks, and more than 32 rows
    at = lambda ctx, nodes, heads=8: plan([ctx], [nodes], heads, 2, 512, 0)["rows"]  # noqa: E731
    assert at(4096, 16) == 32 and at(16384, 16) == 64
    assert at(128 * 74 - 16, 16) == 64 and at(128 * 73 - 16, 16) == 32
    assert at(100000, 8) == 32 and at(100000, 4) == 16 and at(100000, 9) == 64
