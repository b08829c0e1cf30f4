"""The buffers that a context replaces as its calls grow (dev_buf.h), compiled
for the host with an allocator that fails: a request that fails leaves what
was there, under its own size."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import pytest

from helpers import ROOT

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(ROOT, "raster-inference_b200", "csrc")


@pytest.fixture(scope="module")
def host():
    out = os.path.join(tempfile.mkdtemp(prefix="dev-buf-"), "dev_buf.so")
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, os.path.join(HERE, "dev_buf_host.cpp"),
                        "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    L = C.CDLL(out)
    L.workspace.argtypes = [C.c_uint64, C.c_uint64]
    L.passes.argtypes = [C.c_int, C.c_uint64]
    L.growing.argtypes = [C.c_int, C.c_int]
    return L


def runtime():
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "runtime.cu")).read())


@pytest.mark.parametrize("first", range(4))
@pytest.mark.parametrize("second", range(4))
def test_a_failed_workspace_keeps_its_size(host, first, second):
    assert host.workspace(first, second) == 0


def test_the_tree_workspace_is_reserved_before_the_pass():
    # nothing is allocated between the layers of a pass that has begun
    code = runtime()
    body = code[code.index("static void tree_attention("):]
    body = body[:body.index("\n}\n")]
    assert "dalloc" not in body and "reserve" not in body
    assert "tree.ws_bytes" not in code


@pytest.mark.parametrize("victim", range(7))
def test_a_failed_pass_keeps_the_trees_before_it(host, victim):
    for fail in range(64):
        assert host.passes(victim, fail) == 0, fail


def test_a_pass_takes_its_memory_at_once():
    # tree_decode allocates through reserve_pass alone, which ends the trees before it last
    code = runtime()
    body = code[code.index("static void tree_decode("):]
    body = body[:body.index("\n}\n")]
    assert "dalloc" not in body and "epoch +=" not in body and body.count("reserve_pass(") == 1
    assert not re.search(r"\btr\.(dec_out|logits|pos|rows)\s*=", body[:body.index("reserve_pass(")])


def test_growing_passes_replace_their_buffers_rarely_and_keep_none(host):
    assert 0 < host.growing(4000, 4096) <= 3 * 12
    assert 0 < host.growing(40, 40) <= 3 * 6
