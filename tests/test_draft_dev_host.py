"""The tree attention's softmax helpers (det_dev.cuh) compiled for the host,
against the forms they replace: every exp term there is, and weights at
random, at ties and at the ends."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from helpers import ROOT

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host():
    out = os.path.join(tempfile.mkdtemp(prefix="draft-dev-"), "draft_dev.so")
    r = subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-DRDET_HD=static inline", "-I",
                        os.path.join(ROOT, "raster-inference_b200", "csrc"),
                        os.path.join(HERE, "draft_dev_host.cpp"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    L = C.CDLL(out)
    for name, args in (("requantize_random", [C.c_uint64, C.c_int64]), ("digits_random", [C.c_uint64, C.c_int64]),
                        ("exp_all", [C.c_int32]), ("exp_second", []), ("weights_random", [C.c_uint64, C.c_int64]),
                       ("weights_ties", [C.c_uint64, C.c_int64]), ("weights_open", [C.c_uint64, C.c_int64]), ("weights_one", [C.c_int64])):
        getattr(L, name).argtypes, getattr(L, name).restype = args, C.c_int64
    return L


@pytest.mark.parametrize("top", [0, 2**31 - 1, -2**31 + (16 << 16), -2**31 + 12345, 777777])
def test_every_exp_term(host, top):
    assert host.exp_all(top) == 0


def test_the_code_of_one_is_free(host):
    assert host.exp_second() <= 2**32 - 2**15


@pytest.mark.parametrize("seed", range(4))
def test_weights(host, seed):
    assert host.weights_random(seed * 10**9, 2_000_000) == 0
    assert host.weights_ties(seed * 10**9, 400_000) == 0


def test_rounding_without_branches(host):
    assert host.requantize_random(5, 2_000_000) == 0
    assert host.digits_random(7 * 10**12, 4_000_000) == 0


def test_weights_of_a_lone_key(host):
    assert host.weights_one(300_000) == 0


def test_few_weights_are_left_open(host):
    # 12 of 2^16 positions between two halves
    assert host.weights_open(7, 1_000_000) < 400
