"""Copies and memsets of the runtime are ordered with the context's stream.
That stream is non-blocking: a copy on the legacy default stream neither
waits for it nor is waited for by it, so the runtime makes none."""
import os
import re

from helpers import ROOT


def test_no_copy_reads_back_on_the_default_stream():
    text = open(os.path.join(ROOT, "raster-inference_b200", "csrc", "runtime.cu")).read()
    code = re.sub(r"//[^\n]*", "", text)
    assert "cudaStreamNonBlocking" in code
    assert not re.findall(r"cudaMemcpy\([^;]*DeviceToHost\)", code)


def test_no_copy_or_memset_on_the_default_stream():
    text = open(os.path.join(ROOT, "raster-inference_b200", "csrc", "runtime.cu")).read()
    code = re.sub(r"//[^\n]*", "", text)
    assert not re.findall(r"cudaMemcpy\(|cudaMemset\(|cudaMemcpy2D\(|cudaMemcpyToSymbol\(", code)


def test_error_words_are_not_copied_one_by_one():
    # a symbol copy runs on the legacy default stream and waits for itself
    csrc = os.path.join(ROOT, "raster-inference_b200", "csrc")
    for name in sorted(os.listdir(csrc)):
        if name.endswith(".cu"):
            code = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
            assert not re.findall(r"cudaMemcpy(?:From|To)Symbol\(", code), name


def test_overlapping_grids_load_coherently():
    # kernels that may be resident while the grid before them writes their inputs:
    # the non-coherent path wants data that nobody writes while the kernel lives
    csrc = os.path.join(ROOT, "raster-inference_b200", "csrc")
    for name in ("draft_ops.cu", "tree_attn.cu"):
        code = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        assert "griddepcontrol.wait" in code
        assert not re.findall(r"__ldg\(|ld\.global\.nc|__restrict__", code), name
