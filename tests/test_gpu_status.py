"""A pipeline wait that gives up is reported: by rdet_det_status to callers of
the kernel-level entry points, and by the calls of a context.  No wait is made
to run out here: the host sets the words that such a kernel sets."""
import ctypes as C

import numpy as np
import pytest

from helpers import mini_config, rdet

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

RDET_E_CUDA = -4


class Words(C.Structure):
    _fields_ = [("w", C.c_void_p * 5)]


def words():
    f = getattr(rdet.lib(), "_ZN4rdet11error_wordsEv")
    f.restype, f.argtypes = Words, []
    return list(f().w)


def set_word(p):
    torch.cuda.synchronize()
    assert C.CDLL("libcuda.so.1").cuMemsetD32_v2(C.c_uint64(p), 1, C.c_size_t(1)) == 0
    torch.cuda.synchronize()


@pytest.fixture(scope="module")
def model():
    return rdet.Model.synthetic(mini_config(), seed=4, width=16, max_prefill=16)


def test_status_is_clean_after_calls(model):
    s = model.new_sequence(16)
    s.prefill([1, 2, 3])
    rdet.tree_decode(model, [s], [[5, 6, 7]], [[-1, 0, 0]])
    rdet.det_status()
    rdet.det_status(torch.cuda.current_stream().cuda_stream)
    rdet.det_status(torch.cuda.Stream().cuda_stream)


@pytest.mark.parametrize("i", range(5))
def test_every_word_is_reported_once(model, i):
    at = words()
    assert len({p for p in at if p}) == 5
    set_word(at[i])
    with pytest.raises(rdet.RdetError) as e:
        rdet.det_status()
    assert e.value.code == RDET_E_CUDA and "pipeline wait" in e.value.msg
    rdet.det_status()


@pytest.mark.parametrize("i", range(5))
def test_a_context_reports_it_too(model, i):
    s, r = model.new_sequence(16), model.new_sequence(16)
    for x in (s, r):
        x.prefill([1, 2, 3])
    set_word(words()[i])
    with pytest.raises(rdet.RdetError) as e:
        s.decode(4)
    assert e.value.code == RDET_E_CUDA and "pipeline wait" in e.value.msg
    r.decode(4)  # cleared
    assert np.array_equal(s.read(rdet.BUF_LOGITS), r.read(rdet.BUF_LOGITS))


def test_a_token_out_of_range_is_told_apart(model):
    with pytest.raises(rdet.RdetError) as e:
        model.new_sequence(16).prefill([97])
    assert "out of bounds" in e.value.msg
    rdet.det_status()
