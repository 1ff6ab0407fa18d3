"""What the readings operators refuse, checked on the host (no GPU needed)."""

import ctypes as C

import pytest
import torch

from sheetsage2_refined_b200 import _lib, ops


def sample_args(**kw):
    a = _lib.SampleArgs(logits=16, logits_stride=8, logits_dtype=_lib.S2R_F32, rows=2, vocab=8, uniforms=16,
                        temperature_all=1.0, top_p_all=1.0, tokens=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), b"NULL"), (dict(uniforms=None), b"NULL"), (dict(tokens=None), b"NULL"),
    (dict(rows=0), b"rows"), (dict(vocab=0), b"vocab"), (dict(rows=65537), b"65536"), (dict(vocab=524289), b"524288"),
    (dict(logits_dtype=3), b"float32"), (dict(logits_stride=-1), b"stride"), (dict(allowed_stride=-8), b"stride"),
    (dict(temperature_all=-0.5), b"temperature"), (dict(temperature_all=float("nan")), b"temperature"),
    (dict(top_p_all=1.5), b"top_p"), (dict(top_p_all=float("nan")), b"top_p"), (dict(min_p_all=-0.1), b"min_p"),
    (dict(top_k_all=-1), b"top_k"),
])
def test_sample_entry_point_refuses(change, word):
    lib = _lib.load()
    assert lib.s2r_sample(C.byref(sample_args(**change)), None) == _lib.S2R_EINVAL
    assert word in lib.s2r_last_error()


def test_sample_refuses_null_arguments():
    lib = _lib.load()
    assert lib.s2r_sample(None, None) == _lib.S2R_EINVAL


def test_sample_wrapper_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample(torch.zeros(2, 8), torch.zeros(2))
