"""Refusals of the activation GEMM that need no GPU: the C entry checks its arguments before any device call."""
import ctypes

import pytest
import torch

from npu_ai_b200 import _lib, kernels


def _call(activation, m=8, n=8, k=8, ldo=8, out=16, out_dtype=0, bias_dtype=0):
    p = ctypes.c_void_p
    return _lib.call("npub200_gemm_act", p(16), k, m, k, p(16), k, n, None, bias_dtype, activation, None, 0, p(out), ldo,
                     out_dtype, None, 0, 0, None)


@pytest.mark.parametrize("code", [0, -1, 6, 100])
def test_unknown_activation_codes(code):
    with pytest.raises(ValueError, match="activation"):
        _call(code)


@pytest.mark.parametrize("kw", [dict(m=0), dict(n=0), dict(k=-1), dict(ldo=4), dict(out=None), dict(out_dtype=7),
                                dict(bias_dtype=9)])
def test_bad_sizes_and_types(kw):
    with pytest.raises(ValueError):
        _call(1, **kw)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        kernels.gemm(torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16), activation="gelu")


def test_codes_match_the_header():
    import os
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "npu_b200.h")).read()
    codes = {n.lower(): int(v) for n, v in re.findall(r"#define NPUB200_ACT_(\w+) (\d+)", src)}
    assert codes == _lib.ACTIVATIONS
