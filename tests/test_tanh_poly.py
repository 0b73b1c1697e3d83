"""The capped scores' polynomial (kTanhRatio in attention_masked.cuh): its constants are the ones the committed fit
produces, and evaluated in f32 the way the kernel does it, its relative error stays below 1e-6 on the kernel's range."""
import importlib.util
import pathlib
import re

import numpy as np

CSRC = pathlib.Path(__file__).resolve().parents[1] / "npu_ai_b200" / "csrc"


def _fit_module():
    spec = importlib.util.spec_from_file_location("fit_tanh_poly", CSRC / "fit_tanh_poly.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _kernel_coeffs():
    src = (CSRC / "attention_masked.cuh").read_text()
    body = src[src.index("float kTanhRatio[6]"):]
    body = body[:body.index("};")]
    return np.float32([float(v) for v in re.findall(r"(-?[0-9]\.[0-9]+e[-+][0-9]+)f", body)])


def test_kernel_constants_match_fit():
    mod = _fit_module()
    c, err = mod.fit()
    assert err < 6e-7
    np.testing.assert_allclose(_kernel_coeffs(), c, rtol=3e-4)


def test_f32_evaluation_error_bound():
    mod = _fit_module()
    c, _ = mod.fit()
    y = np.concatenate([np.linspace(1e-30, 1.0, 1_000_001), 2.0 ** -np.arange(0, 100)]).astype(np.float32)
    rel = np.abs(mod.poly_f32(y, c).astype(np.float64) / np.tanh(y.astype(np.float64)) - 1.0)
    assert rel.max() < 1e-6, rel.max()
    np.testing.assert_array_equal(mod.poly_f32(-y, c), -mod.poly_f32(y, c))
