"""The far negative side of the sigmoid activations in the GEMM's epilogue, on the B200, against the formula in 64 bits.

Tolerance, from the arithmetic: y sigmoid(s) = y / (1 + 2^t) with t = -s log2 e in f32. t carries the roundings of its
constants and products, four half steps at most, so the result is off by a relative |t| ln 2 4 2^-24; exp2 and the
reciprocal are within 2^-22 each and two products round. Below 2^-126 f32 has no normal numbers: the power flushes to 0,
which misses up to |y| 2^-126. sum and product of x W^T are exact here (one nonzero product)."""
import math

import pytest
import torch

from test_gemm_act_gpu import _act64

pytestmark = pytest.mark.gpu

LOG2E = math.log2(math.e)


def _t(act, y):
    if act == "gelu_tanh":
        return -2.0 * math.sqrt(2.0 / math.pi) * LOG2E * (y + 0.044715 * y ** 3)
    return -(1.702 if act == "quick_gelu" else 1.0) * LOG2E * y


def _exact(act, y):
    """y 2^-t / (1 + 2^-t), which 64 bits hold on the far side (1 + tanh would cancel)."""
    e = torch.exp2(-_t(act, y).clamp(max=1000.0))
    return torch.where(y < 0, y * e / (1.0 + e), _act64(act, y))


@pytest.mark.parametrize("act", ["silu", "quick_gelu", "gelu_tanh"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(16, 64, 64), (300, 64, 256), (64, 5120, 128)])
def test_far_negative_values(cuda_device, act, out_dtype, M, K, N):
    """Rows and columns of values from 0 to past the last one whose result f32 holds, next to ordinary ones (a value
    shares its reciprocal with three others); split K too."""
    from npu_ai_b200 import kernels
    x = torch.zeros(M, K, dtype=torch.bfloat16)
    x[:, 0] = -torch.linspace(0.0, 1.0, M).to(torch.bfloat16)
    w = torch.zeros(N, K, dtype=torch.bfloat16)
    w[:, 0] = (torch.arange(N) * 37 % 101).float().to(torch.bfloat16) * torch.where(torch.arange(N) % 5 == 3, -1.0, 1.0)
    y = x[:, :1].double() @ w[:, :1].double().t()
    out = kernels.gemm(x.to(cuda_device), w.to(cuda_device), activation=act, out_dtype=out_dtype).double().cpu()
    kernels.check_status(cuda_device)
    ref, t = _exact(act, y), _t(act, y).abs()
    # (ordinary values, t near 0, keep the bound of the other tests)
    tol = ref.abs() * (t * math.log(2.0) * 2.0 ** -22 + 2.0 ** -20) + y.abs() * 2.0 ** -126 + 2.0 ** -19 * torch.where(y > 0, y, 0.0)
    if out_dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    err = (out - ref).abs()
    assert bool((err <= tol).all()), f"{float((err / (tol + 1e-300)).max())} of the tolerance"


@pytest.mark.parametrize("act", ["silu", "quick_gelu", "gelu_tanh"])
def test_values_without_end(cuda_device, act):
    """Past every number that f32 holds the result is 0; -infinity gives 0 as well, +infinity itself, NaN a NaN, and none
    of them reaches its neighbours."""
    from npu_ai_b200 import kernels
    x = torch.zeros(8, 64, dtype=torch.bfloat16).to(cuda_device)
    w = torch.zeros(96, 64, dtype=torch.bfloat16).to(cuda_device)
    b = torch.zeros(96)
    b[::4] = torch.tensor([-1e3, -1e12, -3e38, -math.inf]).repeat(6)
    b[5], b[9], b[13] = math.inf, math.nan, 2.5
    out = kernels.gemm(x, w, b.to(cuda_device), activation=act).cpu()
    kernels.check_status(cuda_device)
    assert bool((out[:, ::4] == 0).all()) and bool((out[:, 5] == math.inf).all()) and bool(out[:, 9].isnan().all())
    ref = float(_act64(act, torch.tensor(2.5, dtype=torch.float64)))
    assert bool(((out[:, 13].double() - ref).abs() <= 2.0 ** -19 * 2.5).all())
    rest = [i for i in range(96) if i % 4 and i not in (5, 9, 13)]
    assert bool((out[:, rest] == 0).all())
