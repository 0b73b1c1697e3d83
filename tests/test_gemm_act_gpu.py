"""GEMM with bias, activation and residual in its epilogue (npub200_gemm_act) on the B200 against the same formula in
64 bits: out = act(x W^T + bias) + residual.

Tolerance, per element, from the arithmetic and not from a run. Products of bf16 values are exact in f32; summing K of
them in f32 in any order is off by at most K 2^-23 sum|x w| (2^-23: the tensor core may truncate where it aligns). No
activation here is steeper than 1.2. The activation itself: gelu's erf is off by 1.5e-7, the sigmoids by a relative
2^-20 (exp2 and the division at 2^-22 each, the rounding of the argument); both below 2^-19 |y|. The residual add and
the cast round once more, by half a step of f32 and of the output type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ("gelu", "gelu_tanh", "quick_gelu", "silu", "relu")


def _act64(name, y):
    if name == "gelu":
        return 0.5 * y * torch.special.erfc(-y / math.sqrt(2.0))
    if name == "gelu_tanh":
        return y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    if name == "quick_gelu":
        return y * torch.sigmoid(1.702 * y)
    if name == "silu":
        return y * torch.sigmoid(y)
    return y.clamp_min(0.0)


def _case(M, K, N, bias, residual, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K + pad, generator=g).to(torch.bfloat16)[:, :K]
    w = (torch.randn(N, K + pad, generator=g) * 2.0 * K ** -0.5).to(torch.bfloat16)[:, :K]
    b = None if bias is None else torch.randn(N, generator=g).to(bias)
    r = torch.randn(M, N + pad, generator=g).to(torch.bfloat16)[:, :N] if residual else None
    return x, w, b, r


def _check(out, x, w, b, r, act):
    xd, wd = x.double(), w.double()
    y = xd @ wd.t() + (0.0 if b is None else b.double())
    ref = _act64(act, y) + (0.0 if r is None else r.double())
    tol = 1.2 * x.shape[1] * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -19 * y.abs() + 2.0 ** -23 * ref.abs() + 1e-30
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{act}: {float((err / tol).max())} of the tolerance"


def _run(cuda_device, x, w, b, r, act, **kw):
    from npu_ai_b200 import kernels
    dev = [None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=cuda_device).copy_(t)
           for t in (x, w, b, r)]
    out = kernels.gemm(dev[0], dev[1], dev[2], residual=dev[3], activation=act, **kw)
    kernels.check_status(cuda_device)
    return out


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("MKN", [(1, 64, 64), (1, 1280, 5120), (77, 768, 1280), (130, 72, 200), (300, 320, 1288),
                                 (5, 101, 33), (4096, 320, 1280), (64, 5120, 1280)])
def test_activation_with_bias_and_residual(cuda_device, act, MKN):
    """Single rows, ragged tiles, split K (64 x 5120 x 1280), rows TMA cannot address (K = 101)."""
    x, w, b, r = _case(*MKN, torch.bfloat16, True, seed=sum(MKN))
    _check(_run(cuda_device, x, w, b, r, act, out_dtype=torch.bfloat16), x, w, b, r, act)
    x, w, b, r = _case(*MKN, torch.float32, False, seed=sum(MKN) + 1)
    _check(_run(cuda_device, x, w, b, r, act, out_dtype=torch.float32), x, w, b, r, act)


@pytest.mark.parametrize("variant", [64, 96, 128, 160, 192, 256, 1128, 1192, 1256])
def test_every_tile(cuda_device, variant):
    x, w, b, r = _case(333, 328, 600, torch.float32, True, seed=variant)
    for act in ("gelu", "quick_gelu"):
        _check(_run(cuda_device, x, w, b, r, act, out_dtype=torch.bfloat16, variant=variant), x, w, b, r, act)
        _check(_run(cuda_device, x, w, None, None, act, out_dtype=torch.float32, variant=variant), x, w, None, None, act)


@pytest.mark.parametrize("M,K,N,out_dtype", [(700, 728, 387, torch.bfloat16), (700, 728, 387, torch.float32),
                                             (129, 147, 99, torch.bfloat16), (33, 2360, 665, torch.float32),
                                             (513, 3594, 73, torch.bfloat16), (20000, 72, 325, torch.bfloat16)])
def test_rows_that_tma_does_not_address(cuda_device, M, K, N, out_dtype):
    """Odd N: output and residual rows at any 2-byte address; K off a multiple of 8: repacked operands. What lies beside
    the output rows stays as it was, and the residual may be the output."""
    from npu_ai_b200 import kernels
    x, w, b, r = _case(M, K, N, torch.float32, True, seed=M + N)
    for act, res in (("gelu", r), ("silu", None)):
        _check(_run(cuda_device, x, w, b, res, act, out_dtype=out_dtype), x, w, b, res, act)
    buf = torch.full((M + 2, N + 6), 7.0, dtype=torch.bfloat16, device=cuda_device)
    view = buf[1:M + 1, 3:N + 3]
    view.copy_(r)
    out = kernels.gemm(x.to(cuda_device), w.to(cuda_device), b.to(cuda_device), out=view, residual=view, activation="relu")
    kernels.check_status(cuda_device)
    _check(out.contiguous(), x, w, b, r, "relu")
    buf[1:M + 1, 3:N + 3] = 7.0
    assert bool((buf == 7.0).all())


def test_strided_operands_and_in_place_residual(cuda_device):
    """Row strides past the row length for every operand; the residual may be the output itself; columns and rows
    outside the output view stay as they were."""
    from npu_ai_b200 import kernels
    x, w, b, r = _case(200, 96, 120, torch.bfloat16, True, seed=9, pad=8)
    buf = torch.full((203, 128), 7.0, dtype=torch.bfloat16, device=cuda_device)
    buf[:200, :120] = r.to(cuda_device)
    view = buf[:200, :120]
    xd, wd = (torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=cuda_device).copy_(t) for t in (x, w))
    out = kernels.gemm(xd, wd, b.to(cuda_device), out=view, residual=view, activation="silu")
    kernels.check_status(cuda_device)
    assert out.data_ptr() == view.data_ptr()
    _check(out, x, w, b, r, "silu")
    assert bool((buf[200:] == 7.0).all()) and bool((buf[:, 120:] == 7.0).all())


@pytest.mark.parametrize("act", ACTS)
def test_large_and_extreme_values(cuda_device, act):
    """Arguments far out on both sides (the sigmoid's exponent under- and overflows), zero, infinities and NaN: the
    finite ones to tolerance, +inf stays, a NaN in x reaches every output of its row and no other row."""
    y = torch.tensor([-300.0, -90.0, -60.0, -30.0, -10.0, -1.0, -2.0 ** -20, 0.0, 2.0 ** -20, 1.0, 10.0, 90.0, 300.0, 3e38,
                      1.0, 1.0])
    x = torch.zeros(16, 64)
    x[:, 0] = y
    x = x.to(torch.bfloat16)
    w = torch.zeros(64, 64)
    w[:, 0] = 1.0
    w = w.to(torch.bfloat16)
    out = _run(cuda_device, x, w, None, None, act, out_dtype=torch.float32)
    assert bool(torch.isfinite(out).all())
    _check(out, x, w, None, None, act)
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    w[:, 1:] = 0.5
    out = _run(cuda_device, x, w, None, None, act, out_dtype=torch.float32).cpu()
    assert bool(out[3].isnan().all()) and bool((out[7] == float("inf")).all())
    keep = [i for i in range(16) if i not in (3, 7)]
    _check(out[keep], x[keep], w, None, None, act)


def test_captured_into_a_graph_and_on_another_stream(cuda_device):
    x, w, b, r = (None if t is None else t.to(cuda_device) for t in _case(154, 768, 1280, torch.float32, True, seed=4))
    from npu_ai_b200 import kernels
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        y0 = kernels.gemm(x, w, b, out_dtype=torch.bfloat16, residual=r, activation="gelu")
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y1 = kernels.gemm(x, w, b, out_dtype=torch.bfloat16, residual=r, activation="gelu")
    x.copy_(torch.flip(x, (0,)))
    g.replay()
    torch.cuda.synchronize()
    _check(y1, x.cpu(), w.cpu(), b.cpu(), r.cpu(), "gelu")
    y2 = kernels.gemm(x.flip(0).contiguous(), w, b, out_dtype=torch.bfloat16, residual=r, activation="gelu")
    assert torch.equal(y0, y2)  # the same call gives the same bits


def test_runner_linear_with_activation(cuda_device):
    """NpuGemm.linear / matmul_t: resident weights, n-D inputs, numpy out; no activation gives the plain product."""
    from npu_ai_b200.runner import NpuGemm
    g = NpuGemm(verbose=False)
    x, w, b, r = _case(2 * 77, 768, 1280, torch.float32, True, seed=6)
    nw = g.upload_weight(w, layout="nk")
    y = g.linear(x.view(2, 77, 768), nw, b, out_dtype=torch.bfloat16, residual=r.to(cuda_device).view(2, 77, 1280),
                 activation="quick_gelu")
    assert y.shape == (2, 77, 1280)
    _check(y.view(154, 1280), x, w, b, r, "quick_gelu")
    _check(torch.from_numpy(g.linear(x.float().numpy(), nw, b, activation="relu")), x, w, b, None, "relu")
    with pytest.raises(ValueError, match="activation"):
        g.linear(x, nw, b, activation="swish")


def test_refusals(cuda_device):
    from npu_ai_b200 import kernels
    x, w, b, r = (t.to(cuda_device) for t in _case(16, 64, 32, torch.float32, True, seed=2))
    with pytest.raises(ValueError, match="unknown activation"):
        kernels.gemm(x, w, b, activation="tanh")
    with pytest.raises(ValueError, match="residual"):
        kernels.gemm(x, w, b, residual=r[:8], activation="gelu")
    with pytest.raises(ValueError, match="bias"):
        kernels.gemm(x, w, b[:8], activation="gelu")


@pytest.mark.parametrize("act", ACTS)
def test_values_of_every_size(cuda_device, act):
    """One value a row from 2^-60 to 2^100, both signs, and infinities: sums that are those values exactly. For negative
    ones the result falls to 0, which the kernel may miss by 2.8e-8 (30 x 2^-30). A NaN stays in its own place."""
    from npu_ai_b200 import kernels
    v = torch.tensor([s * m * 2.0 ** e for e in range(-60, 101) for m in (1.0, 1.5) for s in (1.0, -1.0)])
    M = v.numel()
    x = torch.zeros(M, 64, dtype=torch.bfloat16)
    x[:, 0] = v.to(torch.bfloat16)
    w = torch.zeros(128, 64, dtype=torch.bfloat16)
    w[:, 0] = 1.0
    y = v.double()[:, None].expand(M, 128)
    out = kernels.gemm(x.to(cuda_device), w.to(cuda_device), activation=act)
    ref = torch.where((y == -float("inf")) | (y < -1e4), 0.0, _act64(act, y))
    assert bool(((out.double().cpu() - ref).abs() <= 2.0 ** -19 * ref.abs() + 2.8e-8 + 1.5e-7 * y.abs().clamp(max=64.0)).all())
    # a bias carries the infinities and the NaN (0 x inf would be a NaN on the way)
    b = torch.zeros(128)
    b[5], b[6], b[7] = float("inf"), float("-inf"), float("nan")
    out = kernels.gemm(torch.zeros_like(x).to(cuda_device), w.to(cuda_device), b.to(cuda_device), activation=act).cpu()
    kernels.check_status(cuda_device)
    assert bool((out[:, 5] == float("inf")).all()) and bool((out[:, 6].abs() <= 2.8e-8).all())
    assert bool(out[:, 7].isnan().all()) and bool((out[:, [i for i in range(128) if i not in (5, 6, 7)]] == 0).all())


@pytest.mark.parametrize("shift", [0, 1])
def test_rows_far_apart(cuda_device, shift):
    """Output and residual rows more than 2^32 bytes from the first to the last, aligned (TMA) and not."""
    from npu_ai_b200 import kernels
    M, K, N, ld = 40, 72, 96, 2 ** 26
    if torch.cuda.mem_get_info(cuda_device)[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    x, w, b, r = _case(M, K, N, torch.float32, True, seed=4)
    big = torch.empty(M * ld, dtype=torch.bfloat16, device=cuda_device)
    out, res = big.as_strided((M, N), (ld, 1), shift), big.as_strided((M, N), (ld, 1), 4096 + shift)
    res.copy_(r)
    kernels.gemm(x.to(cuda_device), w.to(cuda_device), b.to(cuda_device), out=out, residual=res, activation="gelu")
    kernels.check_status(cuda_device)
    _check(out.contiguous(), x, w, b, r, "gelu")


def test_operands_of_the_kernel_before(cuda_device):
    """x, w, bias and residual may each be what the kernel before on the stream has written (launches overlap)."""
    from npu_ai_b200 import kernels
    x, w, b, r = _case(512, 512, 512, torch.float32, True, seed=3)
    xd, wd, bd, rd = (t.to(cuda_device) for t in (x, w, b, r))
    eye = torch.eye(512, dtype=torch.bfloat16, device=cuda_device)
    for _ in range(20):
        w2 = torch.empty_like(wd).fill_(float("nan"))
        kernels.gemm(wd, eye, out=w2)          # w again
        y = kernels.gemm(xd, w2, bd, residual=rd, activation="silu", out_dtype=torch.float32)
        r2 = torch.empty_like(rd).fill_(float("nan"))
        kernels.gemm(rd, eye, out=r2)
        z = kernels.gemm(xd, wd, bd, residual=r2, activation="silu", out_dtype=torch.float32)
        kernels.check_status(cuda_device)
        assert torch.equal(y, z)
    _check(y, x, w, b, r, "silu")
