"""The GEMM with an activation over many rows and a long K, the compute-bound feed-forward product, on the B200: the ring of
operand stages goes round many times, in CTA pairs too. Against the formula in 64 bits on the GPU; tolerances of
test_gemm_act_gpu.py."""
import pytest
import torch

from test_gemm_act_gpu import _act64, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N,variant", [(4096, 1280, 5120, 0), (2000, 5120, 1280, 0), (8200, 1288, 2568, 0),
                                           (1024, 4096, 4096, 0)] +
                         [(1000, 2048, 1000, v) for v in (64, 96, 128, 160, 192, 256, 1128, 1192, 1256)])
@pytest.mark.parametrize("act,residual,out_dtype", [("gelu", False, torch.bfloat16), ("silu", True, torch.bfloat16),
                                                    ("gelu_tanh", True, torch.float32)])
def test_many_rows_and_a_long_k(cuda_device, M, K, N, variant, act, residual, out_dtype):
    from npu_ai_b200 import kernels
    x, w, b, r = (t if t is None else t.to(cuda_device) for t in _case(M, K, N, torch.float32, residual, seed=M + K))
    out = kernels.gemm(x, w, b, residual=r, activation=act, out_dtype=out_dtype, variant=variant)
    kernels.check_status(cuda_device)
    for at in range(0, M, 2048):
        rows = slice(at, at + 2048)
        xd, wd = x[rows].double(), w.double()
        y = xd @ wd.t() + b.double()
        ref = _act64(act, y) + (0.0 if r is None else r[rows].double())
        tol = 1.2 * K * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -19 * y.abs() + 2.0 ** -23 * ref.abs() + 1e-30
        if out_dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (ref.abs() + tol)
        assert bool(((out[rows].double() - ref).abs() <= tol).all())
