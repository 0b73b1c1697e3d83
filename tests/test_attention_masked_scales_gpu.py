"""Scales and caps at the ends of what the masked attention takes, on the B200; tolerances of test_attention_masked_gpu.py."""
import pytest
import torch

from test_attention_masked_gpu import _qkv, check, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_slopes", [False, True])
@pytest.mark.parametrize("softcap,scale", [(1e30, 1e-7), (1e-30, 5e7), (1e-20, 1e-30), (1e10, 1e-25)])
def test_scales_far_from_the_cap(cuda_device, softcap, scale, with_slopes):
    """Scores of at most the cap or far below 1, so every key weighs the same: the average of V, with a slope of 0 (the
    kernel for any modifier) as without. P is 1 exactly, the sums are f32: 2^-16 of the average of |V|."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(2, 4, 2, 70, 300, 64, 3, cuda_device)
    slopes = torch.zeros(4, device=cuda_device) if with_slopes else None
    if softcap > 1.0:  # scale q.k is far below 2^-16
        assert scale * 64 * 36 < 1e-3
    out = kernels.attention(q, k, v, 4, scale=scale, softcap=softcap, slopes=slopes, kv_heads=2).double()
    kernels.check_status(cuda_device)
    w = v.double().unflatten(-1, (2, 64)).repeat_interleave(2, 2).flatten(2)
    near = scale * 64 * 36 if softcap > 1.0 else 0.0
    tol = (2.0 ** -16 + 2.0 ** -8 * (near > 2.0 ** -9) + 2.0 * near) * w.abs().mean(1, keepdim=True)
    assert bool(((out - w.mean(1, keepdim=True)).abs() <= tol).all())


def test_refused_scales(cuda_device):
    from npu_ai_b200 import kernels
    q, k, v = _qkv(1, 2, 2, 5, 30, 64, 3, cuda_device)
    for softcap, scale in ((1e30, 1e-16), (1e-30, 1e9), (None, 3e38)):
        with pytest.raises(ValueError, match="scale"):
            kernels.attention(q, k, v, 2, causal=True, scale=scale, softcap=softcap)


def test_cap_with_a_scale_of_its_own(cuda_device):
    from npu_ai_b200 import kernels
    q, k, v = _qkv(2, 4, 2, 70, 300, 64, 5, cuda_device, 3.0)
    for softcap, scale in ((2.0, 1.5), (1e-3, 0.01), (1e4, 0.5)):
        kw = dict(softcap=softcap, scale=scale, causal=True)
        out = kernels.attention(q, k, v, 4, kv_heads=2, **kw)
        kernels.check_status(cuda_device)
        check(out, *oracle(q, k, v, 4, 2, **kw), 4, False)
