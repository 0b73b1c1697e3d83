"""Grouped key/value heads without kv_heads and without another modifier: k's shape says how many there are."""
import pytest
import torch

from test_attention_masked_gpu import BF16, _qkv, check, ints, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hk", [1, 2, 8])
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("Sq,Skv", [(1, 400), (130, 300)])
def test_kv_heads_by_the_shape_of_k(cuda_device, Hk, head_major, Sq, Skv):
    from npu_ai_b200 import kernels
    from npu_ai_b200.runner import NpuGemm
    q, k, v = _qkv(2, 8, Hk, Sq, Skv, 64, Sq, cuda_device, head_major=head_major)
    ref = oracle(q, k, v, 8, Hk, head_major)
    out = kernels.attention(q, k, v, 8, head_major_in=head_major, head_major_out=head_major, out_dtype=BF16)
    kernels.check_status(cuda_device)
    check(out, *ref, 8, head_major)
    g = NpuGemm(device=cuda_device, verbose=False)
    out = g.attention(q, k, v, 8, skip_reshape=head_major, skip_output_reshape=head_major)
    check(out, *ref, 8, head_major)


def test_a_start_position_alone_is_checked(cuda_device):
    """It changes nothing without a rule that looks at positions, and a bad one is refused all the same."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(2, 4, 4, 20, 30, 64, 1, cuda_device)
    check(kernels.attention(q, k, v, 4, q_start=ints(cuda_device, 3, 7)), *oracle(q, k, v, 4, 4), 4, False)
    with pytest.raises(ValueError, match="q_start"):
        kernels.attention(q, k, v, 4, q_start=torch.zeros(2, device=cuda_device))
    with pytest.raises(ValueError, match="heads"):
        kernels.attention(q, k[..., :192], v[..., :192], 4)
