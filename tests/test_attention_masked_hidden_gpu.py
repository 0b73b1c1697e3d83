"""What a mask hides has no say, on the B200: the scores of hidden keys are replaced, not added to, in every form of the
mask."""
import pytest
import torch

from test_attention_masked_gpu import BF16, INF, _qkv, check, ints, oracle

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("shape", ["shared", "own"])
@pytest.mark.parametrize("dtype", [torch.bool, BF16, torch.float32])
@pytest.mark.parametrize("Sq,Skv,variant", [(5, 150, 1), (130, 400, 1), (1, 400, 2), (5, 1500, 24), (300, 1000, 40)])
@pytest.mark.parametrize("cap", [None, 8.0])
def test_scores_of_masked_keys_have_no_say(cuda_device, shape, dtype, Sq, Skv, variant, cap):
    """Keys that the mask hides from every row hold NaN, infinities or values past every cap (V finite); a query of a
    sequence that the mask leaves nothing holds NaN: zeros."""
    from npu_ai_b200 import kernels
    dev, H, Hk = cuda_device, 4, 2
    q, k, v = _qkv(3, H, Hk, Sq, Skv, 64, Skv, dev)
    n = ints(dev, Skv - 20, 67, 0).view(3, 1, 1, 1)
    keep = (torch.arange(Skv, device=dev) < n).expand(3, 1, 1 if shape == "shared" else Sq, Skv).contiguous()
    mask = keep if dtype == torch.bool else torch.where(keep, 0.5, -INF).to(dtype)
    kw = dict(mask=mask, softcap=cap)
    ref = oracle(q, k, v, H, Hk, **kw)
    for fill in (NAN, INF, -INF, 1e30):
        bad = k.clone()
        bad[0, Skv - 20:, ::3], bad[1, 67:], bad[2] = fill, fill, fill
        qn = q.clone()
        qn[2] = NAN
        out = kernels.attention(qn, bad, v, H, variant=variant, **kw)
        kernels.check_status(dev)
        check(out, *ref, H, False)
