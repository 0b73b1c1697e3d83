"""The ComfyUI node on the GPU: attention calls with masks and grouped heads reach the masked attention kernel, and
Linear -> activation pairs the GEMM's epilogue. Results against the formulas in 64 bits, at the operators' own
tolerances; calls that stay with the model are its own results, bit for bit."""
import pytest
import torch
import torch.nn.functional as F

from test_attention_masked_gpu import check, oracle

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def runtime(cuda_device):
    from npu_ai_b200 import comfy_nodes as cn
    rt = cn._get_runtime(cuda_device)
    mode, least, tokens = rt.attn.mode, rt.attn.min_tokens, rt.min_tokens
    rt.attn.reset()
    rt.attn.mode, rt.attn.min_tokens, rt.min_tokens, rt.enabled = "auto", 1, 1, True
    try:
        yield rt
    finally:
        rt.release()
        rt.attn.reset()
        rt.attn.mode, rt.attn.min_tokens, rt.min_tokens = mode, least, tokens


def model_attention(q, k, v, heads, mask=None, attn_precision=None, skip_reshape=False, skip_output_reshape=False,
                    scale=None, enable_gqa=False, **kwargs):
    if not skip_reshape:
        d = q.shape[-1] // heads
        q, k, v = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in (q, k, v))
    if mask is not None:
        if mask.dim() == 3:
            mask = mask[:, None]
        if mask.dtype != torch.bool:
            mask = mask.to(q.dtype)
    o = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=scale, enable_gqa=enable_gqa)
    return o if skip_output_reshape else o.transpose(1, 2).flatten(2)


def _call(rt, q, k, v, heads, **kw):
    from npu_ai_b200 import comfy_nodes as cn
    before = rt.attn.fused_calls, rt.attn.model_calls
    y = cn._gpu_attention_override(model_attention, q, k, v, heads, **kw)
    ref = model_attention(q, k, v, heads, **kw)
    assert y.shape == ref.shape and y.dtype == q.dtype
    return y, ref, rt.attn.fused_calls - before[0], rt.attn.model_calls - before[1]


def _check(y, q, k, v, hk, mask, head_major=False, head_major_out=False, scale=None):
    if mask is not None and mask.dtype == torch.float16:
        mask = mask.float()
    check(y, *oracle(q, k, v, 8, hk, head_major, scale=scale, mask=mask), 8, head_major_out)


def _qkv(dev, b, h, hk, tq, tk, d, head_major, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn((b, n, t, d) if head_major else (b, t, n * d), generator=g, device=dev).to(BF16)
            for n, t in ((h, tq), (hk, tk), (hk, tk))]


@pytest.mark.parametrize("dtype", [torch.bool, BF16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(96, 77), (2, 1, 1, 77), (1, 8, 96, 77), (2, 8, 96, 77)])
@pytest.mark.parametrize("head_major", [False, True])
def test_masked_calls_run_the_kernel(runtime, cuda_device, dtype, shape, head_major):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    mask = torch.rand(shape, generator=g, device=cuda_device) < 0.6
    mask[..., 5] = True
    if dtype != torch.bool:
        mask = torch.where(mask, torch.randn(shape, generator=g, device=cuda_device).to(BF16).float(),
                           float("-inf")).to(dtype)
    q, k, v = _qkv(cuda_device, 2, 8, 8, 96, 77, 40, head_major)
    for _ in range(2):
        y, _, fused, model = _call(runtime, q, k, v, 8, mask=mask, skip_reshape=head_major,
                                   skip_output_reshape=head_major)
        assert (fused, model) == (1, 0)
        _check(y, q, k, v, 8, mask, head_major, head_major)
    (key, rec), = runtime.attn.shapes.items()
    assert key[5].endswith("mask") and rec.variant == 0 and list(rec.variant_ms) == [0]


@pytest.mark.parametrize("hk", [1, 2, 8])
def test_grouped_heads_run_the_kernel(runtime, cuda_device, hk):
    q, k, v = _qkv(cuda_device, 2, 8, hk, 64, 200, 64, True)
    mask = torch.ones(64, 200, dtype=torch.bool, device=cuda_device).tril(136)
    for m in (None, mask):
        y, _, fused, model = _call(runtime, q, k, v, 8, mask=m, skip_reshape=True, enable_gqa=True, scale=0.2)
        assert (fused, model) == (1, 0)
        _check(y, q, k, v, hk, m, True, False, 0.2)
    assert len(runtime.attn.shapes) == 2


def test_rows_without_a_key_are_zero(runtime, cuda_device):
    q, k, v = _qkv(cuda_device, 1, 8, 8, 64, 64, 64, False)
    mask = torch.zeros(64, 64, device=cuda_device)
    mask[7] = float("-inf")
    y, _, fused, _ = _call(runtime, q, k, v, 8, mask=mask)
    assert fused == 1 and bool((y[:, 7] == 0).all())
    _check(y, q, k, v, 8, mask)


def test_masked_calls_that_stay_with_the_model(runtime, cuda_device):
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 40, False)
    three = torch.zeros(2, 64, 64, device=cuda_device)
    y, ref, fused, model = _call(runtime, q, k, v, 8, mask=three)
    assert (fused, model) == (0, 1) and torch.equal(y, ref)
    assert any(r.model_reason == "masked attention" for r in runtime.attn.shapes.values())
    # the unmasked call of the same shape still runs the fused kernel and its variants
    y, ref, fused, model = _call(runtime, q, k, v, 8)
    assert (fused, model) == (1, 0) and len(runtime.attn.shapes[(2, 64, 64, 8, 40)].variant_ms) > 1


def test_runner_attention_takes_the_masking_keywords(cuda_device):
    from npu_ai_b200.runner import NpuGemm
    g = NpuGemm(device=cuda_device, verbose=False)
    q, k, v = _qkv(cuda_device, 2, 8, 2, 33, 100, 64, False)
    lens = torch.tensor([100, 61], dtype=torch.int32)  # on the host: the runner brings it over, like its operands
    out = g.attention(q.cpu(), k, v, 8, kv_heads=2, causal=True, kv_lens=lens, softcap=10.0)
    assert out.dtype == torch.float32 and g.stats["attn_fused_calls"] == 1
    check(out, *oracle(q, k, v, 8, 2, causal=True, kv_lens=lens.to(cuda_device), softcap=10.0), 8, False)
    with pytest.raises(ValueError, match="group"):
        g.attention(q, k, v, 8, kv_heads=2, group=object())
    with pytest.raises(TypeError):
        g.attention(q, k, v, 8, sliding=4)


@pytest.mark.parametrize("act,ref_act", [
    (lambda: torch.nn.GELU(), F.gelu), (lambda: torch.nn.GELU(approximate="tanh"), lambda y: F.gelu(y, approximate="tanh")),
    (lambda: torch.nn.SiLU(), F.silu), (lambda: torch.nn.ReLU(inplace=True), F.relu)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_feed_forward_without_gating(runtime, cuda_device, act, ref_act, dtype):
    """net = [[Linear, activation], Dropout, Linear], as feed-forward blocks without gating nest it."""
    from test_gemm_act_gpu import _check as check_act
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Sequential(torch.nn.Linear(320, 1280), act()), torch.nn.Dropout(0.0),
                              torch.nn.Linear(1280, 320)).to(cuda_device, dtype).eval()
    own = net[0].forward
    runtime.take_over(net, 320, ())
    assert runtime.act_modules == {id(net[0])}
    x = torch.randn(2, 100, 320, device=cuda_device).to(BF16).to(dtype)
    with torch.no_grad():
        u, y = net[0](x), net(x)
        assert u.dtype == y.dtype == dtype and y.shape == x.shape
        # the intermediate against the formula, at the operator's own tolerance
        name = {"GELU": "gelu", "SiLU": "silu", "ReLU": "relu"}[type(net[0][1]).__name__]
        if getattr(net[0][1], "approximate", "none") == "tanh":
            name = "gelu_tanh"
        w = net[0][0].weight.detach().to(BF16).cpu()
        check_act(u.reshape(-1, 1280), x.reshape(-1, 320).to(BF16).cpu(), w, net[0][0].bias.detach().float().cpu(), None, name)
        # short inputs and a runtime that is off keep the modules' own forwards
        runtime.min_tokens = 64
        calls = runtime.gemm.stats["calls"]
        few = net[0](x[:, :3])
        assert runtime.gemm.stats["calls"] == calls and torch.equal(few, ref_act(F.linear(x[:, :3], net[0][0].weight,
                                                                                        net[0][0].bias)))
        runtime.enabled = False
        off = net[0](x)
        assert runtime.gemm.stats["calls"] == calls and torch.equal(off, ref_act(F.linear(x, net[0][0].weight,
                                                                                        net[0][0].bias)))
    runtime.release()
    assert net[0].forward == own and not runtime.act_modules
