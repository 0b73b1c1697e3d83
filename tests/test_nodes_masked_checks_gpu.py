"""The ComfyUI node's first-call check of masked attention and the calls that stay with the model, on the GPU."""
import pytest
import torch

from test_attention_masked_gpu import BF16
from test_nodes_masked_gpu import _call, _check, _qkv, model_attention, runtime  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _plain_model(q, k, v, heads, mask=None, skip_output_reshape=False, **kw):
    """A softmax in f32 of head-major operands, NaN where the mask leaves nothing (what SDPA gives there is its backend's)."""
    n = q.shape[1] // k.shape[1]
    s = q.float() @ k.float().repeat_interleave(n, 1).transpose(-1, -2) * q.shape[-1] ** -0.5
    if mask is not None:
        s = s.masked_fill(~mask, -INF) if mask.dtype == torch.bool else s + mask.float()
    o = (s.softmax(-1) @ v.float().repeat_interleave(n, 1)).to(q.dtype)
    return o if skip_output_reshape else o.transpose(1, 2).flatten(2)


@pytest.mark.parametrize("kind", ["bool", "additive", "pad", "grouped"])
@pytest.mark.parametrize("head_major_out", [False, True])
def test_nan_in_a_query_raises_on_the_first_call(runtime, cuda_device, kind, head_major_out):
    """As for an unmasked call: a result that is not finite is not checked, so the shape is not accepted."""
    from npu_ai_b200 import comfy_nodes as cn
    q, k, v = _qkv(cuda_device, 2, 8, 2 if kind == "grouped" else 8, 64, 64, 64, True)
    mask = torch.ones(64, 64, dtype=torch.bool, device=cuda_device).tril(8)
    mask[9] = False  # and a row that the mask does hide
    kw = {"bool": dict(mask=mask), "additive": dict(mask=torch.where(mask, 0.0, -INF).to(BF16)),
          "pad": dict(mask=torch.zeros(2, 1, 1, 64, device=cuda_device, dtype=BF16)), "grouped": dict(enable_gqa=True)}[kind]
    good = q.clone()
    q[1, 3, 40] = NAN
    kw.update(skip_reshape=True, skip_output_reshape=head_major_out)
    for bad in (q, torch.full_like(q, NAN)):
        with pytest.raises(RuntimeError, match="does not match"):
            cn._gpu_attention_override(_plain_model, bad, k, v, 8, **kw)
        assert all(r.variant is None for r in runtime.attn.shapes.values())
    before = runtime.attn.fused_calls
    y = cn._gpu_attention_override(_plain_model, good, k, v, 8, **kw)
    assert runtime.attn.fused_calls == before + 1
    _check(y, good, k, v, 2 if kind == "grouped" else 8, kw.get("mask"), True, head_major_out)


@pytest.mark.parametrize("shape", [(64, 64), (2, 1, 1, 64), (1, 8, 64, 64), (2, 8, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.bool, BF16, torch.float32])
@pytest.mark.parametrize("head_major_out", [False, True])
def test_rows_that_the_mask_hides_are_told_from_the_others(runtime, cuda_device, shape, dtype, head_major_out):
    """Each form of mask with some rows hidden: accepted, and zeros there, whatever the model gives (NaN)."""
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 40, False)
    mask = torch.ones(shape, dtype=torch.bool, device=cuda_device)
    mask[..., 50:] = False
    (mask[7] if len(shape) == 2 else mask[-1, -1, min(7, shape[2] - 1)])[:] = False
    if dtype != torch.bool:
        mask = torch.where(mask, 0.0, -INF).to(dtype)

    def nan_model(*a, **kw):  # a plain softmax: rows without a key are NaN
        o = model_attention(*a, **kw)
        m4 = mask if mask.dim() == 4 else mask[None, None]
        none = (~m4 if dtype == torch.bool else m4 == -INF).all(-1).expand(2, 8, 64)
        hm = o if head_major_out else o.unflatten(-1, (8, 40)).transpose(1, 2)
        hm = torch.where(none[..., None], NAN, hm)
        return hm if head_major_out else hm.transpose(1, 2).flatten(2)
    from npu_ai_b200 import comfy_nodes as cn
    y = cn._gpu_attention_override(nan_model, q, k, v, 8, mask=mask, skip_output_reshape=head_major_out)
    (rec,) = runtime.attn.shapes.values()
    assert rec.variant == 0 and rec.max_rel_err < 0.1
    _check(y, q, k, v, 8, mask, False, head_major_out)


def test_each_form_of_mask_is_checked(runtime, cuda_device):
    """The kernel reads a mask row for all queries another way than one per query: a check of one form does not vouch for
    another."""
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 64, False)
    for n, shape in enumerate([(64, 64), (2, 1, 1, 64), (1, 1, 1, 64), (1, 8, 1, 64), (2, 8, 64, 64), (2, 1, 64, 64)]):
        mask = torch.zeros(shape, dtype=BF16, device=cuda_device)
        for _ in range(2):
            _call(runtime, q, k, v, 8, mask=mask)
        assert len(runtime.attn.shapes) == n + 1
    assert all(r.max_rel_err is not None for r in runtime.attn.shapes.values())
    _call(runtime, q, k, v, 8, mask=torch.zeros(1, 1, 64, 64, dtype=BF16, device=cuda_device))  # as [64, 64]
    assert len(runtime.attn.shapes) == 6


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_keys_shared_by_the_batch(runtime, cuda_device, head_major, masked):
    """k and v expanded over the batch (stride 0), which TMA does not address: through the node and the runner."""
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 77, 40, head_major)
    k, v = (t[:1].expand(2, *t.shape[1:]) for t in (k, v))
    mask = torch.ones(64, 77, dtype=torch.bool, device=cuda_device).tril(20) if masked else None
    y, _, fused, _ = _call(runtime, q, k, v, 8, mask=mask, skip_reshape=head_major, skip_output_reshape=head_major)
    assert fused == 1
    _check(y, q, k, v, 8, mask, head_major, head_major)
    y = runtime.gemm.attention(q, k, v, 8, skip_reshape=head_major, skip_output_reshape=head_major, mask=mask)
    _check(y, q, k, v, 8, mask, head_major, head_major)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("case", ["mask", "grouped", "mixed"])
def test_operands_of_more_bits_stay_with_the_model(runtime, cuda_device, dtype, case):
    """Masked and grouped calls are computed in the caller's type: bit for bit the model's result."""
    q, k, v = (t.to(dtype) for t in _qkv(cuda_device, 2, 8, 2 if case == "grouped" else 8, 64, 64, 64, True))
    if case == "mixed":
        q, k = q.to(BF16), k.to(BF16)

    def func(q, k, v, *a, **kw):
        return model_attention(q.to(v.dtype), k.to(v.dtype), v, *a, **kw)
    kw = dict(enable_gqa=True) if case == "grouped" else \
        dict(mask=torch.ones(64, 64, dtype=torch.bool, device=cuda_device).tril(8))
    from npu_ai_b200 import comfy_nodes as cn
    before = runtime.attn.fused_calls
    for _ in range(2):
        y = cn._gpu_attention_override(func, q, k, v, 8, skip_reshape=True, **kw)
        assert torch.equal(y, func(q, k, v, 8, skip_reshape=True, **kw)) and y.dtype == dtype
    assert runtime.attn.fused_calls == before
    assert any("bf16" in (r.model_reason or "") for r in runtime.attn.shapes.values())


def _stays(rt, func, q, k, v, heads, **kw):
    """The call runs the model's own attention, twice, bit for bit."""
    from npu_ai_b200 import comfy_nodes as cn
    before = rt.attn.fused_calls
    for _ in range(2):
        assert torch.equal(cn._gpu_attention_override(func, q, k, v, heads, **kw), func(q, k, v, heads, **kw))
    assert rt.attn.fused_calls == before


def test_operands_that_the_kernel_does_not_take_stay_with_the_model(runtime, cuda_device):
    """v of another width, k and v of one batch entry broadcast by the model, a scale of the model's own, no queries."""
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 64, True)
    mask = torch.ones(64, 64, dtype=torch.bool, device=cuda_device).tril(8)
    kw = dict(mask=mask, skip_reshape=True, skip_output_reshape=True)
    _stays(runtime, model_attention, q, k, v[..., :40], 8, **kw)
    _stays(runtime, model_attention, q, k[:1], v[:1], 8, **kw)
    _stays(runtime, model_attention, q, k, v, 8, scale=-0.125, **kw)
    _stays(runtime, model_attention, q, k, v, 8, scale=torch.tensor(0.125).item() * 0.0, **kw)
    assert all(r.variant is None for r in runtime.attn.shapes.values())


def test_gradients_stay_with_the_model(runtime, cuda_device):
    from npu_ai_b200 import comfy_nodes as cn
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 64, False)
    mask = torch.ones(64, 64, dtype=torch.bool, device=cuda_device).tril(8)
    k.requires_grad_()
    y = cn._gpu_attention_override(model_attention, q, k, v, 8, mask=mask)
    y.float().square().sum().backward()
    assert k.grad is not None and bool(k.grad.abs().sum() > 0)
    with torch.no_grad():  # nothing to lose: the kernel
        y, _, fused, _ = _call(runtime, q, k, v, 8, mask=mask)
    assert fused == 1


@pytest.mark.parametrize("dtype", [torch.bool, BF16, torch.float32])
def test_models_with_other_rows_without_a_key(runtime, cuda_device, dtype):
    """A model that fills with a finite value gives the average of v where its mask leaves nothing; a model that casts f32's
    lowest value to bf16 gives NaN where the kernel gives the average. Their calls stay with them instead of failing."""
    from npu_ai_b200 import comfy_nodes as cn
    q, k, v = _qkv(cuda_device, 2, 8, 8, 64, 64, 64, True)
    mask = torch.ones(64, 64, dtype=torch.bool, device=cuda_device)
    mask[5] = False
    hide = mask
    if dtype == BF16:
        mask = torch.where(mask, 0.0, -INF).to(BF16)
    elif dtype == torch.float32:
        mask = torch.where(mask, 0.0, torch.finfo(torch.float32).min)

    def func(q, k, v, heads, mask=None, **kw):
        s = (q.float() @ k.float().transpose(-1, -2)) * 0.125
        s = s + mask.to(BF16).float() if dtype == torch.float32 else s.masked_fill(~hide, -1e30)
        return (s.softmax(-1) @ v.float()).to(BF16)
    before = runtime.attn.fused_calls
    for _ in range(2):
        y = cn._gpu_attention_override(func, q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)
        ref = func(q, k, v, 8, mask=mask)
        assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(ref)) and torch.equal(y.isnan(), ref.isnan())
    assert runtime.attn.fused_calls == before
    (rec,) = runtime.attn.shapes.values()
    assert "no key" in rec.model_reason
    # any other difference is still an error

    def wrong(*a, **kw):
        o = func(*a, **kw).clone()
        o[:, :, 9] += 5.0
        return o
    runtime.attn.reset()
    with pytest.raises(RuntimeError, match="does not match"):
        cn._gpu_attention_override(wrong, q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)


def test_shapes_on_which_the_model_is_faster_stay_with_it(runtime, cuda_device):
    """Auto mode keeps a masked shape with the model's attention when that took clearly less time; gpu mode does not."""
    from npu_ai_b200 import comfy_nodes as cn
    q, k, v = _qkv(cuda_device, 2, 8, 8, 4096, 4096, 40, True)
    mask = torch.zeros(4096, 4096, dtype=BF16, device=cuda_device)
    ref = model_attention(q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)

    def func(*a, **kw):  # a model as fast as can be
        return ref
    for _ in range(2):
        before = runtime.attn.fused_calls, runtime.attn.model_calls
        y = cn._gpu_attention_override(func, q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)
        assert y is ref and (runtime.attn.fused_calls, runtime.attn.model_calls) == (before[0], before[1] + 1)
    (rec,) = runtime.attn.shapes.values()
    assert "faster" in rec.model_reason and rec.model_ms < rec.variant_ms[0]
    runtime.attn.reset()
    runtime.attn.mode = "gpu"
    before = runtime.attn.fused_calls
    y = cn._gpu_attention_override(func, q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)
    assert runtime.attn.fused_calls == before + 1 and y is not ref


def test_shapes_on_which_the_kernel_is_faster_use_it(runtime, cuda_device):
    q, k, v = _qkv(cuda_device, 2, 8, 8, 1024, 1024, 80, True)
    mask = torch.rand(1024, 1024, device=cuda_device) < 0.5
    mask[:, 0] = True
    y, _, fused, _ = _call(runtime, q, k, v, 8, mask=mask, skip_reshape=True, skip_output_reshape=True)
    assert fused == 1
