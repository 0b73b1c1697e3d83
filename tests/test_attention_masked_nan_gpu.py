"""NaN where a row looks, on the B200: masked attention gives a NaN row for a query that sees a NaN score, as the formula,
torch and the unmasked kernel do, and every other row its usual result. Rows that see nothing stay zero whatever their
query holds. Tolerances are those of test_attention_masked_gpu.py."""
import pytest
import torch

from test_attention_masked_gpu import BF16, INF, _heads, _qkv, check, ints, oracle

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _seen(B, H, Sq, Skv, dev, causal=False, kv_lens=None, mask=None):
    """[B, H, Sq, Skv]: the keys that a row may see (a NaN mask value does not hide)."""
    i, j = torch.arange(Sq, device=dev)[:, None], torch.arange(Skv, device=dev)[None]
    seen = torch.ones(B, H, Sq, Skv, dtype=torch.bool, device=dev)
    if causal:
        seen &= j <= i + Skv - Sq
    if kv_lens is not None:
        seen &= j < kv_lens.view(B, 1, 1, 1)
    if mask is not None:
        m4 = mask if mask.dim() == 4 else mask[None, None]
        seen &= m4 if mask.dtype == torch.bool else ~(m4 == -INF)
    return seen


def _clean(t):
    return t if t is None or t.dtype == torch.bool else torch.nan_to_num(t, nan=0.0, posinf=INF, neginf=-INF)


def _check_nan(dev, q, k, v, H, Hk, mask=None, variant=0, **kw):
    """Runs the call and compares: NaN rows exactly where the formula has them, the others to tolerance."""
    from npu_ai_b200 import kernels
    out = kernels.attention(q, k, v, H, kv_heads=Hk, mask=mask, variant=variant, **kw)
    kernels.check_status(dev)
    seen = _seen(q.shape[0], H, q.shape[1], k.shape[1], dev, kw.get("causal", False), kw.get("kv_lens"), mask)
    bad = _heads(q, H, False).isnan().any(-1)[..., None] | \
        _heads(k, Hk, False).isnan().any(-1).repeat_interleave(H // Hk, 1)[:, :, None]
    if mask is not None and mask.dtype != torch.bool:
        bad = bad | (mask if mask.dim() == 4 else mask[None, None]).isnan()
    bad = (bad & seen).any(-1)
    o = _heads(out, H, False)
    assert bool(o[bad].isnan().all()), "a row that sees a NaN is finite"
    ref, tol = oracle(_clean(q), _clean(k), v, H, Hk, mask=_clean(mask), **kw)
    o = torch.where(bad[..., None], ref, o)
    check(o.transpose(1, 2).flatten(2).float(), ref, tol, H, False)
    return bad


def _mask(kind, B, H, Sq, Skv, dev, seed=5):
    g = torch.Generator(device=dev).manual_seed(seed)
    if kind == "none":
        return None
    shape = {"own": (B, 1, Sq, Skv), "head": (1, H, Sq, Skv), "shared": (B, 1, 1, Skv)}[kind.split("_")[1]]
    keep = torch.rand(shape, generator=g, device=dev) < 0.6
    keep[..., -1] = True
    if kind.startswith("bool"):
        return keep
    add = torch.where(keep, torch.randn(shape, generator=g, device=dev), -INF)
    return add.to(BF16 if kind.startswith("bf16") else torch.float32)


KINDS = ["none", "bool_own", "bool_shared", "bf16_own", "f32_own", "f32_head", "bf16_shared", "f32_shared"]
# one part in one stream of key tiles, in two streams, a cluster's join, the workspace join by four warps a row and by one
FORMS = [(5, 150, 1), (130, 400, 1), (1, 400, 2), (5, 400, 3), (5, 1500, 24), (130, 400, 2), (130, 600, 9), (300, 1000, 40)]


@pytest.mark.parametrize("Sq,Skv,variant", FORMS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("extra", ["", "softcap", "slopes"])
def test_nan_in_a_query_and_in_a_key(cuda_device, kind, Sq, Skv, variant, extra):
    dev, B, H, Hk, D = cuda_device, 2, 4, 2, 64
    kw = {"softcap": dict(softcap=8.0), "slopes": dict(slopes=torch.rand(H, device=dev))}.get(extra, {})
    mask = _mask(kind, B, H, Sq, Skv, dev)
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, Sq + Skv, dev)
    q[0, Sq // 2, 1 * D + 3] = NAN            # one query of one head
    bad = _check_nan(dev, q, k, v, H, Hk, mask, variant, **kw)
    assert bool(bad[0, 1, Sq // 2]) and int(bad.sum()) == 1
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, Sq + Skv + 1, dev)
    k[1, Skv - 1, 0 * D + 5] = NAN            # one key, which every mask leaves to every row
    bad = _check_nan(dev, q, k, v, H, Hk, mask, variant, **kw)
    assert bool(bad[1, :2].all()) and int(bad.sum()) == 2 * Sq
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, Sq + Skv + 2, dev)
    k[0] = NAN                                # every key
    bad = _check_nan(dev, q, k, v, H, Hk, mask, variant, **kw)
    assert bool(bad[0].all()) and not bool(bad[1].any())


@pytest.mark.parametrize("variant", [0, 1, 2, 40])
@pytest.mark.parametrize("D", [40, 128, 160, 256])
def test_nan_in_the_first_key_of_a_causal_call(cuda_device, D, variant):
    """Row 0 sees that key alone, the others among finite ones; the sequence of length 0 sees none."""
    dev = cuda_device
    q, k, v = _qkv(3, 4, 2, 200, 200, D, D, dev)
    k[:, 0, 0] = NAN
    bad = _check_nan(dev, q, k, v, 4, 2, variant=variant, causal=True, kv_lens=ints(dev, 200, 0, 70))
    assert bool(bad[0, :2].all()) and not bool(bad[1].any())
    q, k, v = _qkv(3, 4, 2, 200, 200, D, D, dev)
    k[:, 150, 0] = NAN                        # seen from row 150 on: a tile's later rows only
    bad = _check_nan(dev, q, k, v, 4, 2, variant=variant, causal=True, kv_lens=ints(dev, 200, 0, 151))
    assert int(bad.sum()) == 2 * 50 * 2


@pytest.mark.parametrize("kind", ["bf16_own", "f32_own", "f32_head", "bf16_shared", "f32_shared"])
@pytest.mark.parametrize("Sq,Skv,variant", FORMS)
def test_nan_in_the_mask(cuda_device, kind, Sq, Skv, variant):
    """A NaN among a row's values, next to the type's lowest one, and as all of them."""
    dev, B, H, Hk = cuda_device, 2, 4, 2
    q, k, v = _qkv(B, H, Hk, Sq, Skv, 64, Skv, dev)
    for fill in ("one", "low", "all"):
        mask = _mask(kind, B, H, Sq, Skv, dev)
        row = mask[-1, 0, min(1, mask.shape[2] - 1)]
        if fill == "low":
            row[:] = torch.finfo(mask.dtype).min
        row[3 if fill != "all" else slice(None)] = NAN
        bad = _check_nan(dev, q, k, v, H, Hk, mask, variant)
        assert bool(bad.any()) and not bool(bad.all())
