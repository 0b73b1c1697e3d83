"""Which operands of a masked call the ComfyUI node hands to the kernel, decided on the host."""
import pytest
import torch

from npu_ai_b200 import comfy_nodes as cn

BF16 = torch.bfloat16


def _qkv(head_major, hk=8):
    if head_major:
        return [torch.zeros(2, n, t, 16, dtype=BF16) for n, t in ((8, 5), (hk, 9), (hk, 9))]
    return [torch.zeros(2, t, n * 16, dtype=BF16) for n, t in ((8, 5), (hk, 9), (hk, 9))]


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("hk", [1, 2, 8])
def test_operands_that_fit(head_major, hk):
    q, k, v = _qkv(head_major, hk)
    for scale in (None, 0.25, 1, 1e-37, 1e38):
        assert cn._kernel_operands(q, k, v, 8, head_major, scale)


@pytest.mark.parametrize("head_major", [False, True])
def test_operands_that_stay_with_the_model(head_major):
    q, k, v = _qkv(head_major)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38, 1e-50, torch.tensor(0.5)):
        assert not cn._kernel_operands(q, k, v, 8, head_major, scale)
    assert not cn._kernel_operands(q, k[:1], v[:1], 8, head_major, None)
    assert not cn._kernel_operands(q, k, v[..., :8], 8, head_major, None)
    assert not cn._kernel_operands(q, k[..., :8], v[..., :8], 8, head_major, None)
    assert not cn._kernel_operands(q, k[0], v[0], 8, head_major, None)
    k.requires_grad_()
    assert not cn._kernel_operands(q, k, v, 8, head_major, None)
    with torch.no_grad():
        assert cn._kernel_operands(q, k, v, 8, head_major, None)


def test_forms_of_masks():
    z = torch.zeros
    assert [cn._mask_form(m) for m in (z(5, 9), z(1, 9), z(2, 1, 1, 9), z(1, 8, 5, 9), z(2, 8, 5, 9), z(1, 1, 5, 9))] == \
        ["11q", "111", "b11", "1hq", "bhq", "11q"]


@pytest.mark.parametrize("head_major", [False, True])
def test_rows_without_a_key(head_major):
    m = torch.zeros(2, 1, 3, 4)
    m[1, 0, 2] = -float("inf")
    m[0, 0, 1] = torch.finfo(torch.float32).min
    m[0, 0, 0, 1:] = -float("inf")
    none, lowest = (t.expand(2, 8, 3, 16) if head_major else t.unflatten(-1, (8, 16)).transpose(1, 2)
                    for t in cn._rows_without_a_key(m, 2, 8, 3, 16, head_major))
    assert bool(none[1, :, 2].all()) and int(none.sum()) == 8 * 16
    assert bool(lowest[0, :, 1].all()) and bool(lowest[1, :, 2].all()) and int(lowest.sum()) == 2 * 8 * 16
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1] = False
    none, lowest = cn._rows_without_a_key(keep, 2, 8, 3, 16, head_major)
    assert int(none.expand(2, 8, 3, 16).sum() if head_major else none.sum()) == 2 * 8 * 16 and none is lowest
