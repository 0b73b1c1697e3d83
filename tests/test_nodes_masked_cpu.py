"""What the ComfyUI node hands to the masked attention kernel and to the GEMM with an activation, decided on the host."""
import types

import pytest
import torch

from npu_ai_b200 import comfy_nodes as cn

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [torch.bool, torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(5, 7), (1, 7), (1, 1, 5, 7), (2, 1, 1, 7), (2, 3, 5, 7), (1, 3, 1, 7)])
def test_masks_the_kernel_reads(dtype, shape):
    m = torch.zeros(shape, dtype=dtype)
    got = cn._kernel_mask(m, 2, 3, 5, 7, CPU)
    assert tuple(got.shape) == shape and got.dtype == (torch.float32 if dtype == torch.float16 else dtype)
    if dtype != torch.float16:
        assert got is m  # nothing is copied


def test_masks_that_stay_with_the_model():
    z = torch.zeros
    for m in (z(2, 5, 7), z(7), z(5, 1), z(5, 8), z(4, 7), z(3, 1, 5, 7), z(2, 2, 5, 7), z(5, 7, dtype=torch.float64),
              z(5, 7, dtype=torch.int32), z(5, 7, device="meta"), z(5, 7, requires_grad=True), [[0.0]]):
        assert cn._kernel_mask(m, 2, 3, 5, 7, CPU) is None


def test_mask_keys_become_contiguous():
    m = torch.arange(35.0).view(7, 5).t()
    got = cn._kernel_mask(m, 2, 3, 5, 7, CPU)
    assert got.stride(-1) == 1 and torch.equal(got, m)
    f16 = torch.full((5, 7), torch.finfo(torch.float16).min, dtype=torch.float16)
    assert torch.equal(cn._kernel_mask(f16, 2, 3, 5, 7, CPU), f16.float())


def test_activations_of_the_epilogue():
    nn = torch.nn
    assert [cn._activation_name(m) for m in (nn.GELU(), nn.GELU(approximate="tanh"), nn.SiLU(), nn.ReLU(inplace=True),
                                             nn.Sigmoid(), nn.LeakyReLU(), nn.Identity())] == \
        ["gelu", "gelu_tanh", "silu", "relu", None, None, None]


def test_linear_activation_pairs():
    nn = torch.nn
    seq = nn.Sequential(nn.Linear(8, 8), nn.GELU(), nn.Dropout(0.0), nn.Linear(8, 8), nn.Identity(), nn.Linear(8, 8),
                        nn.SiLU())
    rt = types.SimpleNamespace(weights={id(m): None for m in seq}, fused_member={}, fused_groups={})
    assert cn._linear_act_pairs(seq, rt) == [0, 5]
    del rt.weights[id(seq[0])]
    assert cn._linear_act_pairs(seq, rt) == [5]
    rt.fused_member[id(seq[5])] = 0
    assert cn._linear_act_pairs(seq, rt) == []
    del rt.fused_member[id(seq[5])]
    handle = seq[6].register_forward_hook(lambda *a: None)
    assert cn._linear_act_pairs(seq, rt) == []
    handle.remove()
    assert cn._linear_act_pairs(seq, rt) == [5]
    assert cn._linear_act_pairs(nn.ModuleList(seq), rt) == []


def test_gate_names_calls_by_their_mask():
    gate = cn.AttentionGate()
    gate.record((2, 64, 77, 8, 40)).variant = 0
    gate.record((2, 64, 77, 8, 40, "torch.bool mask")).variant = 0
    assert gate.model_route_reason((2, 64, 77, 8, 40, ""), True, False, True) == "masked attention"
    assert "torch.bool mask" in gate.table() and gate.table().index("(2, 64, 77, 8, 40):") == 0
