"""Linear -> activation pairs of the ComfyUI node leave modules alone whose forward somebody replaced."""
import types

import torch

from npu_ai_b200 import comfy_nodes as cn


def test_replaced_forwards_are_not_passed_by():
    nn = torch.nn
    seq = nn.Sequential(nn.Linear(8, 8), nn.GELU(), nn.Linear(8, 8), nn.SiLU())
    rt = types.SimpleNamespace(weights={id(m): None for m in seq}, fused_member={}, fused_groups={})
    seq[0].forward = types.MethodType(cn._gpu_linear_forward, seq[0])  # as take_over leaves it
    assert cn._linear_act_pairs(seq, rt) == [0, 2]
    own = seq[0].forward
    seq[0].forward = lambda x: own(x) + 1.0  # an adapter put on after the takeover
    assert cn._linear_act_pairs(seq, rt) == [2]
    seq[0].forward = own
    seq[3].forward = types.MethodType(lambda self, x: x, seq[3])
    assert cn._linear_act_pairs(seq, rt) == [0]
    del seq[3].forward
    assert cn._linear_act_pairs(seq, rt) == [0, 2]
