"""Which kernel an attention call goes to, decided on the host, and what a group refuses."""
import pytest
import torch

from npu_ai_b200 import kernels, sharding

BF16 = torch.bfloat16


@pytest.fixture
def route(monkeypatch):
    """The name of the path that a call takes."""
    seen = []
    monkeypatch.setattr(kernels, "_attention_masked", lambda *a: seen.append("masked"))

    def plain(t, name):
        seen.append("unmasked")
        raise StopIteration
    monkeypatch.setattr(kernels, "_require_cuda", plain)

    def call(*a, **kw):
        seen.clear()
        try:
            kernels.attention(*a, **kw)
        except StopIteration:
            pass
        return seen[0]
    return call


def test_fewer_key_heads_than_query_heads(route):
    """kv_heads defaults to what k's shape says, in both layouts."""
    q, k = torch.zeros(2, 5, 8 * 64, dtype=BF16), torch.zeros(2, 9, 2 * 64, dtype=BF16)
    assert route(q, k, k, 8) == "masked" and route(q, k, k, 8, kv_heads=2) == "masked"
    q, k = torch.zeros(2, 8, 5, 64, dtype=BF16), torch.zeros(2, 2, 9, 64, dtype=BF16)
    assert route(q, k, k, 8, head_major_in=True) == "masked"
    for hm, shape in ((False, (2, 9, 512)), (True, (2, 8, 9, 64))):
        q = torch.zeros(shape, dtype=BF16)
        assert route(q, q, q, 8, head_major_in=hm) == "unmasked"
        assert route(q, q, q, 8, head_major_in=hm, kv_heads=8) == "unmasked"


def test_a_start_position_is_checked_with_the_others(route):
    q = torch.zeros(2, 9, 512, dtype=BF16)
    assert route(q, q, q, 8, q_start=0) == "masked"


@pytest.mark.parametrize("head_major", [False, True])
def test_a_group_refuses_grouped_heads(head_major):
    """Slicing the pairs of a rank out of k and v needs one head each for every query head."""
    q = torch.zeros((2, 8, 5, 16) if head_major else (2, 5, 128), dtype=BF16)
    k = torch.zeros((2, 2, 9, 16) if head_major else (2, 9, 32), dtype=BF16)
    for kv in ((k, k), (q, k), (q[:1], q[:1])):
        with pytest.raises(ValueError, match="do not hold"):
            sharding.attention_shard(q, *kv, 8, 0, 2, head_major_in=head_major, compute=lambda *a: None)
