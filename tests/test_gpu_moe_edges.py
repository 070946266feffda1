"""Routing and experts' layers at sizes that belong to them and are easily left out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_routing_without_choices():
    """No choice per token: no rows, every expert's range empty."""
    from llmcompressor_amd.moe import route_tokens
    for ids in (torch.zeros(5, 0, dtype=torch.int64), torch.zeros(0, 0, dtype=torch.int64)):
        want, got = route_tokens(ids, 4), route_tokens(ids.cuda(), 4)
        assert got[1] == want[1] == [0] * 5
        for a, b in ((got[0], want[0]), (got[2], want[2])):
            assert a.dtype == b.dtype and torch.equal(a.cpu(), b)


@pytest.mark.parametrize("tokens,routed", [(6, 4), (4, 6), (0, 2), (3, 0)])
def test_experts_refuse_ids_of_another_number_of_tokens(tokens, routed):
    from llmcompressor_amd import W4A16Experts
    packed = torch.zeros(2, 32, 4, dtype=torch.int32)
    down = torch.zeros(2, 32, 2, dtype=torch.int32)
    scale = torch.ones(2, 32, 1, dtype=torch.bfloat16)
    layer = W4A16Experts((packed, scale, None, None), (down, scale, None, None), 2, 16).cuda()
    x = torch.ones(tokens, 32, dtype=torch.bfloat16, device="cuda")
    ids, w = torch.zeros(routed, 2, dtype=torch.int64, device="cuda"), torch.ones(routed, 2, device="cuda")
    with pytest.raises(ValueError, match="tokens"):
        layer(x, ids, w)
    assert layer(x[:0], ids[:0], w[:0]).shape == (0, 32)
