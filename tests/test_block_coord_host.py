"""What a block hands to its attention: coordinates of both sides, and nothing that was not given."""

import pytest
import torch
import torch.nn as nn

from nanobrain_b200 import modules


class Recorder(nn.Module):
    def forward(self, x, **kwargs):
        self.seen = kwargs
        return x


class OldAttention(nn.Module):
    """An attention that knows nothing of coordinates."""

    def forward(self, x, context=None, cu_seqlens=None, max_seqlen=None):
        return x


def block(attn=None, **kwargs):
    b = modules.Block(128, 2, context_dim=128, **kwargs)
    if attn is not None:
        b.attn = attn
    return b


@pytest.mark.parametrize("given", [(), ("coord",), ("context_coord",), ("coord", "context_coord")])
def test_what_is_given_arrives(given):
    x, coords = torch.zeros(1, 4, 128), {name: torch.zeros(1, 4, 3) for name in given}
    b = block(Recorder())
    b(x, context=x, **coords)
    assert {k for k in b.attn.seen if "coord" in k} == set(given)
    assert all(b.attn.seen[k] is v for k, v in coords.items())


def test_an_attention_without_coordinates_in_its_signature():
    x = torch.zeros(1, 4, 128)
    assert block(OldAttention())(x, context=x).shape == x.shape
    with pytest.raises(TypeError, match="context_coord"):
        block(OldAttention())(x, context=x, context_coord=torch.zeros(1, 4, 3))


def test_a_rotating_block_says_which_coordinates_are_missing():
    x, c = torch.zeros(1, 4, 128), torch.zeros(1, 4, 3)
    b = block(qk_norm=True, rope_grid=(4, 4, 4))
    with pytest.raises(ValueError, match="^coord is required"):
        b(x, context=x, context_coord=c)
    with pytest.raises(ValueError, match="^context_coord is required"):
        b(x, context=x, coord=c)
