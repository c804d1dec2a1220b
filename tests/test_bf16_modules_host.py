"""Modules converted to another type: the rotation's frequencies stay what they were made as."""

import copy

import pytest
import torch

from nanobrain_b200 import model as M
from nanobrain_b200 import modules

GRID = (6, 5, 7)


def attention():
    return modules.Attention(128, 2, qk_norm=True, rope_grid=GRID)


@pytest.mark.parametrize("convert", [
    lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
    lambda m: m.to("cpu", torch.bfloat16), lambda m: m.type(torch.bfloat16), lambda m: m.bfloat16().float(),
    lambda m: copy.deepcopy(m.bfloat16()), lambda m: m.to(torch.bfloat16).to("meta"),
])
def test_frequencies_stay_in_float32(convert):
    want = modules.axial_frequencies(GRID)
    model = convert(attention())
    assert model.rope_freqs.dtype == torch.float32 and model.rope_freqs.device == model.q.weight.device
    if not model.rope_freqs.is_meta:
        assert torch.equal(model.rope_freqs, want)
    assert "rope_freqs" in dict(model.named_buffers()) and "rope_freqs" not in model.state_dict()


def test_everything_else_is_converted():
    model = attention().bfloat16()
    assert all(p.dtype == torch.bfloat16 for p in model.parameters())
    plain = modules.Attention(128, 2).bfloat16()
    assert plain.rope_freqs is None and all(p.dtype == torch.bfloat16 for p in plain.parameters())


def test_frequencies_that_were_set_stay_as_well():
    model = attention()
    model.rope_freqs = torch.full((3, 32), 1 / 3)
    model.bfloat16()
    assert torch.equal(model.rope_freqs, torch.full((3, 32), 1 / 3))


def test_a_whole_model():
    model = M.ViTMAE3D(grid_size=(16, 16, 16), patch_size=4, depth=1, embed_dim=128, num_heads=2, decoder_depth=1,
                       decoder_embed_dim=64, decoder_num_heads=1, qk_norm=True, rope=True).bfloat16()
    for block in (*model.blocks, *model.decoder_blocks):
        assert torch.equal(block.attn.rope_freqs, modules.axial_frequencies((4, 4, 4)))
        assert block.attn.q.weight.dtype == torch.bfloat16
    assert model.coord_grid.dtype == torch.int64
