"""Whole modules pickled (``torch.save(model)``) before attentions could normalise and rotate load and work as they did."""

import copy
import io

import pytest
import torch

from nanobrain_b200 import model as M
from nanobrain_b200 import modules


def as_saved_before(model):
    """The model's pickle without what such a pickle does not hold, read back."""
    model = copy.deepcopy(model)
    for m in model.modules():
        if isinstance(m, modules.Attention):
            for name in ("q_norm", "k_norm", "rope_freqs"):
                for place in (vars(m), m._parameters, m._buffers):
                    place.pop(name, None)
            m._non_persistent_buffers_set.discard("rope_freqs")
        if isinstance(m, M.ViTMAE3D):
            del m.rope
    file = io.BytesIO()
    torch.save(model, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


def test_attention():
    want = modules.Attention(128, 2, qkv_bias=True)
    attn = as_saved_before(want)
    assert attn.q_norm is None and attn.k_norm is None and attn.rope_freqs is None
    assert attn.bfloat16().q.weight.dtype == torch.bfloat16
    assert set(attn.state_dict()) == set(want.state_dict())
    x = torch.zeros(1, 4, 128)
    with pytest.raises(Exception) as refusal:  # (attention has no CPU path: the same one as of a new module)
        want(x)
    with pytest.raises(type(refusal.value)):
        as_saved_before(want)(x)


def test_model():
    want = M.ViTMAE3D(grid_size=(16, 16, 16), patch_size=4, depth=1, embed_dim=64, num_heads=1, decoder_depth=1,
                      decoder_embed_dim=64, decoder_num_heads=1)
    model = as_saved_before(want)
    assert model.rope is False and model._rotation(torch.zeros(1, 4, 3)) == {}
    assert model.blocks[0].attn.q_norm is None
    assert all(torch.equal(a, b) for a, b in zip(model.parameters(), want.parameters()))


def test_what_is_pickled_now_keeps_what_it_has():
    attn = modules.Attention(128, 2, qk_norm=True, rope_grid=(4, 4, 4))
    again = copy.deepcopy(attn)
    assert torch.equal(again.q_norm, attn.q_norm) and torch.equal(again.rope_freqs, attn.rope_freqs)
    assert isinstance(again.q_norm, torch.nn.Parameter) and "rope_freqs" not in again.state_dict()
