"""Models whose methods someone has replaced: ``forward`` calls them as it always has."""

import torch

from nanobrain_b200 import model as M

SIZES = dict(grid_size=(16, 16, 16), patch_size=4, depth=1, embed_dim=64, num_heads=1, decoder_depth=1, decoder_embed_dim=64,
             decoder_num_heads=1)


class OwnDecoder(M.ViTMAE3D):
    """With the reference's two arguments of the decoder (``model.py:143-165``)."""

    def forward_encoder(self, patches, coord):
        return patches.new_zeros(patches.shape[0], patches.shape[1] + self.class_tokens, self.embed_dim)

    def forward_decoder(self, embeds, target_coord):
        self.seen = embeds.shape, target_coord.shape
        return embeds.new_zeros(*target_coord.shape[:2], self.decoder_head.out_features)


class OwnRotatingDecoder(OwnDecoder):
    def forward_decoder(self, embeds, target_coord, coord=None):
        self.seen = target_coord.shape, coord.shape
        return embeds.new_zeros(*target_coord.shape[:2], self.decoder_head.out_features)


def test_a_decoder_of_the_reference_signature():
    images = torch.randn(2, 16, 16, 16)
    model = OwnDecoder(**SIZES)
    loss, state = model(images, torch.ones_like(images), num_visible=16, num_predict=30)
    assert model.seen == ((2, 17, 64), (2, 30, 3))
    assert torch.allclose(loss, state["target_patches"].square().mean())


def test_a_rotating_model_hands_over_the_visible_coordinates():
    images = torch.randn(2, 16, 16, 16)
    model = OwnRotatingDecoder(**SIZES, qk_norm=True, rope=True)
    model(images, torch.ones_like(images), num_visible=16, num_predict=30)
    assert model.seen == ((2, 30, 3), (2, 16, 3))
