"""Blocks and models with norms and rotation of queries and keys and the gated MLP: the operators in their places, dense
and packed, forward and backward."""

import pytest
import torch

from nanobrain_b200 import model as M
from nanobrain_b200 import modules, ops
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bf(t):
    return t.to(torch.bfloat16).double()


@pytest.mark.parametrize("mlp,activation", [("swiglu", "silu"), ("geglu", "gelu")])
@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
def test_gated_mlp_module(mlp, activation, checkpoint):
    torch.manual_seed(0)
    layer = modules._make_mlp(mlp, 64, 4, True, checkpoint).to(DEV)
    for b in (layer.fc_gate.bias, layer.fc_up.bias, layer.fc2.bias):
        torch.nn.init.normal_(b, std=0.3)
    assert layer.fc_gate.weight.shape == (176, 64)  # two thirds of 256, up to a multiple of 8
    x = torch.randn(3, 50, 64, device=DEV, requires_grad=True)
    dy = torch.randn(3, 50, 64, device=DEV).bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
    y.backward(dy)
    ops.check_status()
    params = (layer.fc_gate.weight, layer.fc_up.weight, layer.fc2.weight, layer.fc_gate.bias, layer.fc_up.bias, layer.fc2.bias)
    want, grads = O.mlp(x.detach().view(150, 64).bfloat16(), *[p.detach().bfloat16() for p in params], activation=activation,
                        dy=dy.view(150, 64), bits=int(checkpoint[:-3]))
    got = (y.view(150, 64), x.grad.view(150, 64), *[p.grad for p in params])
    for a, b in zip(got, (want, *grads)):
        assert (a.double() - b).norm() <= 2.6 * O.HALF_STEP * b.norm()
    assert all(p.grad.dtype == torch.float32 for p in params)


def test_what_the_modules_refuse():
    with pytest.raises(ValueError, match="qk_norm"):
        modules.Attention(128, 2, rope_grid=(4, 4, 4))
    with pytest.raises(ValueError, match="mlp must be"):
        modules.Block(128, 2, mlp="relu")
    attn = modules.Attention(128, 2, qk_norm=True, rope_grid=(4, 4, 4)).to(DEV).bfloat16()
    x = torch.randn(2, 10, 128, device=DEV).bfloat16()
    with pytest.raises(ValueError, match="coord"):
        attn(x)
    with pytest.raises(ValueError, match="context_coord"):
        attn(x, context=x, coord=torch.zeros(2, 10, 3, dtype=torch.int64, device=DEV))


def test_defaults_have_the_reference_parameters():
    names = set(modules.Block(128, 2, qkv_bias=True, proj_bias=True).state_dict())
    assert not any("norm" in n and "attn" in n or "rope" in n or "gate" in n for n in names)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("cross", [False, True])
def test_attention_with_norms_and_rotation(packed, cross):
    torch.manual_seed(1)
    grid = (6, 5, 7)
    attn = modules.Attention(128, 2, qkv_bias=True, proj_bias=True, qk_norm=True, rope_grid=grid).to(DEV)
    for w in (attn.q_norm, attn.k_norm):
        torch.nn.init.normal_(w, mean=1.0, std=0.3)
    n, m = 60, 90 if cross else 60
    x = torch.randn(n, 128, device=DEV, requires_grad=True)
    ctx = torch.randn(m, 128, device=DEV, requires_grad=True) if cross else None
    coord = torch.randint(0, 5, (n, 3), device=DEV)
    ccoord = torch.randint(0, 5, (m, 3), device=DEV) if cross else None
    dy = torch.randn(n, 128, device=DEV).bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        if packed:
            cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
            cuk = torch.tensor([0, m], dtype=torch.int32, device=DEV)
            y = attn(x, context=ctx, cu_seqlens=cu, max_seqlen=n, cu_seqlens_k=cuk, max_seqlen_k=m, coord=coord,
                     context_coord=ccoord)
        else:
            y = attn(x[None], context=None if ctx is None else ctx[None], coord=coord[None],
                     context_coord=None if ccoord is None else ccoord[None])[0]
    y.backward(dy)
    ops.check_status()

    # the same in 64 bits on the rounded inputs
    x64 = bf(x.detach()).requires_grad_(True)
    src = bf(ctx.detach()).requires_grad_(True) if cross else x64
    wq, wk = (w.detach().double().requires_grad_(True) for w in (attn.q_norm, attn.k_norm))
    lin = lambda layer, t: t @ bf(layer.weight.detach()).t() + bf(layer.bias.detach())
    q, k, v = lin(attn.q, x64).view(n, 2, 64), lin(attn.k, src).view(m, 2, 64), lin(attn.v, src).view(m, 2, 64)
    freqs = modules.axial_frequencies(grid).to(DEV)
    q = O.norm_rope(q, wq, O.angles(coord, freqs, False), 1e-6, False)[0].transpose(0, 1)
    k = O.norm_rope(k, wk, O.angles(ccoord if cross else coord, freqs, False), 1e-6, False)[0].transpose(0, 1)
    out = (torch.softmax(q @ k.transpose(1, 2) / 8, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(n, 128)
    want = lin(attn.proj, out)
    leaves = [x64, wq, wk] + ([src] if cross else [])
    grads = torch.autograd.grad(want, leaves, dy.double())
    got = [y, x.grad, attn.q_norm.grad, attn.k_norm.grad] + ([ctx.grad] if cross else [])
    # each of these has come through at most twelve roundings of half a step
    for a, b in zip(got, (want, *grads)):
        assert (a.double() - b).norm() <= 12 * O.HALF_STEP * b.norm()


def build(checkpoint="16bit", **kwargs):
    torch.manual_seed(3)
    model = M.ViTMAE3D(grid_size=(16, 16, 16), patch_size=4, depth=2, embed_dim=128, num_heads=2, decoder_depth=1,
                       decoder_embed_dim=64, decoder_num_heads=1, mlp_checkpoint=checkpoint, **kwargs).to(DEV)
    torch.nn.init.normal_(model.decoder_head.weight, std=0.02)
    return model


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
def test_training_step_and_packed_form(checkpoint):
    model = build(checkpoint, qk_norm=True, rope=True, mlp="swiglu")
    g = torch.Generator(device=DEV).manual_seed(0)
    images = torch.randn(3, 16, 16, 16, generator=g, device=DEV)
    mask = torch.ones_like(images)
    counts = torch.full((3,), 20, device=DEV)
    order = torch.stack([torch.randperm(64, generator=g, device=DEV) for _ in range(3)])[:, None, :48]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, _ = model.forward_packed(images, mask, counts, 24, 48, order=order)
    loss.backward()
    ops.check_status()
    packed = {name: p.grad.clone() for name, p in model.named_parameters() if p.grad is not None}
    assert torch.isfinite(loss) and all(torch.isfinite(t).all() for t in packed.values())
    for name in ("blocks.0.attn.q_norm", "blocks.1.attn.k_norm", "blocks.0.mlp.fc_gate.weight", "decoder_blocks.0.attn.q_norm",
                 "decoder_blocks.0.mlp.fc2.bias"):
        assert packed[name].abs().max() > 0

    # dense: the same patches through the encoder and decoder of fixed lengths
    patches = M.patchify3d(images, 4)
    bid = torch.arange(3, device=DEV)[:, None]
    coord = model.coord_grid.expand(3, -1, -1)[bid, order[:, 0]]
    patches = patches[bid, order[:, 0]]
    model.zero_grad()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        embeds = model.forward_encoder(patches[:, :20], coord[:, :20])
        pred = model.forward_decoder(embeds, coord[:, 20:], coord=coord[:, :20])
        dense = torch.nn.functional.mse_loss(pred, patches[:, 20:])
    dense.backward()
    ops.check_status()
    assert abs(dense.item() - loss.item()) <= 1e-2 * abs(loss.item())
    for name, p in model.named_parameters():
        if p.grad is not None and packed[name].norm() > 1e-2 * max(t.norm() for t in packed.values()):
            # the same arithmetic on other row layouts: the roundings of two runs, some dozen each
            assert (p.grad - packed[name]).norm() <= 0.1 * packed[name].norm(), name
    with pytest.raises(ValueError, match="coord"):
        model.forward_decoder(embeds, coord[:, 20:])


def test_forward_of_the_reference_signature_and_embedding():
    model = build(qk_norm=True, rope=True, mlp="geglu").eval()
    g = torch.Generator(device=DEV).manual_seed(0)
    images = torch.randn(2, 16, 16, 16, generator=g, device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, state = model(images, torch.ones_like(images), num_visible=16, num_predict=30)
    assert torch.isfinite(loss) and state["pred_patches"].shape == (2, 30, 64)
    samples = []
    for n in (5, 40):
        m = torch.zeros(64, dtype=torch.bool, device=DEV)
        m[torch.randperm(64, generator=g, device=DEV)[:n]] = True
        samples.append((torch.randn(64, 64, generator=g, device=DEV), m))
    assert model._native_encoder(samples) is None  # (it knows the reference's blocks alone)
    out = model.embed_packed(samples)
    ops.check_status()
    for (patches, m), o in zip(samples, out):
        with torch.inference_mode(), torch.autocast("cuda", dtype=torch.bfloat16):
            tokens = model.forward_encoder(patches[m][None], model.coord_grid[:, m])[0, 1:].float()
        assert (o["global_embedding"] - tokens.mean(0)).norm() <= 3e-2 * tokens.mean(0).norm()


def test_rotation_sees_relative_places_only():
    # moving all tokens by the same step leaves scores, and so the attention's output, unchanged up to roundings
    torch.manual_seed(2)
    attn = modules.Attention(64, 1, qk_norm=True, rope_grid=(8, 8, 8)).to(DEV)
    x = torch.randn(1, 30, 64, device=DEV)
    coord = torch.randint(0, 8, (1, 30, 3), device=DEV)
    with torch.inference_mode(), torch.autocast("cuda", dtype=torch.bfloat16):
        a, b, c = attn(x, coord=coord), attn(x, coord=coord + 5), attn(x, coord=coord.flip(1))
    assert (a - b).norm() <= 8 * O.HALF_STEP * a.norm()
    assert (a - c).norm() > 0.1 * a.norm()


def test_compiled_block():
    torch.manual_seed(4)
    block = modules.Block(128, 2, qkv_bias=True, proj_bias=True, qk_norm=True, rope_grid=(4, 4, 4), mlp="swiglu").to(DEV)
    x = torch.randn(2, 40, 128, device=DEV)
    coord = torch.randint(0, 4, (2, 40, 3), device=DEV)
    outs = []
    for fn in (block, torch.compile(block, backend="aot_eager")):
        xi = x.clone().requires_grad_(True)
        block.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = fn(xi, coord=coord)
        y.float().square().sum().backward()
        outs.append((y.detach(), xi.grad, block.mlp.fc_up.weight.grad.clone(), block.attn.q_norm.grad.clone()))
    ops.check_status()
    for a, b in zip(*outs):
        assert (a - b).norm() <= 2e-2 * a.norm()
