"""Rotating modules and models whose parameters are bfloat16, without autocast: forward and backward."""

import copy

import pytest
import torch

from nanobrain_b200 import model as M
from nanobrain_b200 import modules, ops
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
GRID = (6, 5, 7)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("coord_type", [torch.int64, torch.int32, torch.float32])
def test_attention_in_bf16(packed, coord_type):
    torch.manual_seed(1)
    n = 75
    attn = modules.Attention(128, 2, qkv_bias=True, proj_bias=True, qk_norm=True, rope_grid=GRID).to(DEV)
    for w in (attn.q_norm, attn.k_norm):
        torch.nn.init.normal_(w, mean=1.0, std=0.3)
    attn = attn.bfloat16()
    x = torch.randn(n, 128, device=DEV).bfloat16().requires_grad_(True)
    coord = torch.stack([torch.randint(0, g, (n,), device=DEV) for g in GRID], 1)
    dy = torch.randn(n, 128, device=DEV).bfloat16()
    if packed:
        cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        y = attn(x, cu_seqlens=cu, max_seqlen=n, coord=coord.to(coord_type))
    else:
        y = attn(x[None], coord=coord.to(coord_type)[None])[0]
    y.backward(dy)
    ops.check_status()

    x64 = x.detach().double().requires_grad_(True)
    wq, wk = (w.detach().double().requires_grad_(True) for w in (attn.q_norm, attn.k_norm))
    lin = lambda layer, t: t @ layer.weight.detach().double().t() + layer.bias.detach().double()
    theta = O.angles(coord, modules.axial_frequencies(GRID).to(DEV), False)
    q, k, v = (lin(layer, x64).view(n, 2, 64) for layer in (attn.q, attn.k, attn.v))
    q, k = (O.norm_rope(t, w, theta, 1e-6, False)[0].transpose(0, 1) for t, w in ((q, wq), (k, wk)))
    out = (torch.softmax(q @ k.transpose(1, 2) / 8, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(n, 128)
    want = lin(attn.proj, out)
    leaves = (x64, wq, wk)
    grads = torch.autograd.grad(want, leaves, dy.double())
    # at most twelve roundings of half a step, as under autocast, and two more where x's three gradients are added in bf16
    for a, b in zip((y, x.grad, attn.q_norm.grad, attn.k_norm.grad), (want, *grads)):
        assert a.dtype == torch.bfloat16
        assert (a.double() - b).norm() <= 14 * O.HALF_STEP * b.norm()


def test_model_in_bf16():
    torch.manual_seed(3)
    model = M.ViTMAE3D(grid_size=(16, 16, 16), patch_size=4, depth=2, embed_dim=128, num_heads=2, decoder_depth=1,
                       decoder_embed_dim=64, decoder_num_heads=1, qk_norm=True, rope=True, mlp="swiglu").to(DEV)
    torch.nn.init.normal_(model.decoder_head.weight, std=0.02)
    half = copy.deepcopy(model).bfloat16()
    g = torch.Generator(device=DEV).manual_seed(0)
    images = torch.randn(3, 16, 16, 16, generator=g, device=DEV)
    mask = torch.ones_like(images)
    torch.manual_seed(7)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want, _ = model(images, mask, num_visible=16, num_predict=30)
    torch.manual_seed(7)
    loss, _ = half(images.bfloat16(), mask.bfloat16(), num_visible=16, num_predict=30)
    loss.backward()
    ops.check_status()
    # the loss' sums and their quotient are rounded to bf16 three times; the rest hardly moves a mean of squares near 1
    assert abs(loss.item() - want.item()) <= (3 * O.HALF_STEP + 8e-3) * want.item()
    for block in (*half.blocks, *half.decoder_blocks):
        for p in (block.attn.q_norm, block.attn.k_norm, block.mlp.fc_gate.weight):
            assert torch.isfinite(p.grad).all() and p.grad.abs().max() > 0

    counts = torch.tensor([5, 16, 11], device=DEV)
    loss, state = half.forward_packed(images.bfloat16(), mask.bfloat16(), counts, 16, 40)
    loss.backward()
    ops.check_status()
    assert torch.isfinite(loss) and torch.isfinite(state["pred_patches"]).all()


def test_embeddings_of_a_model_in_bf16():
    torch.manual_seed(3)
    model = M.ViTMAE3D(grid_size=(16, 16, 16), patch_size=4, depth=2, embed_dim=128, num_heads=2, decoder_depth=1,
                       decoder_embed_dim=64, decoder_num_heads=1, qk_norm=True, rope=True).to(DEV).eval()
    half = copy.deepcopy(model).bfloat16()
    g = torch.Generator(device=DEV).manual_seed(0)
    samples = []
    for n in (5, 40):
        m = torch.zeros(64, dtype=torch.bool, device=DEV)
        m[torch.randperm(64, generator=g, device=DEV)[:n]] = True
        samples.append((torch.randn(64, 64, generator=g, device=DEV), m))
    want = model.embed_packed(samples)
    got = half.embed_packed([(patches.bfloat16(), m) for patches, m in samples])
    ops.check_status()
    for a, b in zip(got, want):
        a, b = a["global_embedding"], b["global_embedding"]
        # two blocks of some ten roundings on either side
        assert (a - b).norm() <= 2 * 2 * 10 * O.HALF_STEP * b.norm()
