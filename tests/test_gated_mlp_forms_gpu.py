"""``gated_mlp`` in every form that its kernels take: teams of one and two CTAs, tiles of 64 to 256 columns, products in one
piece and in parts, few tokens at depths on both sides of what is requested ahead, operands that are copied first, and all
of it in one stream between attention kernels."""

import pytest
import torch

import nanobrain_b200 as nb
import test_gated_mlp_gpu as G
from nanobrain_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"

# Which team and tile a product gets follows from the sizes and the SM count. The rules, gone through on the host for 148 SMs
# over tokens to 60000 and widths to 5000, give 72 combinations of product (gate, h Wd^T, the activation's backward, dx,
# gradients of Wg or Wu, of Wd), CTAs, columns and whether it is cut; the sizes of test_gated_mlp_gpu.py take 41 of them. Here
# are the others, each size with those that it is for ("2 x 64": pairs on 64 columns; "cut": in parts).
FORMS = [
    (9000, 512, 1368),    # the decoder's forms: gate 2 x 128, y 2 x 256, activation's backward 2 x 128, gradients cut
    (2201, 768, 2048),    # y 2 x 128, activation's backward 2 x 128, dx cut 2 x 256
    (20431, 768, 1536),   # y 2 x 256, activation's backward 2 x 192
    (6647, 136, 136),     # y 1 x 128, dx 1 x 192, dWg and dWd cut 1 x 192
    (12063, 472, 64),     # y 1 x 192, dx 1 x 256, dWg cut 1 x 256, dWd cut 1 x 64
    (6180, 72, 3424),     # gate 1 x 256, activation's backward 1 x 192, dx and dWg cut 2 x 128
    (834, 64, 64),        # all gradients 2 x 64
    (1484, 72, 752),      # dx and dWg cut 1 x 128, dWd cut 1 x 256
    (21, 144, 584),       # dx cut 1 x 192, dWg 1 x 192
    (2534, 64, 64),       # dWg and dWd cut 2 x 64
    (1791, 136, 136),     # dWg and dWd cut 2 x 192
    (26630, 400, 72),     # y 1 x 256, dWd cut 2 x 128
    (6502, 64, 5120),     # activation's backward 1 x 256, dx cut 2 x 64
    (8887, 168, 4864),    # activation's backward 2 x 256, dx cut 2 x 192
    (20, 64, 1040),       # dx cut 1 x 64
]


@pytest.mark.parametrize("activation,bias,checkpoint", [("silu", False, "16bit"), ("gelu", True, "8bit")])
@pytest.mark.parametrize("tokens,dim,hidden", FORMS)
def test_training_in_every_form(tokens, dim, hidden, activation, bias, checkpoint):
    args = G.problem(tokens, dim, hidden, bias)
    dy = G.randn(tokens, dim, seed=9, std=0.1)
    first = G.run(args, dy, activation, checkpoint)
    G.compare(args, activation, checkpoint, first, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, G.run(args, dy, activation, checkpoint)))


@pytest.mark.parametrize("tokens", [1, 7, 8, 9, 16])
@pytest.mark.parametrize("dim,hidden", [(1024, 2736), (64, 2048), (72, 2056), (64, 2088), (2056, 4104), (8, 5120)])
@pytest.mark.parametrize("bias", [False, True])
def test_few_tokens_behind_what_is_requested_ahead(tokens, dim, hidden, bias):
    # (a warp of the second kernel requests 4 chunks of 32 ahead, 16 warps: 2048 features)
    args = G.problem(tokens, dim, hidden, bias)
    for activation in ("silu", "gelu"):
        with torch.inference_mode():
            y = nb.gated_mlp(*args, activation=activation)
        ops.check_status()
        G.close(y, G.O.mlp(*args, activation=activation)[0], 2)


def off_by_one(t):
    """The same values at an address that is no multiple of 16 bytes, rows at odd places."""
    if t.dim() == 1:
        return torch.cat((t[:1], t))[1:]
    return torch.cat((t[:, :1], t), 1)[:, 1:]


@pytest.mark.parametrize("tokens", [5, 60])
@pytest.mark.parametrize("moved", [(0,), (1,), (2,), (3,), (4,), (5,), (6,), (0, 1, 2, 3, 4, 5, 6)])
def test_operands_at_odd_addresses(tokens, moved):
    args = G.problem(tokens, 64, 96, True)
    dy = G.randn(tokens, 64, seed=9)
    views = [off_by_one(t) if i in moved else t for i, t in enumerate(args)]
    assert all(views[i].data_ptr() % 16 for i in moved)
    with torch.inference_mode():
        assert torch.equal(nb.gated_mlp(*views), nb.gated_mlp(*args))
    for checkpoint in ("16bit", "8bit"):
        for a, b in zip(G.run(views, off_by_one(dy), checkpoint=checkpoint), G.run(args, dy, checkpoint=checkpoint)):
            assert torch.equal(a, b)


def test_no_tokens_of_other_shapes():
    args = G.problem(0, 64, 96, True)
    for shape in ((0, 5, 64), (5, 0, 64), (0, 64)):
        x = args[0].view(shape).requires_grad_(True)
        y = nb.gated_mlp(x, *args[1:])
        assert y.shape == shape
        (dx,) = torch.autograd.grad(y, x, torch.empty_like(y))
        assert dx.shape == shape


def test_pairs_and_single_blocks_between_attention_kernels():
    # Kernels that hold tensor memory, in one stream without a host that waits: attention forward and backward, products by
    # pairs and by single blocks, few tokens, many times. Every pass has the bits of one whose kernels ran one at a time. One
    # result may differ: the attention's backward adds dQ's fp32 parts in the order they come (nb_attn.h), so a value of dQ may
    # be rounded to the bf16 next to the other, two half steps, and its image under the norm's and rotation's backward, which is
    # linear and made of the same r w, again: four half steps of its norm.
    blocks = [(1, 64, 2056), (20, 64, 1040), (834, 64, 64), (1484, 72, 752), (2201, 768, 2048), (6647, 136, 136)]
    problems = [(G.problem(t, d, f, True), G.randn(t, d, seed=9, std=0.1)) for t, d, f in blocks]
    q, k, v, do = (G.randn(700, 4, 64, seed=s) for s in (20, 21, 22, 23))
    cu = torch.tensor([0, 1, 300, 300, 690], dtype=torch.int32, device=DEV)
    dense = [G.randn(2, 4, 130, 64, seed=s) for s in (30, 31, 32, 33)]
    weight = torch.ones(64, device=DEV)

    def attention(i, wait):
        leaves = [t.detach().requires_grad_(True) for t in ((q, k, v) if i % 2 else dense[:3])]
        a, b = nb.qk_norm_rope(leaves[0], leaves[1], weight, weight)
        wait()
        y = nb.sdpa_varlen(a, b, leaves[2], cu, cu, 390, 390) if i % 2 else nb.sdpa(a, b, leaves[2])
        wait()
        out = (y.detach(), *torch.autograd.grad(y, leaves, do if i % 2 else dense[3]))
        wait()
        by_order.append(out[1])
        return out[0], *out[2:]

    def one_pass(wait=lambda: None):
        out = []
        by_order.clear()
        for i, (args, dy) in enumerate(problems):
            leaves = [t.detach().requires_grad_(True) for t in args]
            y = nb.gated_mlp(*leaves, checkpoint="8bit" if i % 2 else "16bit")
            wait()
            out += attention(i, wait)
            out += [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            wait()
            with torch.no_grad():
                out.append(nb.gated_mlp(*args))
            wait()
        return out, list(by_order)

    by_order = []
    want, want_dq = one_pass(torch.cuda.synchronize)
    ops.check_status()
    for _ in range(12):
        got = [one_pass() for _ in range(3)]
        ops.check_status()
        for run, dq in got:
            assert all(torch.equal(a, b) for a, b in zip(run, want))
            for a, b in zip(dq, want_dq):
                assert (a.double() - b.double()).norm() <= 4 * G.O.HALF_STEP * b.double().norm()
