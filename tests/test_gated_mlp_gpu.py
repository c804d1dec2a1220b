"""``gated_mlp`` against its definition in 64 bits: sizes around its tiles, both activations and checkpoints, biases,
layouts, forward and every gradient."""

import math

import pytest
import torch

import nanobrain_b200 as nb
from nanobrain_b200 import ops
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def randn(*shape, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).bfloat16()


def problem(tokens, dim, hidden, bias, seed=0):
    std = 1 / math.sqrt(dim)
    x = randn(tokens, dim, seed=seed)
    w = [randn(hidden, dim, seed=seed + 1, std=std), randn(hidden, dim, seed=seed + 2, std=std),
         randn(dim, hidden, seed=seed + 3, std=1 / math.sqrt(hidden))]
    b = [randn(n, seed=seed + 4 + i, std=0.5) for i, n in enumerate((hidden, hidden, dim))] if bias else [None] * 3
    return x, *w, *b


def close(got, want, roundings, name=""):
    """``roundings`` to bf16 on the way, each at most half a step of what is rounded; they are independent of what
    they are multiplied with, so each moves the result's norm by about half a step of it at most. fp32 sums add less than a tenth."""
    assert got.shape == want.shape and got.dtype == torch.bfloat16, name
    off = (got.double() - want).norm()
    assert off <= (roundings + 0.1) * O.HALF_STEP * want.norm() + 1e-30, (name, (off / want.norm()).item())
    # and no single value far off: eight times what that is per value, next to its own rounding
    rms = want.square().mean().sqrt()
    far = (got.double() - want).abs() - O.HALF_STEP * want.abs()
    assert (far <= 8 * roundings * O.HALF_STEP * rms + 1e-30).all(), (name, (far.max() / rms).item())


def run(args, dy, activation="silu", checkpoint="16bit"):
    leaves = [t.detach().requires_grad_(True) for t in args if t is not None]
    it = iter(leaves)
    full = [None if t is None else next(it) for t in args]
    y = nb.gated_mlp(*full, activation=activation, checkpoint=checkpoint)
    grads = torch.autograd.grad(y, leaves, dy)
    ops.check_status()
    return (y.detach(), *grads)


def compare(args, activation, checkpoint, got, dy):
    y, grads = O.mlp(*args, activation=activation, dy=dy, bits=int(checkpoint[:-3]))
    want = (y, *[g for g, t in zip(grads, args) if t is not None])
    names = [n for n, t in zip(NAMES, ("y", *args)) if t is not None]
    for name, a, b in zip(names, got, want):
        # y: h and y. Gradients: da, db or h, and the result; a and b keep 2^-12 (16 bits), or are off by a step now and then
        # where the sum's order decides between two codes (8 bits).
        close(a, b, 2.5, name)


SIZES = [
    # tokens, dim, hidden: one, a tile's edges, widths that end inside a tile, a group, a 16-byte piece
    (1, 64, 64), (2, 8, 8), (9, 16, 40), (127, 64, 136), (128, 128, 128), (129, 72, 264), (198, 128, 344),
    (300, 264, 72), (513, 200, 520), (1000, 512, 1368),
]


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
@pytest.mark.parametrize("activation,bias", [("silu", False), ("gelu", True)])
@pytest.mark.parametrize("tokens,dim,hidden", SIZES)
def test_training_against_64_bits(tokens, dim, hidden, activation, bias, checkpoint):
    args = problem(tokens, dim, hidden, bias)
    dy = randn(tokens, dim, seed=9, std=0.1)
    compare(args, activation, checkpoint, run(args, dy, activation, checkpoint), dy)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 100, 700])
@pytest.mark.parametrize("dim,hidden,activation,bias", [(768, 2048, "silu", False), (264, 72, "gelu", True), (8, 16, "silu", True),
                                                        (2320, 1000, "silu", True)])
def test_inference_against_64_bits(tokens, dim, hidden, activation, bias):
    args = problem(tokens, dim, hidden, bias)
    with torch.inference_mode():
        y = nb.gated_mlp(*args, activation=activation)
    ops.check_status()
    close(y, O.mlp(*args, activation=activation)[0], 2)
    with torch.no_grad():
        assert torch.equal(nb.gated_mlp(*args, activation=activation, checkpoint="8bit"), y)


@pytest.mark.parametrize("tokens", [17, 129, 300, 500, 1200, 2000, 3000])
@pytest.mark.parametrize("dim,hidden", [(1024, 2736), (512, 1368), (128, 344)])
def test_inference_in_every_tiling(tokens, dim, hidden):
    # single CTAs and pairs, tiles of 64 to 256 columns, in launches that follow on one another
    args = problem(tokens, dim, hidden, False)
    with torch.inference_mode():
        calls = [nb.gated_mlp(*args) for _ in range(4)]
    ops.check_status()
    close(calls[0], O.mlp(*args)[0], 2)
    assert all(torch.equal(calls[0], y) for y in calls)


@pytest.mark.parametrize("tokens,dim,hidden", [(20000, 64, 72), (6000, 256, 680), (2500, 768, 2048)])
def test_many_tokens_twice_the_same_bits(tokens, dim, hidden):
    # weight gradients over many tokens (products cut into parts), more tiles than CTAs
    args = problem(tokens, dim, hidden, True)
    dy = randn(tokens, dim, seed=9, std=0.1)
    first, second = run(args, dy, checkpoint="8bit"), run(args, dy, checkpoint="8bit")
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    compare(args, "silu", "8bit", first, dy)
    compare(args, "silu", "16bit", run(args, dy), dy)


def test_shapes_and_strides():
    args = problem(60, 64, 96, True)
    x, wg, wu, wd, bg, bu, bd = args
    dy = randn(60, 64, seed=9)
    want = run(args, dy)
    wide = torch.cat((x, x), 1)
    both = torch.cat((wg, wu), 0)          # one parameter for both projections
    odd = torch.cat((wd, wd), 1)[:, 1:97].clone()
    views = (wide[:, :64], both[:96], both[96:], torch.cat((wd, wd), 1)[:, :96], bg, bu, bd)
    for a, b in zip(run(views, dy), want):
        assert torch.equal(a, b)
    shifted = torch.cat((x.new_zeros(60, 1), x), 1)[:, 1:]   # rows that start at odd places: copied
    for a, b in zip(run((shifted, wg.t().contiguous().t(), *args[2:]), dy), want):
        assert torch.equal(a, b)
    x4 = x.view(2, 3, 10, 64).requires_grad_(True)
    y = nb.gated_mlp(x4, *args[1:])
    assert y.shape == x4.shape and torch.equal(y.view(60, 64), want[0])
    (dx,) = torch.autograd.grad(y, x4, dy.view(2, 3, 10, 64).transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(dx.view(60, 64), want[1])
    y1 = nb.gated_mlp(x[0].detach(), *args[1:])
    assert y1.shape == (64,)
    assert odd.shape == wd.shape


def test_no_tokens():
    args = problem(0, 64, 96, True)
    got = run(args, args[0].clone())
    assert got[0].shape == (0, 64) and got[1].shape == (0, 64)
    assert all(not g.any() for g in got[2:])
    assert nb.gated_mlp(args[0].view(0, 5, 64) if False else args[0].view(5, 0, 64), *args[1:]).shape == (5, 0, 64)


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
@pytest.mark.parametrize("wanted", [(0,), (1,), (3,), (0, 3), (1, 2), (4,), (6,), (2, 5, 6)])
def test_some_gradients_alone(wanted, checkpoint):
    args = problem(140, 64, 96, True)
    dy = randn(140, 64, seed=9)
    want = run(args, dy, checkpoint=checkpoint)
    full = [t.detach() for t in args]
    for i in wanted:
        full[i].requires_grad_(True)
    y = nb.gated_mlp(*full, checkpoint=checkpoint)
    grads = torch.autograd.grad(y, [full[i] for i in wanted], dy)
    for i, g in zip(wanted, grads):
        close(g, want[1 + i].double(), 1)


@pytest.mark.parametrize("missing", [4, 5, 6])
def test_some_biases(missing):
    args = list(problem(70, 64, 96, True))
    args[missing] = None
    dy = randn(70, 64, seed=9)
    compare(args, "silu", "16bit", run(args, dy), dy)
    with torch.inference_mode():
        close(nb.gated_mlp(*[t if t is None else t[:3] if i == 0 else t for i, t in enumerate(args)]),
              O.mlp(args[0][:3], *args[1:])[0], 2)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_wide_range(activation):
    # tokens from 1e-20 to 100 times the usual size, one of zeros: every token's gradient and result by its own norm
    args = list(problem(12, 64, 96, False))
    scale = torch.tensor([1e-20, 1e-6, 1e-3, 0.1, 1, 3, 10, 30, 100, 0, 1, 1], device=DEV)
    args[0] = (args[0].float() * scale[:, None]).bfloat16()
    dy = randn(12, 64, seed=9)
    got = run(args, dy, activation)
    y, grads = O.mlp(*args, activation=activation, dy=dy)
    for t in range(12):
        # (values below bf16's and fp32's normal range have no relative accuracy)
        assert (got[0][t].double() - y[t]).norm() <= 2.5 * O.HALF_STEP * y[t].norm() + 1e-36
        assert (got[1][t].double() - grads[0][t]).norm() <= 2.5 * O.HALF_STEP * grads[0][t].norm() + 1e-36


def test_values_that_are_not_finite_stay_in_their_token():
    args = list(problem(200, 64, 96, False))
    args[0][5, 3], args[0][140, 9] = float("nan"), float("inf")
    dy = randn(200, 64, seed=9)
    fine = torch.ones(200, dtype=torch.bool, device=DEV)
    fine[[5, 140]] = False
    clean = [t if t is None else t.clone() for t in args]
    clean[0][~fine] = 0
    for checkpoint in ("16bit", "8bit"):
        got, want = run(args, dy, checkpoint=checkpoint), run(clean, dy, checkpoint=checkpoint)
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a[fine], b[fine]) and torch.isnan(a[5]).all()
            assert not torch.isfinite(a[140]).all()
        assert torch.isnan(got[2]).any()
    with torch.inference_mode():
        y = nb.gated_mlp(args[0][3:8], *args[1:])
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]].float()).all()


def test_saturated_activations():
    # a of +-200 and beyond: silu and gelu are a or 0, their slopes 1 or 0, nothing is NaN
    x = torch.full((3, 8), 10.0, device=DEV).bfloat16()
    x[1] = -10
    x[2] = 1e4
    wg, wu, wd = torch.ones(8, 8, device=DEV).bfloat16() * 4, torch.eye(8, device=DEV).bfloat16(), torch.eye(8, device=DEV).bfloat16()
    dy = torch.ones(3, 8, device=DEV).bfloat16()
    for activation in ("silu", "gelu"):
        for checkpoint in ("16bit", "8bit"):
            got = run((x, wg, wu, wd, None, None, None), dy, activation, checkpoint)
            y, grads = O.mlp(x, wg, wu, wd, activation=activation, dy=dy, bits=int(checkpoint[:-3]))
            assert all(torch.isfinite(t.float()).all() for t in got)
            close(got[0], y, 2)
            close(got[1], grads[0], 2.5)


def test_gradient_against_differences():
    args = problem(64, 64, 96, True)
    dy = randn(64, 64, seed=9)
    grads = run(args, dy)[1:]
    with torch.no_grad():
        y = nb.gated_mlp(*args)
        # two losses of 4096 values off by two roundings each
        noise = 2 * 2 * O.HALF_STEP * (dy.double() * y.double().abs().mean()).norm() * math.sqrt(2)
        for i, (leaf, grad) in enumerate(zip(args, grads)):
            step = (grad.float() * (0.1 * leaf.float().norm() / grad.float().norm())).bfloat16()
            up, down = list(args), list(args)
            up[i], down[i] = leaf + step, leaf - step
            diff = ((nb.gated_mlp(*up).double() - nb.gated_mlp(*down).double()) * dy.double()).sum()
            want = (grad.double() * (up[i].double() - down[i].double())).sum()
            # steps of a tenth: the third derivative adds some 0.1^2 of the first
            assert (diff - want).abs() <= noise + 0.02 * want.abs(), NAMES[1 + i]


def test_other_stream_and_captured():
    args = problem(300, 64, 96, True)
    with torch.no_grad():
        want = nb.gated_mlp(*args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = nb.gated_mlp(*args)
        side.synchronize()
        assert torch.equal(got, want)
    # a whole step captured, replayed on other inputs
    leaves = [t.clone().requires_grad_(True) for t in args]
    dy = randn(300, 64, seed=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(nb.gated_mlp(*leaves, checkpoint="8bit"), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = nb.gated_mlp(*leaves, checkpoint="8bit")
        grads = torch.autograd.grad(y, leaves, dy)
    other = problem(300, 64, 96, True, seed=50)
    with torch.no_grad():
        for a, b in zip(leaves, other):
            a.copy_(b)
    graph.replay()
    for a, b in zip((y, *grads), run(other, dy, checkpoint="8bit")):
        assert torch.equal(a.detach(), b)


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
def test_opcheck_and_flops(checkpoint):
    from torch.utils.flop_counter import FlopCounterMode

    args = [t.requires_grad_(True) for t in problem(20, 64, 96, True)]
    code = {"16bit": 1, "8bit": 2}[checkpoint]
    torch.library.opcheck(torch.ops.nanobrain_b200.gated_mlp_fwd.default, (*args, 0, code))
    dy = randn(20, 64, seed=9)
    with FlopCounterMode(display=False) as counter:
        y = nb.gated_mlp(*args, checkpoint=checkpoint)
        torch.autograd.grad(y, args, dy)
    assert counter.get_total_flops() == 18 * 20 * 64 * 96


def test_what_is_refused():
    x, wg, wu, wd, bg, bu, bd = problem(10, 64, 96, True)
    bad = [
        ((x.float(), wg, wu, wd), "bfloat16"),
        ((x, wg.float(), wu, wd), "bfloat16"),
        ((x, wg.cpu(), wu, wd), "CUDA"),
        ((x[:, :56].contiguous(), wg, wu, wd), "dim of x"),
        ((x, wg, wu[:64], wd), "dim of x"),
        ((x, wg, wu, wd.t()), "w_down"),
        ((x[:, :60], wg[:, :60], wu[:, :60], wd[:60]), "multiples of 8"),
        ((x, wg[:90], wu[:90], wd[:, :90]), "multiples of 8"),
        ((x, wg, wu, wd, bg[:64]), "b_gate"),
        ((x, wg, wu, wd, bg, bu, bd.float()), "b_down"),
    ]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            nb.gated_mlp(*args)
    with pytest.raises(ValueError, match="activation"):
        nb.gated_mlp(x, wg, wu, wd, activation="relu")
    with pytest.raises(ValueError, match="checkpoint"):
        nb.gated_mlp(x, wg, wu, wd, checkpoint="4bit")
    with pytest.raises(RuntimeError, match="checkpoint"):
        torch.ops.nanobrain_b200.gated_mlp_fwd(x.clone().requires_grad_(True), wg, wu, wd, None, None, None, 0, 0)
