"""The operators around attention where addresses and counts are large, on several streams, in graphs that share nothing,
and over what a caller may do between calls."""

import pytest
import torch

import nanobrain_b200 as nb
from nanobrain_b200 import ops
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).bfloat16()


def weights(dim, hidden, seed=1):
    return (randn(hidden, dim, seed=seed, std=dim ** -0.5), randn(hidden, dim, seed=seed + 1, std=dim ** -0.5),
            randn(dim, hidden, seed=seed + 2, std=hidden ** -0.5))


def test_rows_farther_apart_than_32_bits():
    # 20 rows of a buffer of 2.6e9 values: the last ones begin behind 2^31 values and 2^32 bytes
    stride = 1 << 27
    big = torch.empty(19 * stride + 4096, dtype=torch.bfloat16, device=DEV)
    small = randn(20, 2, 64, seed=1)
    far = big.as_strided((20, 2, 64), (stride, 64, 1))
    far.copy_(small)
    pos, freqs = torch.arange(20, device=DEV)[:, None], torch.full((1, 32), 0.1, device=DEV)
    outs = []
    for q in (small, far):
        q = q.detach().requires_grad_(True)
        y = nb.qk_norm_rope(q, q, positions=pos, freqs=freqs)
        outs.append((*y, *torch.autograd.grad(y, q, [small, small])))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    x = big.as_strided((20, 64), (stride, 1))
    w = weights(64, 96)
    outs = []
    for rows in (x.contiguous(), x):
        leaf = rows.detach().requires_grad_(True)
        y = nb.gated_mlp(leaf, *w)
        outs.append((y, *torch.autograd.grad(y, leaf, small[:, 0])))
    ops.check_status()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
def test_inner_activations_of_more_than_32_bits(checkpoint):
    # 1.1e6 tokens x 2048 features: h, the checkpoint and da, db hold 2.3e9 values each
    tokens, dim, hidden = 1_100_000, 8, 2048
    x, w = randn(tokens, dim, seed=5), weights(dim, hidden)
    dy = randn(tokens, dim, seed=6)
    leaf = x.requires_grad_(True)
    y = nb.gated_mlp(leaf, *w, checkpoint=checkpoint)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    ops.check_status()
    for part in (slice(0, 300), slice(tokens // 2, tokens // 2 + 300), slice(tokens - 300, tokens)):
        want, grads = O.mlp(x[part], *w, dy=dy[part], bits=int(checkpoint[:-3]))
        assert (y[part].double() - want).norm() <= 2.6 * O.HALF_STEP * want.norm()
        assert (dx[part].double() - grads[0]).norm() <= 2.6 * O.HALF_STEP * grads[0].norm()


def test_more_gradient_tiles_than_units_of_a_wave_and_wide_layers():
    # a wide layer over few tokens: weight gradients are all the work, nothing is cut
    tokens, dim, hidden = 40, 2048, 4104
    args = [randn(tokens, dim, seed=5), *weights(dim, hidden)]
    leaves = [t.requires_grad_(True) for t in args]
    dy = randn(tokens, dim, seed=6)
    y = nb.gated_mlp(*leaves, activation="gelu")
    got = torch.autograd.grad(y, leaves, dy)
    ops.check_status()
    want, grads = O.mlp(*args, activation="gelu", dy=dy)
    for a, b in zip((y, *got), (want, *grads)):
        assert (a.double() - b).norm() <= 2.6 * O.HALF_STEP * b.norm()


def test_two_streams_at_once():
    # independent training steps side by side, many times: each has scratch of its own
    sizes = ((700, 128, 344), (300, 256, 680))
    problems = [([randn(t, d, seed=5), *weights(d, f)], randn(t, d, seed=6)) for t, d, f in sizes]
    q, k = randn(500, 4, 64, seed=7), randn(500, 4, 64, seed=8)

    def step(args, dy):
        leaves = [t.detach().requires_grad_(True) for t in args]
        y = nb.gated_mlp(*leaves, checkpoint="8bit")
        qq = q.detach().requires_grad_(True)
        r = nb.qk_norm_rope(qq, k)
        return (y, *torch.autograd.grad(y, leaves, dy), *r, *torch.autograd.grad(r[0], qq, k))

    want = [step(*p) for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    got = [[] for _ in problems]
    for _ in range(10):
        for i, (stream, p) in enumerate(zip(streams, problems)):
            with torch.cuda.stream(stream):
                got[i].append(step(*p))
    torch.cuda.synchronize()
    ops.check_status()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_two_graphs_replayed_in_turns():
    args, dy = [randn(260, 64, seed=5), *weights(64, 96)], randn(260, 64, seed=6)
    x2 = randn(260, 64, seed=9)

    def step(leaves):
        y = nb.gated_mlp(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    def fresh(x):
        return [t.detach().clone().requires_grad_(True) for t in (x, *args[1:])]

    want = [step(fresh(x)) for x in (args[0], x2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(args[0]))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in (args[0], x2):
        leaves, graph = fresh(x), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(leaves))
        graphs.append((graph, leaves))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    ops.check_status()
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_backward_twice_and_changed_inputs():
    args, dy = [randn(70, 64, seed=5), *weights(64, 96)], randn(70, 64, seed=6)
    leaves = [t.requires_grad_(True) for t in args]
    y = nb.gated_mlp(*leaves)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    second = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    y = nb.gated_mlp(*leaves)
    with torch.no_grad():
        leaves[0].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    # there is no second derivative
    y = nb.gated_mlp(*leaves)
    (g,) = torch.autograd.grad(y, leaves[0], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaves[0])


def test_one_weight_in_two_places():
    x, (w, _, wd) = randn(50, 64, seed=5), weights(64, 96)
    w = w.requires_grad_(True)
    y = nb.gated_mlp(x, w, w, wd)
    (g,) = torch.autograd.grad(y, w, x)
    want, grads = O.mlp(x, w, w, wd, dy=x)
    assert (y.double() - want).norm() <= 2.6 * O.HALF_STEP * want.norm()
    total = grads[1] + grads[2]
    # (their sum is rounded once more)
    assert (g.double() - total).norm() <= 3.6 * O.HALF_STEP * (grads[1].norm() + grads[2].norm())


def test_checkpoints_keep_what_they_say():
    # what is saved from the forward to the backward besides the arguments: 16 bits keep a, b and h, 8 bits a little more
    # than a byte each of a and b (the saved tensors' own sizes: the allocator's count has its blocks' slack in it)
    tokens, dim, hidden = 8192, 256, 1024
    x, w = randn(tokens, dim, seed=5), [t.requires_grad_(True) for t in weights(dim, hidden)]
    arguments = {t.data_ptr() for t in (x, *w)}
    for checkpoint, want in (("16bit", 6.125), ("8bit", 2.125)):
        kept = []

        def pack(t):
            if t.data_ptr() not in arguments:
                kept.append(t.numel() * t.element_size())
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            nb.gated_mlp(x, *w, checkpoint=checkpoint)
        assert sum(kept) == want * tokens * hidden


def test_a_run_of_both_with_attention():
    # a pre-norm block written out: norms and rotation, attention over packed sequences, gated MLP, a step of each gradient
    torch.manual_seed(0)
    t, h, hidden = 300, 2, 344
    cu = torch.tensor([0, 1, 150, 150, 290], dtype=torch.int32, device=DEV)   # (ten rows of padding behind)
    pos, freqs = torch.randint(0, 9, (t, 3), device=DEV), torch.rand(3, 32, device=DEV)
    wq = [randn(128, 128, seed=s, std=0.09).requires_grad_(True) for s in (1, 2, 3)]
    ws = [w.requires_grad_(True) for w in weights(128, hidden, seed=10)]
    norms = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    x = randn(t, 128, seed=5).requires_grad_(True)
    dy = randn(t, 128, seed=6)

    q, k, v = ((x @ w.t()).view(t, h, 64) for w in wq)
    q, k = nb.qk_norm_rope(q, k, *norms, positions=pos, freqs=freqs)
    a = nb.sdpa_varlen(q, k, v, cu, cu, 160, 160).reshape(t, 128)
    y = nb.gated_mlp(a, *ws, checkpoint="8bit")
    leaves = [x, *wq, *norms, *ws]
    got = torch.autograd.grad(y, leaves, dy)
    ops.check_status()
    assert not y[290:].any()

    ref = [p.detach().double().requires_grad_(True) for p in leaves]
    q, k, v = ((ref[0] @ w.t()).view(t, h, 64) for w in ref[1:4])
    theta = O.angles(pos, freqs, False)
    q, k = (O.norm_rope(z, w, theta, 1e-6, False)[0] for z, w in ((q, ref[4]), (k, ref[5])))
    rows = []
    for lo, hi in zip(cu[:-1].tolist(), cu[1:].tolist()):
        p = torch.softmax(q[lo:hi].transpose(0, 1) @ k[lo:hi].permute(1, 2, 0) / 8, -1)
        rows.append((p @ v[lo:hi].transpose(0, 1)).transpose(0, 1))
    a = torch.cat(rows + [torch.zeros(10, h, 64, dtype=torch.float64, device=DEV)]).reshape(t, 128)
    out = (O.act(a @ ref[6].t(), "silu") * (a @ ref[7].t())) @ ref[8].t()
    want = torch.autograd.grad(out, ref, dy.double())
    # some ten roundings on the way, and 8 bits of a and b: half a step of 1/127 of a group's largest value, 0.25 % of it,
    # which is about 2.2 times the rms: 0.6 % of a and of b
    for g, r in zip((y, *got), (out, *want)):
        assert (g.double() - r).norm() <= (12 * O.HALF_STEP + 2 * 0.006) * r.norm()
