"""``qk_norm_rope`` against its definition in 64 bits: layouts, head counts, positions and orders of pairs, forward,
gradients, and together with the attention that reads its results."""

import math

import pytest
import torch

import nanobrain_b200 as nb
from nanobrain_b200 import ops
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def randn(*shape, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def heads(memory, batch, length, n, seed, std=1.0):
    if memory == "packed":
        return randn(length, n, 64, seed=seed, std=std)
    if memory == "blhd":
        return randn(batch, length, n, 64, seed=seed, std=std).transpose(1, 2)
    if memory == "qkv":  # one projection for all three: strided rows
        return randn(batch, length, 3, n, 64, seed=seed, std=std)[:, :, 1].transpose(1, 2)
    if memory == "odd":  # rows at strides that are no multiple of 8: copied
        return randn(batch, n, length, 65, seed=seed, std=std)[..., :64]
    return randn(batch, n, length, 64, seed=seed, std=std)


def frequencies(axes, span=64.0):
    pair = torch.arange(32)
    per = -(-32 // axes)
    f = torch.zeros(axes, 32, dtype=torch.float64)
    f[pair // per, pair] = span ** (-(pair % per).double() / per)
    return f.float().to(DEV)


def check(x, w, theta, interleaved, y, dy=None, dx=None, dw=None, eps=EPS):
    """Errors against 64 bits. Forward: half a step of bf16, and 2e-6 of the pair for fp32 (the root's 2^-22, three products'
    2^-24 each, cosine and sine to 2e-7). Backward: the same, plus sums of 64 products, 2^-18 of the sum of their
    magnitudes. dw: a lane adds fewer than 64 terms in a row before the tree sums (2^-18), and each term is off by 3e-6."""
    ref, n = O.norm_rope(x, w, theta, eps, interleaved)
    lo, hi = O.split_pairs(n.abs(), interleaved)
    pair = O.join_pairs(lo + hi, lo + hi, interleaved)
    assert ((y.double() - ref).abs() <= O.HALF_STEP * ref.abs() + 2e-6 * pair + 1e-37).all()
    if dy is None:
        return
    x64 = x.double().requires_grad_(True)
    w64 = (torch.ones(64, device=DEV) if w is None else w.detach()).double().requires_grad_(True)
    out, _ = O.norm_rope(x64, w64, theta, eps, interleaved)
    want_x, want_w = torch.autograd.grad(out, (x64, w64), dy.double())
    r = 1 / (x64.detach().square().mean(-1, keepdim=True) + eps).sqrt()
    lo, hi = O.split_pairs(dy.double().abs(), interleaved)
    dn = O.join_pairs(lo + hi, lo + hi, interleaved)  # bounds |dn| and what its error is relative to
    g = dn * w64.detach().abs()
    xr = (x64.detach() * r).abs()
    size = r * (g + xr * (g * xr).mean(-1, keepdim=True))
    assert ((dx.double() - want_x).abs() <= O.HALF_STEP * want_x.abs() + (2.0 ** -18 + 4e-6) * size + 1e-37).all()
    terms = (dn * xr).reshape(-1, 64) if x.dim() == 3 else (dn * xr).transpose(1, 2).reshape(-1, 64)
    if dw is not None:
        off = dw.double() - want_w
        assert (off.abs() <= O.HALF_STEP * (dw.dtype == torch.bfloat16) * want_w.abs() + (2.0 ** -18 + 3e-6) * terms.sum(0)).all()


CASES = [
    # memory, batch, len_q, len_k, heads_q, heads_k, axes, position type, interleaved, weights' type
    ("packed", 1, 1, 1, 12, 12, 3, torch.int64, False, torch.float32),
    ("packed", 1, 517, 517, 12, 12, 3, torch.int64, True, torch.float32),
    ("packed", 1, 100, 37, 2, 5, 1, torch.int32, False, torch.bfloat16),
    ("packed", 1, 64, 64, 1, 1, 0, None, False, None),
    ("packed", 1, 33, 33, 17, 3, 4, torch.float32, True, torch.float32),
    ("blhd", 2, 129, 129, 12, 12, 3, torch.int64, False, torch.float32),
    ("blhd", 3, 7, 50, 8, 8, 2, torch.float32, False, torch.bfloat16),
    ("bhld", 2, 65, 65, 16, 16, 3, torch.int32, True, torch.float32),
    ("bhld", 5, 1, 1, 40, 33, 0, None, True, torch.float32),
    ("qkv", 2, 31, 31, 12, 12, 3, torch.int64, False, torch.float32),
    ("odd", 2, 9, 9, 3, 3, 2, torch.int64, False, torch.float32),
]


@pytest.mark.parametrize("memory,batch,lq,lk,hq,hk,axes,ptype,interleaved,wtype", CASES)
def test_against_64_bits(memory, batch, lq, lk, hq, hk, axes, ptype, interleaved, wtype):
    dense = memory != "packed"
    q = heads(memory, batch, lq, hq, 1, 2.0).requires_grad_(True)
    k = heads(memory, batch, lk, hk, 2, 0.1).requires_grad_(True)
    qw = None if wtype is None else (1 + randn(64, seed=3, std=0.3, dtype=torch.float32)).to(wtype).requires_grad_(True)
    kw = None if wtype is None else (1 + randn(64, seed=4, std=0.3, dtype=torch.float32)).to(wtype).requires_grad_(True)
    freqs = frequencies(axes) if axes else None

    def positions(length, seed):
        if not axes:
            return None
        g = torch.Generator(device=DEV).manual_seed(seed)
        shape = (batch, length, axes) if dense else (length, axes)
        return torch.randint(-40, 40, shape, generator=g, device=DEV).to(ptype)

    pos, kpos = positions(lq, 5), positions(lk, 6) if lk != lq else None
    yq, yk = nb.qk_norm_rope(q, k, qw, kw, pos, freqs, kpos, eps=EPS, interleaved=interleaved)
    dyq, dyk = heads(memory, batch, lq, hq, 7), heads(memory, batch, lk, hk, 8, 0.01)
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    grads = torch.autograd.grad((yq, yk), leaves, (dyq, dyk))
    tq = O.angles(pos, freqs, dense)
    tk = tq if kpos is None else O.angles(kpos, freqs, dense)
    check(q.detach(), qw, tq, interleaved, yq.detach(), dyq, grads[0], grads[2] if qw is not None else None)
    check(k.detach(), kw, tk, interleaved, yk.detach(), dyk, grads[1], grads[3] if kw is not None else None)
    for y, x, w in ((yq, q, qw), (yk, k, kw)):
        assert y.shape == x.shape and y.dtype == torch.bfloat16
        assert y.stride()[-1] == 1 and (not dense or y.transpose(1, 2).is_contiguous())
    with torch.inference_mode():
        again = nb.qk_norm_rope(q, k, qw, kw, pos, freqs, kpos, eps=EPS, interleaved=interleaved)
    assert torch.equal(again[0], yq) and torch.equal(again[1], yk)


def test_positions_shared_by_the_batch_and_strided():
    q, k = heads("blhd", 4, 50, 3, 1), heads("blhd", 4, 50, 3, 2)
    freqs = frequencies(3)
    pos = torch.randint(0, 16, (50, 3), device=DEV)
    whole = nb.qk_norm_rope(q, k, positions=pos.expand(4, -1, -1).contiguous(), freqs=freqs)
    for p in (pos, pos.expand(4, -1, -1), torch.cat((pos, pos), 1)[:, :3], pos.t().contiguous().t()):
        got = nb.qk_norm_rope(q, k, positions=p, freqs=freqs)
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


@pytest.mark.parametrize("ptype,far", [(torch.int64, 1 << 40), (torch.int32, (1 << 31) - 100), (torch.float32, 1 << 24)])
def test_far_positions(ptype, far):
    # angles of 10^6 turns and more: the fraction of a turn has to survive. (2^40 x freq: 64 bits leave 2^-13.)
    q, k = heads("packed", 1, 40, 2, 1), heads("packed", 1, 40, 2, 2)
    freqs = frequencies(1, 1e4)
    pos = (far - torch.arange(40, device=DEV)[:, None]).to(ptype)
    yq, yk = nb.qk_norm_rope(q, k, positions=pos, freqs=freqs)
    a = pos.double() @ freqs.double()
    turns = a / (2 * math.pi)
    slack = 4 * a.abs().max() * 2.0 ** -52  # of an angle in 64 bits, here and there
    for y, x in ((yq, q), (yk, k)):
        ref, n = O.norm_rope(x, None, ((turns - turns.round()) * 2 * math.pi)[:, None, :], EPS, False)
        lo, hi = O.split_pairs(n.abs(), False)
        pair = O.join_pairs(lo + hi, lo + hi, False)
        assert ((y.double() - ref).abs() <= O.HALF_STEP * ref.abs() + (2e-6 + slack) * pair).all()


def test_values_that_are_zero_tiny_huge_or_not_finite():
    q = heads("packed", 1, 8, 2, 1)
    q[0] = 0
    q[1] *= 1e-30   # the square underflows: eps decides
    q[2] *= 1e15
    q[3, 0, 5] = float("nan")
    q[4, 1, 7] = float("inf")
    pos, freqs = torch.arange(8, device=DEV)[:, None], frequencies(1)
    y, other = nb.qk_norm_rope(q, q.clone(), positions=pos, freqs=freqs)
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    rows = [0, 1, 2, 5, 6, 7]
    check(q[rows], None, O.angles(pos[rows], freqs, False), False, y[rows])
    assert torch.isnan(y[3, 0]).all() and torch.isfinite(y[3, 1]).all()
    assert torch.isnan(y[4, 1]).any() and torch.isfinite(y[4, 0]).all()
    assert torch.equal(torch.isnan(y), torch.isnan(other))
    # a gradient that is not finite stays in its own side's weight
    qq, kk = (heads("packed", 1, 8, 2, s).requires_grad_(True) for s in (1, 2))
    w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    dyq, dyk = torch.ones_like(qq), torch.ones_like(kk)
    dyk[3, 1, 9] = float("nan")
    g = torch.autograd.grad(nb.qk_norm_rope(qq, kk, *w, positions=pos, freqs=freqs), (qq, kk, *w), (dyq, dyk))
    assert torch.isfinite(g[0]).all() and torch.isfinite(g[2]).all() and torch.isnan(g[3]).any()
    assert torch.isfinite(g[1][:3]).all() and torch.isnan(g[1][3, 1]).any()


def test_gradient_against_differences():
    q = heads("packed", 1, 60, 2, 1).requires_grad_(True)
    k = heads("packed", 1, 60, 2, 2).requires_grad_(True)
    w = [(1 + randn(64, seed=s, std=0.3, dtype=torch.float32)).requires_grad_(True) for s in (3, 4)]
    pos, freqs = torch.randint(0, 16, (60, 3), device=DEV), frequencies(3)
    dy = [heads("packed", 1, 60, 2, s) for s in (5, 6)]

    def loss(q, k, w):
        y = nb.qk_norm_rope(q, k, *w, positions=pos, freqs=freqs)
        return sum((a.double() * b.double()).sum() for a, b in zip(y, dy))

    grads = torch.autograd.grad(nb.qk_norm_rope(q, k, *w, positions=pos, freqs=freqs), (q, k, *w), dy)
    with torch.no_grad():
        # noise: two losses of 2 x 7680 rounded values, each off by at most half a step of a value near 1 (rms 2^-8 / sqrt 3)
        noise = 2 * math.sqrt(2 * 7680) * O.HALF_STEP
        for i, leaf in enumerate((q, k, *w)):
            step = grads[i] * (0.05 * leaf.float().norm() / grads[i].float().norm()).to(grads[i].dtype)
            args = [[q, k, *w], [q, k, *w]]
            args[0][i], args[1][i] = leaf + step, leaf - step
            moved = (args[0][i].double() - args[1][i].double())
            diff = loss(*args[0][:2], args[0][2:]) - loss(*args[1][:2], args[1][2:])
            want = (grads[i].double() * moved).sum()
            # steps of 5 %: the third derivative adds some 0.05^2 of the first
            assert (diff - want).abs() <= noise + 0.01 * want.abs(), i


def test_one_side_alone_and_unused_gradients():
    q, k = heads("packed", 1, 30, 2, 1).requires_grad_(True), heads("packed", 1, 30, 2, 2)
    w = torch.ones(64, device=DEV, requires_grad=True)
    yq, yk = nb.qk_norm_rope(q, k, w)
    dq, dw = torch.autograd.grad(yq, (q, w), torch.ones_like(yq))
    check(q.detach(), w, None, False, yq.detach(), torch.ones_like(yq), dq, dw)
    k2 = k.clone().requires_grad_(True)
    yq, yk = nb.qk_norm_rope(q.detach(), k2)
    (dk,) = torch.autograd.grad(yk.sum(), k2)  # an expanded gradient
    check(k, None, None, False, yk.detach(), torch.ones_like(yk), dk)


@pytest.mark.parametrize("lq,lk", [(0, 0), (0, 5), (5, 0)])
def test_no_tokens(lq, lk):
    q, k = (heads("packed", 1, n, 2, 1).requires_grad_(True) for n in (lq, lk))
    w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    freqs = frequencies(1)
    pos, kpos = (torch.arange(n, device=DEV)[:, None] for n in (lq, lk))
    y = nb.qk_norm_rope(q, k, *w, positions=pos, freqs=freqs, k_positions=kpos)
    g = torch.autograd.grad(y, (q, k, *w), [torch.ones_like(t) for t in y])
    assert y[0].shape == q.shape and y[1].shape == k.shape and g[0].shape == q.shape
    for x, yy, dx, dw, p, ww in zip((q, k), y, g[:2], g[2:], (pos, kpos), w):
        check(x.detach(), ww, O.angles(p, freqs, False), False, yy.detach(), torch.ones_like(yy), dx, dw)


def test_many_tokens_in_turns():
    # more tokens than one round of warps; results do not depend on the launch, and twice the same bits
    q, k = heads("packed", 1, 9001, 3, 1).requires_grad_(True), heads("packed", 1, 9001, 3, 2).requires_grad_(True)
    w = [(1 + randn(64, seed=s, std=0.3, dtype=torch.float32)).requires_grad_(True) for s in (3, 4)]
    pos, freqs = torch.randint(0, 30, (9001, 3), device=DEV), frequencies(3)
    dy = [heads("packed", 1, 9001, 3, s) for s in (5, 6)]
    runs = []
    for _ in range(2):
        y = nb.qk_norm_rope(q, k, *w, positions=pos, freqs=freqs)
        runs.append((*y, *torch.autograd.grad(y, (q, k, *w), dy)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    theta = O.angles(pos, freqs, False)
    check(q.detach(), w[0], theta, False, runs[0][0].detach(), dy[0], runs[0][2], runs[0][4])
    check(k.detach(), w[1], theta, False, runs[0][1].detach(), dy[1], runs[0][3], runs[0][5])


def test_other_stream_and_captured():
    q, k = heads("packed", 1, 300, 4, 1), heads("packed", 1, 300, 4, 2)
    pos, freqs = torch.randint(0, 30, (300, 3), device=DEV), frequencies(3)
    want = nb.qk_norm_rope(q, k, positions=pos, freqs=freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nb.qk_norm_rope(q, k, positions=pos, freqs=freqs)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    q2, k2 = q.clone(), k.clone()
    with torch.cuda.graph(graph):
        held = nb.qk_norm_rope(q2, k2, positions=pos, freqs=freqs)
    q2.copy_(heads("packed", 1, 300, 4, 9))
    graph.replay()
    want = nb.qk_norm_rope(q2, k2, positions=pos, freqs=freqs)
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_opcheck():
    q, k = heads("packed", 1, 30, 2, 1).requires_grad_(True), heads("packed", 1, 30, 2, 2).requires_grad_(True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    args = (q, k, w, w, torch.randint(0, 9, (30, 3), device=DEV), None, frequencies(3), EPS, False)
    torch.library.opcheck(torch.ops.nanobrain_b200.qk_norm_rope_fwd.default, args)


def test_what_is_refused():
    q = heads("packed", 1, 10, 2, 1)
    pos, freqs = torch.zeros(10, 3, dtype=torch.int64, device=DEV), frequencies(3)
    bad = [
        (dict(q=q.float(), k=q), "bfloat16"),
        (dict(q=q[..., :32], k=q), "head_dim"),
        (dict(q=q[0], k=q), r"\[T, H, 64\]"),
        (dict(q=q, k=q[None]), "both"),
        (dict(q=q[None].expand(2, -1, -1, -1), k=q[None]), "batch"),
        (dict(q=q, k=q, positions=pos), "come together"),
        (dict(q=q, k=q, freqs=freqs), "come together"),
        (dict(q=q, k=q[:5], positions=pos, freqs=freqs), "k's"),
        (dict(q=q, k=q, positions=pos[:, :2], freqs=freqs), "axes"),
        (dict(q=q, k=q, positions=pos.double(), freqs=freqs), "int32, int64 or float32"),
        (dict(q=q, k=q, positions=pos, freqs=freqs, k_positions=pos.int()), "one type"),
        (dict(q=q, k=q, positions=pos, freqs=freqs.double()), "freqs"),
        (dict(q=q, k=q, positions=pos, freqs=freqs[:, :16]), "freqs"),
        (dict(q=q, k=q, positions=pos.cpu(), freqs=freqs), "device"),
        (dict(q=q, k=q, positions=pos, freqs=freqs.clone().requires_grad_(True)), "no gradient"),
        (dict(q=q, k=q, q_weight=torch.ones(32, device=DEV)), "q_weight"),
        (dict(q=q, k=q, k_weight=torch.ones(64, device=DEV, dtype=torch.float16)), "k_weight"),
    ]
    for kwargs, text in bad:
        with pytest.raises(RuntimeError, match=text):
            nb.qk_norm_rope(**kwargs)


@pytest.mark.parametrize("dense", [True, False])
def test_in_front_of_attention(dense):
    # as modules use it: norms and rotation, then attention, forward and backward through both
    length, n = 150, 2
    memory = "blhd" if dense else "packed"
    q, k, v = (heads(memory, 2, length, n, s).requires_grad_(True) for s in (1, 2, 3))
    w = [(1 + randn(64, seed=s, std=0.3, dtype=torch.float32)).requires_grad_(True) for s in (4, 5)]
    pos, freqs = torch.randint(0, 16, (length, 3), device=DEV), frequencies(3)
    dy = heads(memory, 2, length, n, 6)
    qq, kk = nb.qk_norm_rope(q, k, *w, positions=pos, freqs=freqs)
    if dense:
        y = nb.sdpa(qq, kk, v)
    else:
        cu = torch.tensor([0, 70, 70, length], dtype=torch.int32, device=DEV)
        y = nb.sdpa_varlen(qq, kk, v, cu, cu, 100, 100)
    leaves = (q, k, v, *w)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    ops.check_status()

    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    theta = O.angles(pos, freqs, dense)
    qr, kr = (O.norm_rope(x, ww, theta, EPS, False)[0] for x, ww in zip(ref[:2], ref[3:]))
    if dense:
        out = torch.softmax(qr @ kr.transpose(-1, -2) / 8, -1) @ ref[2]
    else:
        parts = []
        for lo, hi in ((0, 70), (70, length)):
            a, b, c = (t[lo:hi].transpose(0, 1) for t in (qr, kr, ref[2]))
            parts.append((torch.softmax(a @ b.transpose(-1, -2) / 8, -1) @ c).transpose(0, 1))
        out = torch.cat(parts)
    want = (out, *torch.autograd.grad(out, ref, dy.double()))
    # roundings to bf16 on the way to each: q, k, P, O and, back, dO, dS, dq' and dq: at most eight of half a step
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 8 * O.HALF_STEP * b.norm()
