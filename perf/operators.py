"""The operators of a transformer block around its attention, as cases that can be timed: queries and keys
normed per head and rotated by their positions (``qk_norm_rope``), and the gated feed-forward block
(``gated_mlp``) with its activations kept for the backward pass in 16 or in 8 bits.

``listed()`` are the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes
what a user's program has in hand before the call, ``run(state)`` is one pass: with ``own`` through the
package's public functions, without it in elementary torch operations in 32 bits. ``work(case)`` is what
a pass cannot do without, ``exact(case, seed)`` its result from the definition in 64 bits.

A case is one of

* ``rope``: ``qk_norm_rope`` on ``batch`` x ``seqlen`` tokens of ``heads`` heads with 64 values each.
  ``memory`` is ``packed`` ([T, H, 64]), ``blhd`` (dense, views of the projections' outputs) or ``bhld``
  (dense, contiguous logical order). ``context`` is the number of keys per sequence where they come from
  other tokens than the queries (0: the same). ``axes`` is the number of position coordinates (0: norms
  alone), ``span`` their range, ``interleaved`` which values form a pair.
* ``mlp``: ``gated_mlp`` on ``tokens`` x ``dim`` with ``hidden`` features, ``activation`` silu or gelu, with
  or without ``bias``, ``bits`` of the kept activations.

``train`` cases run forward and backward and return every gradient, the others the forward alone.
"""

import math

import torch

own = False
HEAD_DIM = 64
DEV = "cuda"
EPS = 1e-6
GROUP = 32  # features that share a scale in 8 bits


def _rope(batch, heads, seqlen, train=True, memory="blhd", context=0, axes=3, span=16, interleaved=False):
    return {"kind": "rope", "batch": batch, "heads": heads, "seqlen": seqlen, "train": train, "memory": memory,
            "context": context, "axes": axes, "span": span, "interleaved": interleaved}


def _mlp(tokens, dim, hidden, train=True, activation="silu", bias=False, bits=16):
    return {"kind": "mlp", "tokens": tokens, "dim": dim, "hidden": hidden, "train": train, "activation": activation,
            "bias": bias, "bits": bits}


def listed():
    named = {
        # A class token alone, in ViT-B's heads: nothing but latency.
        "rope_token_infer": _rope(1, 12, 1, train=False, memory="packed"),
        # The CPU-checkable parity configuration in contiguous [B, H, L, 64] memory, pairs side by side.
        "rope_check_train": _rope(2, 12, 820, memory="bhld", interleaved=True),
        # One image per forward, the evaluation loop: all in-mask patches and the class token.
        "rope_image_infer": _rope(1, 12, 3476, train=False),
        # ViT-B encoder attention of one training step over packed tokens: 32 volumes, 80 % of the patches masked.
        "rope_encoder_train": _rope(1, 12, 26253, memory="packed"),
        # Decoder attention over the full grid of 4096 patches, the largest call.
        "rope_decoder_train": _rope(32, 8, 4096),
        # One token through the block of ViT-B: the weights are read once and that is all.
        "mlp_token_infer": _mlp(1, 768, 2048, train=False),
        # The tests' tiny model (6 sequences of a class token and 32 patches): launches and host work.
        "mlp_tiny_train": _mlp(198, 128, 344, bias=True),
        # One image of the evaluation loop.
        "mlp_image_infer": _mlp(3476, 768, 2048, train=False, activation="gelu", bias=True),
        # The ViT-B encoder's training step, activations kept in 16 and in 8 bits.
        "mlp_encoder_train": _mlp(26253, 768, 2048),
        "mlp_encoder_8bit_train": _mlp(26253, 768, 2048, bias=True, bits=8),
        # ViT-L-style encoder on the 20 x 24 x 20 grid.
        "mlp_vitl_train": _mlp(30731, 1024, 2736, activation="gelu"),
        # The decoder's training step over the full grid: the most tokens, whose activations are worth keeping small.
        "mlp_decoder_8bit_train": _mlp(32 * 4096, 512, 1368, bits=8),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case: tokens over the logarithm of their range, widths as the configurations have them or any
    multiple of eight; never more work than the largest listed case of its kind."""
    most = {c["kind"]: work(c) for c in listed()}  # (the last of each kind is the largest)
    while True:
        train = rng.random() < 0.7
        if rng.random() < 0.45:
            memory = rng.choice(("packed", "blhd", "bhld"))
            batch = 1 if memory == "packed" else _log_int(rng, 1, 64)
            axes = rng.choice((0, 1, 2, 3, 3))
            case = _rope(batch, rng.choice((1, 2, 3, 8, 12, 16)), _log_int(rng, 1, 140000 // batch), train, memory,
                         rng.choice((0, 0, 0, _log_int(rng, 1, 140000 // batch))), axes,
                         _log_int(rng, 8, 1 << 20 if axes == 1 else 64), rng.random() < 0.5)
        else:
            dim = rng.choice((128, 512, 768, 1024, 8 * _log_int(rng, 2, 160)))
            hidden = rng.choice(((dim * 8 // 3 + 7) // 8 * 8, dim * 2, 8 * _log_int(rng, 2, 400)))
            case = _mlp(_log_int(rng, 1, 140000), dim, hidden, train, rng.choice(("silu", "gelu")),
                        rng.random() < 0.5, rng.choice((8, 16)) if train else 16)
        w, top = work(case), most[case["kind"]]
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return case


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------
def _frequencies(axes, span):
    """[axes, 32]: the 32 pairs of a head dealt out to the axes, each axis with a geometric series of frequencies
    from 1 down to about 1 / span."""
    freqs = torch.zeros(axes, HEAD_DIM // 2, dtype=torch.float64)
    pair = torch.arange(HEAD_DIM // 2)
    per = -(-(HEAD_DIM // 2) // axes)
    freqs[pair // per, pair] = float(span) ** (-(pair % per).to(torch.float64) / per)
    return freqs.to(device=DEV, dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16, mean=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)

    s = {"case": case}
    if case["kind"] == "rope":
        b, h, lq = case["batch"], case["heads"], case["seqlen"]
        lk = case["context"] or lq

        def heads(length, std):
            if case["memory"] == "packed":
                return normal(length, h, HEAD_DIM, std=std)
            if case["memory"] == "blhd":
                return normal(b, length, h, HEAD_DIM, std=std).transpose(1, 2)
            return normal(b, h, length, HEAD_DIM, std=std)

        def positions(length):
            shape = (length,) if case["memory"] == "packed" else (b, length)
            return torch.randint(0, case["span"], shape + (case["axes"],), generator=g, device=DEV)

        s["q"], s["k"] = heads(lq, 1.5), heads(lk, 0.7)
        # The norms' weights are parameters: in 32 bits under autocast.
        s["q_weight"] = normal(HEAD_DIM, std=0.2, mean=1.0, dtype=torch.float32)
        s["k_weight"] = normal(HEAD_DIM, std=0.2, mean=1.0, dtype=torch.float32)
        s["positions"] = positions(lq) if case["axes"] else None
        s["k_positions"] = positions(lk) if case["axes"] and case["context"] else None
        s["freqs"] = _frequencies(case["axes"], case["span"]) if case["axes"] else None
        s["leaves"] = ["q", "k", "q_weight", "k_weight"]
        if case["train"]:
            s["grads"] = [heads(lq, 0.01), heads(lk, 0.01)]
    else:
        t, d, f = case["tokens"], case["dim"], case["hidden"]
        std = math.sqrt(2.0 / (d + f))
        s["x"] = normal(t, d)  # behind a layer norm
        s["w_gate"], s["w_up"] = normal(f, d, std=std), normal(f, d, std=std)
        s["w_down"] = normal(d, f, std=std)
        s["leaves"] = ["x", "w_gate", "w_up", "w_down"]
        for name, size in (("b_gate", f), ("b_up", f), ("b_down", d)):
            s[name] = normal(size, std=0.1) if case["bias"] else None
            s["leaves"] += [name] if case["bias"] else []
        if case["train"]:
            s["grads"] = [normal(t, d, std=0.01)]
    if case["train"]:
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain_rope(s) if s["case"]["kind"] == "rope" else _plain_mlp(s)


def _own(s):
    import nanobrain_b200 as nb

    case = s["case"]

    def forward():
        if case["kind"] == "rope":
            return nb.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], positions=s["positions"],
                                   freqs=s["freqs"], k_positions=s["k_positions"], eps=EPS,
                                   interleaved=case["interleaved"])
        return (nb.gated_mlp(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"], s["b_down"],
                             activation=case["activation"], checkpoint="%dbit" % case["bits"]),)

    if not case["train"]:
        with torch.inference_mode():
            return {"out": forward()}
    out = forward()
    grads = torch.autograd.grad(out, [s[name] for name in s["leaves"]], s["grads"])
    return {"out": out, **{"d_" + name: grad for name, grad in zip(s["leaves"], grads)}}


def _plain_rope(s):
    case = s["case"]
    packed = case["memory"] == "packed"

    def angles(positions):  # in 64 bits: a far position's angle has no fraction left in 32
        if positions is None:
            return None
        a = positions.double() @ s["freqs"].double()
        a = a[:, None, :] if packed else a[:, None, :, :]
        return a.cos().float(), a.sin().float()

    def halves(x):
        return (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., : HEAD_DIM // 2], x[..., HEAD_DIM // 2 :])

    def join(lo, hi):
        return torch.stack((lo, hi), -1).flatten(-2) if case["interleaved"] else torch.cat((lo, hi), -1)

    def forward(x, w, turn):
        x = x.float()
        n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if turn is not None:
            lo, hi = halves(n)
            n = join(lo * turn[0] - hi * turn[1], hi * turn[0] + lo * turn[1])
        return n.bfloat16()

    def backward(x, w, turn, dy):
        x, dn = x.float(), dy.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        if turn is not None:
            lo, hi = halves(dn)
            dn = join(lo * turn[0] + hi * turn[1], hi * turn[0] - lo * turn[1])
        dw = (dn * x * r).reshape(-1, HEAD_DIM) if packed else (dn * x * r).transpose(1, 2).reshape(-1, HEAD_DIM)
        dx = dn * w
        dx = r * (dx - x * (r * r * (dx * x).mean(-1, keepdim=True)))
        return dx.bfloat16(), dw.sum(0)

    q_turn = angles(s["positions"])
    k_turn = q_turn if s["k_positions"] is None else angles(s["k_positions"])
    out = {"out": (forward(s["q"], s["q_weight"], q_turn), forward(s["k"], s["k_weight"], k_turn))}
    if case["train"]:
        out["d_q"], out["d_q_weight"] = backward(s["q"], s["q_weight"], q_turn, s["grads"][0])
        out["d_k"], out["d_k_weight"] = backward(s["k"], s["k_weight"], k_turn, s["grads"][1])
    return out


def _through_8_bits(v):
    """What 8 bits keep of ``v``: groups of 32 features of a token share a scale, their largest magnitude over 127
    rounded up to bfloat16, and every value is the nearest whole multiple of it."""
    t, f = v.shape
    v = torch.nn.functional.pad(v, (0, -f % GROUP)).reshape(t, -1, GROUP)
    scale = v.abs().amax(-1, keepdim=True) / 127
    scale = ((scale.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)
    v = torch.where(scale > 0, torch.round(v / scale) * scale, torch.zeros_like(v))
    return v.reshape(t, -1)[:, :f]


def _plain_mlp(s):
    case = s["case"]
    x, wg, wu, wd = (s[name].float() for name in ("x", "w_gate", "w_up", "w_down"))
    a, b = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        a, b = a + s["b_gate"].float(), b + s["b_up"].float()

    def gate(a):
        return a * torch.sigmoid(a) if case["activation"] == "silu" else a * (0.5 * (1 + torch.erf(a * math.sqrt(0.5))))

    h = gate(a) * b
    y = h @ wd.t()
    if case["bias"]:
        y = y + s["b_down"].float()
    out = {"out": (y.bfloat16(),)}
    if case["train"]:
        if case["bits"] == 8:
            a, b = _through_8_bits(a), _through_8_bits(b)
            h = gate(a) * b
        dy = s["grads"][0].float()
        dh = dy @ wd
        if case["activation"] == "silu":
            sig = torch.sigmoid(a)
            slope = sig * (1 + a * (1 - sig))
        else:
            slope = 0.5 * (1 + torch.erf(a * math.sqrt(0.5))) + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
        da, db = dh * b * slope, dh * gate(a)
        out["d_x"] = (da @ wg + db @ wu).bfloat16()
        out["d_w_gate"], out["d_w_up"], out["d_w_down"] = ((p.t() @ q).bfloat16() for p, q in ((da, x), (db, x), (dy, h)))
        if case["bias"]:
            out["d_b_gate"], out["d_b_up"], out["d_b_down"] = (p.sum(0).bfloat16() for p in (da, db, dy))
    return out


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs written once, and the products' operations."""
    if case["kind"] == "rope":
        tokens = case["batch"] * (case["seqlen"] + (case["context"] or case["seqlen"]))
        values = tokens * case["heads"] * HEAD_DIM
        coordinates = case["batch"] * (case["seqlen"] + case["context"]) * case["axes"]
        # forward: read and write; backward: read the gradients as well (the inputs are counted once), write theirs
        return {"bytes": 2 * values * (4 if case["train"] else 2) + 8 * coordinates + 4 * HEAD_DIM * (2 + 2 * case["train"]),
                "flops": values * (30 if case["train"] else 10)}
    t, d, f = case["tokens"], case["dim"], case["hidden"]
    params = 3 * d * f + (2 * f + d if case["bias"] else 0)
    product = 2 * t * d * f
    if case["train"]:
        return {"bytes": 2 * (4 * t * d + 2 * params), "flops": 9 * product}
    return {"bytes": 2 * (2 * t * d + params), "flops": 3 * product}


# ------------------------------------------------------------------------------------------
# The definition in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    leaves = {name: s[name].detach().double().requires_grad_(case["train"]) for name in s["leaves"]}
    out = _exact_rope(s, leaves) if case["kind"] == "rope" else _exact_mlp(s, leaves)
    return out


def _exact_rope(s, v):
    case = s["case"]
    pair = torch.arange(HEAD_DIM // 2, device=DEV)
    first = 2 * pair if case["interleaved"] else pair
    second = first + (1 if case["interleaved"] else HEAD_DIM // 2)

    def one(x, w, positions):
        n = x / (x.pow(2).sum(-1, keepdim=True) / HEAD_DIM + EPS).sqrt() * w
        if positions is None:
            return n
        phase = (positions.double().unsqueeze(-1) * s["freqs"].double()).sum(-2)
        phase = phase.unsqueeze(-2 if case["memory"] == "packed" else -3)
        turned = torch.complex(n[..., first], n[..., second]) * torch.polar(torch.ones_like(phase), phase)
        return torch.empty_like(n).index_copy(-1, first, turned.real).index_copy(-1, second, turned.imag)

    out = (one(v["q"], v["q_weight"], s["positions"]),
           one(v["k"], v["k_weight"], s["positions"] if s["k_positions"] is None else s["k_positions"]))
    result = {"out": tuple(t.detach() for t in out)}
    if case["train"]:
        grads = torch.autograd.grad(out, list(v.values()), [t.double() for t in s["grads"]])
        result.update(("d_" + name, grad) for name, grad in zip(v, grads))
    return result


def _kept_in_8_bits(v):
    """``_through_8_bits`` of 64-bit values, by the same words."""
    t, f = v.shape
    groups = torch.zeros(t, -(-f // GROUP) * GROUP, dtype=v.dtype, device=v.device)
    groups[:, :f] = v
    groups = groups.view(t, -1, GROUP)
    wanted = groups.abs().max(-1, keepdim=True).values / 127
    scale = wanted.to(torch.bfloat16)  # nearest, then one up where that is too small
    scale = torch.where(scale.double() < wanted, (scale.view(torch.int16) + 1).view(torch.bfloat16), scale).double()
    codes = (groups / scale.clamp_min(1e-300)).round()
    return (codes * scale).view(t, -1)[:, :f]


def _exact_mlp(s, v):
    case, functional = s["case"], torch.nn.functional
    activation = functional.silu if case["activation"] == "silu" else functional.gelu
    with torch.no_grad():
        a = functional.linear(v["x"], v["w_gate"], v.get("b_gate"))
        b = functional.linear(v["x"], v["w_up"], v.get("b_up"))
        result = {"out": (functional.linear(activation(a) * b, v["w_down"], v.get("b_down")),)}
        if not case["train"]:
            return result
        if case["bits"] == 8:
            a, b = _kept_in_8_bits(a), _kept_in_8_bits(b)
    a.requires_grad_(True), b.requires_grad_(True)
    h = activation(a) * b
    dy = s["grads"][0].double()
    da, db = torch.autograd.grad(h, (a, b), dy.mm(v["w_down"].detach()))
    with torch.no_grad():
        result["d_x"] = torch.cat((da, db), 1).mm(torch.cat((v["w_gate"], v["w_up"])))
        result["d_w_gate"] = torch.einsum("tf,td->fd", da, v["x"])
        result["d_w_up"] = torch.einsum("tf,td->fd", db, v["x"])
        result["d_w_down"] = torch.einsum("td,tf->df", dy, h)
        if case["bias"]:
            ones = torch.ones(1, case["tokens"], dtype=torch.float64, device=DEV)
            result.update(("d_" + name, ones.mm(g)[0]) for name, g in (("b_gate", da), ("b_up", db), ("b_down", dy)))
    return result
