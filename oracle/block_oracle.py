"""The operators around attention from their definitions, in 64 bits: what the GPU tests compare with."""

import math

import torch

HALF_STEP = torch.finfo(torch.bfloat16).eps / 2  # of a rounding to bf16, relative to the value
GROUP = 32


def split_pairs(n, interleaved):
    return (n[..., 0::2], n[..., 1::2]) if interleaved else (n[..., :32], n[..., 32:])


def join_pairs(lo, hi, interleaved):
    return torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)


def angles(positions, freqs, dense):
    """Broadcastable to [T, H, 32] or [B, H, L, 32]; None without positions."""
    if positions is None:
        return None
    a = positions.double() @ freqs.double()
    return a.unsqueeze(-3) if dense else a.unsqueeze(-2)


def norm_rope(x, weight, theta, eps, interleaved):
    """(y, n): the result and the norm's output in front of the rotation."""
    x = x.double()
    w = torch.ones(64, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    if theta is None:
        return n, n
    lo, hi = split_pairs(n, interleaved)
    return join_pairs(lo * theta.cos() - hi * theta.sin(), hi * theta.cos() + lo * theta.sin(), interleaved), n


def act(a, activation):
    return a * torch.sigmoid(a) if activation == "silu" else a * 0.5 * (1 + torch.erf(a / math.sqrt(2)))


def keep_8_bits(v):
    """Whole multiples of max|.| / 127, rounded up to bf16, per 32 features of a row; a group that is not finite is NaN."""
    t, f = v.shape
    g = torch.zeros(t, -(-f // GROUP) * GROUP, dtype=v.dtype, device=v.device)
    g[:, :f] = v
    g = g.view(t, -1, GROUP)
    want = g.abs().amax(-1, keepdim=True) / 127
    scale = want.to(torch.bfloat16)
    scale = torch.where(scale.double() < want, (scale.view(torch.int16) + 1).view(torch.bfloat16), scale).double()
    kept = (g / scale).round() * scale
    kept = torch.where(scale == 0, torch.zeros_like(kept), kept)
    kept = torch.where(torch.isfinite(scale), kept, torch.full_like(kept, float("nan")))
    return kept.reshape(t, -1)[:, :f]


def mlp(x, wg, wu, wd, bg=None, bu=None, bd=None, activation="silu", dy=None, bits=16):
    """(y, gradients of everything in order) of the gated block on [T, dim] rows; gradients are those at the a and b
    that `bits` keep (16: all of them)."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    bias = [None if b is None else b.detach().double() for b in (bg, bu, bd)]
    a, b = x @ wg.t(), x @ wu.t()
    a = a if bias[0] is None else a + bias[0]
    b = b if bias[1] is None else b + bias[1]
    y = (act(a, activation) * b) @ wd.t()
    y = y if bias[2] is None else y + bias[2]
    if dy is None:
        return y, None
    if bits == 8:
        a, b = keep_8_bits(a), keep_8_bits(b)
    a, b = a.requires_grad_(True), b.requires_grad_(True)
    h = act(a, activation) * b
    dy = dy.double()
    da, db = torch.autograd.grad(h, (a, b), dy @ wd)
    h = h.detach()
    return y, (da @ wg + db @ wu, da.t() @ x, db.t() @ x, dy.t() @ h, da.sum(0), db.sum(0), dy.sum(0))
