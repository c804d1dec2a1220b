"""The operators around attention in a transformer block, as ``torch.library`` ops over the C ABI of
``include/nb_block.h``.

``qk_norm_rope(q, k, q_weight=None, k_weight=None, positions=None, freqs=None, k_positions=None, eps=1e-6,
interleaved=False)``
    RMS norm of every head of queries and keys and their rotation by the tokens' positions, in one pass in
    front of :func:`nanobrain_b200.sdpa` (``[B, H, L, 64]``) or :func:`nanobrain_b200.sdpa_varlen`
    (``[T, H, 64]``); the reference has neither at ``src/nanobrain/modules.py:59-62``.

``gated_mlp(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu", checkpoint="16bit")``
    ``(act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)) @ w_down.T + b_down``, the gated form of the
    reference's two-layer MLP (``src/nanobrain/modules.py:68-85``).

Both take bfloat16 CUDA tensors and have their backward (once; a tensor that carries a forward-mode tangent is
refused). As in :mod:`nanobrain_b200.ops` the CUDA and autograd kernels are native code
(``csrc/torch_block.cpp``), schemas and fake kernels are here, and what is outside the supported subset raises:
there is no fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.overrides import has_torch_function

from . import ops

_ACTIVATIONS = {"silu": 0, "gelu": 1}
_CHECKPOINTS = {"16bit": 1, "8bit": 2}
_TILE_ROWS, _GROUP = 128, 32  # of the checkpoint: nb_gated_mlp_checkpoint_bytes


def _like(t: Tensor) -> Tensor:
    return ops._new_dense(t) if t.dim() == 4 else t.new_empty(t.shape)


def _checkpoint_bytes(tokens, hidden, checkpoint: int):
    if checkpoint == 0:
        return 0
    blocks = -(-tokens // _TILE_ROWS) * -(-hidden // _GROUP)
    return blocks * _TILE_ROWS * (_GROUP * 2 * (2 if checkpoint == 1 else 1) + 4)


def _define_ops() -> torch.library.Library:
    library = torch.library.Library("nanobrain_b200", "FRAGMENT")
    for schema in (
        "qk_norm_rope_fwd(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? positions, Tensor? k_positions,"
        " Tensor? freqs, float eps, bool interleaved) -> (Tensor, Tensor)",
        "qk_norm_rope_bwd(Tensor d_q_out, Tensor d_k_out, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight,"
        " Tensor? positions, Tensor? k_positions, Tensor? freqs, float eps, bool interleaved)"
        " -> (Tensor, Tensor, Tensor, Tensor)",
        "gated_mlp_fwd(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor? b_gate, Tensor? b_up, Tensor? b_down,"
        " int activation, int checkpoint) -> (Tensor, Tensor, Tensor)",
        "gated_mlp_bwd(Tensor d_out, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor h, Tensor codes,"
        " int activation, int checkpoint, bool[7] wanted)"
        " -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
    ):
        library.define(schema, tags=(torch.Tag.pt2_compliant_tag,))

    @torch.library.register_fake("nanobrain_b200::qk_norm_rope_fwd", lib=library)
    def _(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved):
        return _like(q), _like(k)

    @torch.library.register_fake("nanobrain_b200::qk_norm_rope_bwd", lib=library)
    def _(d_q_out, d_k_out, q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved):
        weight = q.new_empty((64,), dtype=torch.float32)
        return _like(q), _like(k), weight, torch.empty_like(weight)

    @torch.library.register_fake("nanobrain_b200::gated_mlp_fwd", lib=library)
    def _(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, checkpoint):
        hidden = w_gate.shape[0]
        tokens = x.numel() // x.shape[-1]
        h = x.new_empty((tokens, -(-hidden // 64) * 64))[:, :hidden] if checkpoint == 1 else x.new_empty((0,))
        codes = x.new_empty((_checkpoint_bytes(tokens, hidden, checkpoint),), dtype=torch.uint8)
        return x.new_empty(x.shape), h, codes

    @torch.library.register_fake("nanobrain_b200::gated_mlp_bwd", lib=library)
    def _(d_out, x, w_gate, w_up, w_down, h, codes, activation, checkpoint, wanted):
        hidden, dim = w_gate.shape
        shapes = (x.shape, (hidden, dim), (hidden, dim), (dim, hidden), (hidden,), (hidden,), (dim,))
        return tuple(x.new_empty(shape if want else (0,)) for shape, want in zip(shapes, wanted))

    return library


if "_library" not in globals():  # (a reload of this module keeps them)
    _library = _define_ops()

qk_norm_rope_fwd = torch.ops.nanobrain_b200.qk_norm_rope_fwd.default
qk_norm_rope_bwd = torch.ops.nanobrain_b200.qk_norm_rope_bwd.default
gated_mlp_fwd = torch.ops.nanobrain_b200.gated_mlp_fwd.default
gated_mlp_bwd = torch.ops.nanobrain_b200.gated_mlp_bwd.default


# FLOP formulas for ``FlopCounterMode`` (cf. ops.py): products only, 3 forward and 6 backward.
def _register_flop_formulas() -> None:
    from torch.utils.flop_counter import register_flop_formula

    def product(x_shape, w_gate_shape) -> int:
        flops = 2 * w_gate_shape[0]
        for size in x_shape:
            flops *= size
        return flops

    @register_flop_formula(torch.ops.nanobrain_b200.gated_mlp_fwd)
    def _(x_shape, w_gate_shape, *args, out_shape=None, **kwargs) -> int:
        return 3 * product(x_shape, w_gate_shape)

    @register_flop_formula(torch.ops.nanobrain_b200.gated_mlp_bwd)
    def _(d_out_shape, x_shape, w_gate_shape, *args, out_shape=None, **kwargs) -> int:
        return 6 * product(x_shape, w_gate_shape)


if not globals().get("_flop_formulas"):
    _register_flop_formulas()
    _flop_formulas = True


def _observed(*tensors) -> bool:
    """Tracing and overrides see the op itself."""
    return torch.compiler.is_compiling() or has_torch_function(tensors)


def qk_norm_rope(
    q: Tensor,
    k: Tensor,
    q_weight: Optional[Tensor] = None,
    k_weight: Optional[Tensor] = None,
    positions: Optional[Tensor] = None,
    freqs: Optional[Tensor] = None,
    k_positions: Optional[Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> Tuple[Tensor, Tensor]:
    """Norms of queries and keys per head and their rotation by position; returns new ``(q, k)``.

    ``q``, ``k``: packed ``[T, H, 64]`` or dense logical ``[B, H, L, 64]`` (any strides; a transposed view of a
    projection's output is read in place), with their own numbers of heads and tokens. Results have the layout
    that ``sdpa`` and ``sdpa_varlen`` read in place.

    ``q_weight``, ``k_weight``: ``[64]``, float32 or bfloat16, the norms' weights (default: ones).

    ``positions``: ``[T, axes]`` (packed), ``[L, axes]`` or ``[B, L, axes]`` (dense), int32, int64 or float32;
    ``freqs``: float32 ``[axes, 32]``. Pair ``i`` of a head is turned by ``sum_a positions[a] * freqs[a, i]``,
    computed in 64 bits; pairs are values ``(i, i + 32)``, or ``(2i, 2i + 1)`` where ``interleaved``. Without
    them nothing is turned. ``k_positions``: of the keys, where they are other tokens than the queries. Neither
    positions nor frequencies have a gradient.

    Every token is treated by itself, rows behind the last sequence of a packed buffer too. The sum of squares is
    in float32 (values beyond 1e18 overflow it); the result is rounded once."""
    if _observed(q, k, q_weight, k_weight, positions, k_positions, freqs):
        return qk_norm_rope_fwd(q, k, q_weight, k_weight, positions, k_positions, freqs, float(eps), bool(interleaved))
    native = ops._native or ops._load_native()
    return native.qk_norm_rope(q, k, q_weight, k_weight, positions, k_positions, freqs, float(eps), bool(interleaved))


def gated_mlp(
    x: Tensor,
    w_gate: Tensor,
    w_up: Tensor,
    w_down: Tensor,
    b_gate: Optional[Tensor] = None,
    b_up: Optional[Tensor] = None,
    b_down: Optional[Tensor] = None,
    activation: str = "silu",
    checkpoint: str = "16bit",
) -> Tensor:
    """``(act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)) @ w_down.T + b_down`` for bfloat16 tensors.

    ``x``: ``[..., dim]``; ``w_gate``, ``w_up``: ``[hidden, dim]``; ``w_down``: ``[dim, hidden]`` (as
    ``nn.Linear`` keeps them); ``dim`` and ``hidden`` multiples of 8. ``activation``: ``"silu"`` or ``"gelu"``
    (with erf).

    ``checkpoint`` says what the forward keeps of the two products ``a = x @ w_gate.T + b_gate`` and
    ``b = x @ w_up.T + b_up`` for the backward, where gradients are wanted:

    * ``"16bit"``: float16 with a power of two per 32 features of a token, and the block's inner activations
      (6 bytes per token and feature in all);
    * ``"8bit"``: whole multiples of ``max|.| / 127`` (rounded up to bfloat16) per 32 features of a token
      (2.1 bytes per token and feature; the inner activations are computed again from them). The gradients are
      then those at the rounded ``a`` and ``b``. A group whose multiple would be below 2^-100 is zeros, one with a
      value that is not finite is NaN as a whole.

    Products are summed in float32; the inner activations and, in the backward, the gradients of ``a`` and ``b`` are
    rounded to bfloat16 between two products, as the results are at the end (errors of 0.0025 against 0.0017 of the
    result's rounding alone)."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if checkpoint not in _CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {sorted(_CHECKPOINTS)}, got {checkpoint!r}")
    args = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    codes = _ACTIVATIONS[activation], _CHECKPOINTS[checkpoint]
    if _observed(*args):
        if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)):
            codes = codes[0], 0  # nothing goes back: nothing is kept
        return gated_mlp_fwd(*args, *codes)[0]
    return (ops._native or ops._load_native()).gated_mlp(*args, *codes)
