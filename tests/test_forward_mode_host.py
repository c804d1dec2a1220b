"""Forward-mode derivatives: no operator has them, so a tensor that carries a tangent is refused where losing it would
read as a derivative of zero. On meta tensors, which the autograd kernels see like any other."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import nanobrain_b200 as nb

OPS = torch.ops.nanobrain_b200
REFUSAL = "forward-mode"


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def refuses_a_tangent_of_each(call, args, differentiable):
    """``call(*args)`` works, under a dual level too, and is refused where one of ``differentiable`` carries a tangent."""
    call(*args)
    with fwAD.dual_level():
        call(*args)
        for i in differentiable:
            for leaf in (False, True):
                dual = list(args)
                dual[i] = fwAD.make_dual(args[i].detach().requires_grad_(leaf), torch.empty_like(args[i]))
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(NotImplementedError, match=REFUSAL):
                        call(*dual)
    for i in differentiable:
        with pytest.raises(NotImplementedError, match=REFUSAL):
            torch.func.jvp(lambda t: call(*args[:i], t, *args[i + 1:]), (args[i],), (torch.empty_like(args[i]),))


@pytest.mark.parametrize("q", [(9, 2, 64), (2, 2, 9, 64)])
def test_qk_norm_rope(q):
    q, k = meta(*q), meta(*q)
    weight, pos, freqs = meta(64, dtype=torch.float32), meta(9, 3, dtype=torch.float32), meta(3, 32, dtype=torch.float32)
    refuses_a_tangent_of_each(nb.qk_norm_rope, (q, k, weight, weight, pos, freqs, pos), range(7))
    # no weights, no positions
    refuses_a_tangent_of_each(nb.qk_norm_rope, (q, k), range(2))


@pytest.mark.parametrize("checkpoint", ["16bit", "8bit"])
def test_gated_mlp(checkpoint):
    args = (meta(5, 64), meta(96, 64), meta(96, 64), meta(64, 96), meta(96), meta(96), meta(64))
    refuses_a_tangent_of_each(lambda *a: nb.gated_mlp(*a, checkpoint=checkpoint), args, range(7))
    refuses_a_tangent_of_each(lambda *a: nb.gated_mlp(*a, checkpoint=checkpoint), args[:4], range(4))


def test_the_ops_themselves():
    # (what tracing calls)
    q = meta(9, 2, 64)
    refuses_a_tangent_of_each(lambda a, b: OPS.qk_norm_rope_fwd(a, b, None, None, None, None, None, 1e-6, False), (q, q), range(2))
    mlp = (meta(5, 64), meta(96, 64), meta(96, 64), meta(64, 96))
    refuses_a_tangent_of_each(lambda *a: OPS.gated_mlp_fwd(*a, None, None, None, 0, 1), mlp, range(4))


def test_the_backward_ops():
    # forward over reverse
    q = meta(9, 2, 64)
    with fwAD.dual_level():
        dual = fwAD.make_dual(q, torch.empty_like(q))
        with pytest.raises(NotImplementedError, match="forward AD"):
            OPS.qk_norm_rope_bwd(dual, q, q, q, None, None, None, None, None, 1e-6, False)


def test_sdpa():
    q = meta(2, 3, 9, 64)
    refuses_a_tangent_of_each(nb.sdpa, (q, q, q), range(3))
    refuses_a_tangent_of_each(lambda *a: OPS.sdpa_fwd(*a, 0.125), (q, q, q), range(3))


def test_sdpa_varlen():
    q, cu = meta(9, 2, 64), meta(3, dtype=torch.int32)
    refuses_a_tangent_of_each(lambda *a: nb.sdpa_varlen(*a, cu, cu, 5, 5), (q, q, q), range(3))
    refuses_a_tangent_of_each(lambda *a: OPS.sdpa_varlen_fwd(*a, cu, cu, 5, 5, 0.125), (q, q, q), range(3))
