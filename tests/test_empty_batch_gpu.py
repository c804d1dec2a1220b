"""Dense batches of no sequences, and sides without tokens, through the norms and rotation: empty results, zero gradients."""

import pytest
import torch

import nanobrain_b200 as nb
from nanobrain_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def empty(*shape):
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV, requires_grad=True)


@pytest.mark.parametrize("shape,k_shape", [
    ((0, 2, 10, 64), (0, 2, 10, 64)), ((0, 3, 10, 64), (0, 1, 7, 64)), ((0, 2, 0, 64), (0, 2, 10, 64)),
    ((4, 2, 0, 64), (4, 2, 0, 64)), ((0, 2, 64), (0, 5, 64)),
])
@pytest.mark.parametrize("rotated", [False, True])
def test_nothing_in_nothing_out(shape, k_shape, rotated):
    q, k = empty(*shape), empty(*k_shape)
    w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    more = {}
    if rotated:
        more = dict(positions=torch.zeros(*shape[:-3], shape[-2] if q.dim() == 4 else shape[0], 3, device=DEV),
                    k_positions=torch.zeros(*k_shape[:-3], k_shape[-2] if k.dim() == 4 else k_shape[0], 3, device=DEV),
                    freqs=torch.ones(3, 32, device=DEV))
    y = nb.qk_norm_rope(q, k, *w, **more)
    assert y[0].shape == shape and y[1].shape == k_shape and y[0].dtype == torch.bfloat16
    # (new gradients over memory that held something else)
    torch.full((4, 64), float("nan"), device=DEV)
    grads = torch.autograd.grad(y, (q, k, *w), [torch.empty_like(t) for t in y])
    ops.check_status()
    assert grads[0].shape == shape and grads[1].shape == k_shape
    assert not grads[2].any() and not grads[3].any()


def test_no_queries_but_keys():
    # one side alone has tokens: it gets its results
    q, k = empty(2, 2, 0, 64), torch.randn(2, 3, 9, 64, device=DEV).bfloat16().requires_grad_(True)
    w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    pos, freqs = torch.arange(9, device=DEV)[:, None], torch.ones(1, 32, device=DEV)
    y = nb.qk_norm_rope(q, k, *w, positions=pos[:0], k_positions=pos, freqs=freqs)
    both = nb.qk_norm_rope(k, k, w[1], w[1], positions=pos, freqs=freqs)
    assert y[0].shape == q.shape and torch.equal(y[1], both[1])
    dq, dk, dwq, dwk = torch.autograd.grad(y, (q, k, *w), [torch.empty_like(q), k.detach()])
    ops.check_status()
    assert dq.shape == q.shape and not dwq.any() and dwk.any() and torch.isfinite(dk.float()).all()
