"""``gated_mlp``'s backward thousands of times on the same inputs: every call has the same bits. Its second kernel refills a
block of shared memory as soon as it has been read; sizes with few steps per tile, where that is most of its work."""

import pytest
import torch

import test_gated_mlp_gpu as G
from nanobrain_b200 import ops

pytestmark = pytest.mark.gpu
OPS = torch.ops.nanobrain_b200


@pytest.mark.parametrize("checkpoint", [1, 2])
@pytest.mark.parametrize("tokens,dim,hidden", [(3900, 176, 2328), (7749, 88, 1696), (4940, 232, 1832), (4000, 64, 2048)])
def test_every_call_has_the_same_bits(tokens, dim, hidden, checkpoint):
    x, wg, wu, wd, bg, bu, bd = G.problem(tokens, dim, hidden, True)
    dy = G.randn(tokens, dim, seed=9, std=0.1)
    _, h, codes = OPS.gated_mlp_fwd(x, wg, wu, wd, bg, bu, bd, 0, checkpoint)

    def grads():
        return OPS.gated_mlp_bwd(dy, x, wg, wu, wd, h, codes, 0, checkpoint, [True, False, False, True, False, False, False])

    want = grads()
    wrong = torch.zeros((), dtype=torch.int64, device=G.DEV)
    for _ in range(4000):
        got = grads()
        wrong += (got[0] != want[0]).any() | (got[3] != want[3]).any()
    ops.check_status()
    assert int(wrong) == 0
