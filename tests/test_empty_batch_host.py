"""A dense batch of no sequences at the C ABI of the norms and rotation: as a batch of sequences without tokens."""

import ctypes as C

import pytest

from nanobrain_b200 import _lib, build

P = 0x10000


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def args(batch, tokens, ptr):
    t = _lib.Tensor(ptr, 64 * 20, 64 * 2, 64)
    side = lambda: _lib.QkSide(t, t, t, None, P, ptr, 0, 3, 2, tokens)
    return _lib.QkNormRopeArgs(side(), side(), batch, 3, 1, 0, P, 1e-6, P, 1 << 22)


def test_no_sequences_are_as_no_tokens(lib):
    # (without a GPU both end in the same code for that, with one in 0; neither is an error of the arguments)
    no_tokens, no_batch = args(4, 0, None), args(0, 10, None)
    want = lib.nb_qk_norm_rope_fwd(C.byref(no_tokens), None)
    assert want not in (1, 3, 4, 5)
    assert lib.nb_qk_norm_rope_fwd(C.byref(no_batch), None) == want
    if want != 0:  # (the backward writes zeros: not to these addresses)
        assert lib.nb_qk_norm_rope_bwd(C.byref(no_batch), None) == want
    assert lib.nb_qk_norm_rope_fwd(C.byref(args(-1, 10, P)), None) == 3
    assert lib.nb_qk_norm_rope_fwd(C.byref(args(1, 10, None)), None) == 1
