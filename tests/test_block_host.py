"""The operators around attention on a machine without a GPU: symbols, argument checks of the C ABI, fake kernels."""

import ctypes as C
import re
from pathlib import Path

import pytest
import torch

import nanobrain_b200 as nb
from nanobrain_b200 import _lib, block_ops, build

ROOT = Path(__file__).resolve().parent.parent
OPS = torch.ops.nanobrain_b200
P = 0x10000


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_header_and_binding_list_the_same_symbols(lib):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "nb_block.h").read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(nb_[a-z_0-9]+)\s*\(", text)))
    assert declared == sorted(_lib.BLOCK_SYMBOLS)
    assert all(hasattr(lib, name) for name in declared)


def qk_args(**changes):
    t = _lib.Tensor(P, 64 * 20, 64 * 2, 64)
    side = lambda: _lib.QkSide(t, t, t, None, P, P, 0, 3, 2, 10)
    args = _lib.QkNormRopeArgs(side(), side(), 1, 3, 1, 0, P, 1e-6, P, 1 << 22)
    for path, value in changes.items():
        *owners, name = path.split("__")
        at = args
        for owner in owners:
            at = getattr(at, owner)
        setattr(at, name, value)
    return args


@pytest.mark.parametrize("change,code", [
    (dict(q__x=_lib.Tensor(None, 8, 8, 8)), 1), (dict(k__y=_lib.Tensor(None, 8, 8, 8)), 1),
    (dict(k__positions=None), 1), (dict(freqs=None), 1),
    (dict(q__x=_lib.Tensor(P + 8, 8, 8, 8)), 4), (dict(q__y=_lib.Tensor(P, 8, 12, 8)), 4),
    (dict(q__heads=0), 3), (dict(k__tokens=-1), 3), (dict(batch=-1), 3), (dict(axes=5), 3), (dict(axes=-1), 3),
    (dict(position_type=3), 3), (dict(batch=1 << 30, q__tokens=4), 3),
])
def test_qk_refusals(lib, change, code):
    assert lib.nb_qk_norm_rope_fwd(C.byref(qk_args(**change)), None) == code
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(**change)), None) == code


def test_qk_backward_refusals(lib):
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(workspace=None)), None) == 5
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(workspace_bytes=lib.nb_qk_norm_rope_bwd_workspace_bytes() - 1)), None) == 5
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(workspace=P + 4)), None) == 4
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(q__d_weight=None)), None) == 1
    assert lib.nb_qk_norm_rope_bwd(C.byref(qk_args(q__dy=_lib.Tensor(None, 8, 8, 8))), None) == 1
    assert lib.nb_qk_norm_rope_fwd(None, None) == 1 and lib.nb_qk_norm_rope_bwd(None, None) == 1


def mlp_args(cls, **changes):
    args = cls()
    args.shape = _lib.GatedMlpShape(100, 64, 96, 0, 1)
    for name, cols in (("x", 64), ("w_gate", 64), ("w_up", 64), ("w_down", 96), ("y", 64), ("dy", 64), ("h", 96)):
        if hasattr(args, name):
            setattr(args, name, _lib.Matrix(P, cols))
    args.checkpoint = P
    if cls is _lib.GatedMlpBwdArgs:
        args.workspace, args.workspace_bytes = P, 1 << 30
    for path, value in changes.items():
        *owners, name = path.split("__")
        at = args
        for owner in owners:
            at = getattr(at, owner)
        setattr(at, name, value)
    return args


@pytest.mark.parametrize("change,code", [
    (dict(shape__tokens=0), 3), (dict(shape__dim=60), 3), (dict(shape__hidden=0), 3), (dict(shape__hidden=100), 3),
    (dict(shape__dim=1 << 21), 3), (dict(shape__tokens=1 << 31), 3), (dict(shape__activation=2), 3),
    (dict(shape__checkpoint=3), 3), (dict(shape__checkpoint=-1), 3),
    (dict(x=_lib.Matrix(None, 64)), 1), (dict(w_gate=_lib.Matrix(P + 8, 64)), 4), (dict(w_up=_lib.Matrix(P, 68)), 4),
    (dict(w_down=_lib.Matrix(P, 88)), 4), (dict(checkpoint=None), 1), (dict(checkpoint=P + 16), 4),
    (dict(h=_lib.Matrix(None, 96)), 1),
])
def test_mlp_refusals(lib, change, code):
    assert lib.nb_gated_mlp_fwd(C.byref(mlp_args(_lib.GatedMlpFwdArgs, **change)), None) == code
    assert lib.nb_gated_mlp_bwd(C.byref(mlp_args(_lib.GatedMlpBwdArgs, **change)), None) == code


def test_mlp_refusals_of_one_direction(lib):
    for bias in ("b_gate", "b_up", "b_down"):
        assert lib.nb_gated_mlp_fwd(C.byref(mlp_args(_lib.GatedMlpFwdArgs, **{bias: P + 2})), None) == 4
    assert lib.nb_gated_mlp_fwd(C.byref(mlp_args(_lib.GatedMlpFwdArgs, y=_lib.Matrix(P, 56))), None) == 4
    bwd = _lib.GatedMlpBwdArgs
    assert lib.nb_gated_mlp_bwd(C.byref(mlp_args(bwd, shape__checkpoint=0)), None) == 3
    assert lib.nb_gated_mlp_bwd(C.byref(mlp_args(bwd, dy=_lib.Matrix(None, 64))), None) == 1
    assert lib.nb_gated_mlp_bwd(C.byref(mlp_args(bwd, workspace=P + 64)), None) == 4
    for out in ("dx", "d_w_gate", "d_w_up", "d_w_down"):
        assert lib.nb_gated_mlp_bwd(C.byref(mlp_args(bwd, **{out: _lib.Matrix(P + 2, 96)})), None) == 4
    assert lib.nb_gated_mlp_fwd(None, None) == 1 and lib.nb_gated_mlp_bwd(None, None) == 1
    assert lib.nb_gated_mlp_bwd_workspace_bytes(None) == 0


@pytest.mark.parametrize("tokens,hidden", [(1, 8), (128, 32), (129, 40), (26253, 2048), (131072, 1368)])
def test_checkpoint_bytes(lib, tokens, hidden):
    for mode in (0, 1, 2):
        shape = _lib.GatedMlpShape(tokens, 64, hidden, 0, mode)
        assert lib.nb_gated_mlp_checkpoint_bytes(C.byref(shape)) == block_ops._checkpoint_bytes(tokens, hidden, mode)
    assert lib.nb_gated_mlp_checkpoint_bytes(C.byref(_lib.GatedMlpShape(0, 64, hidden, 0, 1))) == 0


def test_fake_kernels():
    bf = dict(dtype=torch.bfloat16, device="meta")
    q, k = torch.empty(2, 10, 3, 64, **bf).transpose(1, 2), torch.empty(2, 7, 5, 64, **bf).transpose(1, 2)
    y = OPS.qk_norm_rope_fwd(q, k, None, None, None, None, None, 1e-6, False)
    assert [t.shape for t in y] == [q.shape, k.shape] and y[0].transpose(1, 2).is_contiguous()
    g = OPS.qk_norm_rope_bwd(*y, q, k, None, None, None, None, None, 1e-6, False)
    assert [tuple(t.shape) for t in g] == [q.shape, k.shape, (64,), (64,)] and g[2].dtype == torch.float32
    x, w, wd = torch.empty(4, 5, 64, **bf), torch.empty(96, 64, **bf), torch.empty(64, 96, **bf)
    y, h, codes = OPS.gated_mlp_fwd(x, w, w, wd, None, None, None, 0, 1)
    assert y.shape == x.shape and h.shape == (20, 96) and codes.numel() == block_ops._checkpoint_bytes(20, 96, 1)
    y, h, codes = OPS.gated_mlp_fwd(x, w, w, wd, None, None, None, 0, 2)
    assert h.numel() == 0
    g = OPS.gated_mlp_bwd(y, x, w, w, wd, h, codes, 0, 2, [True, True, False, True, True, False, False])
    assert [tuple(t.shape) for t in g] == [x.shape, (96, 64), (0,), (64, 96), (96,), (0,), (0,)]


def test_there_is_no_cpu_path():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        nb.gated_mlp(x, w, w, w)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        nb.qk_norm_rope(q, q)
    with pytest.raises(ValueError, match="activation"):
        nb.gated_mlp(x, w, w, w, activation="relu")
    with pytest.raises(ValueError, match="checkpoint"):
        nb.gated_mlp(x, w, w, w, checkpoint="none")
