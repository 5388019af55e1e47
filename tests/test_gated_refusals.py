"""CPU tests of what the gated recurrence and the group norm refuse, at the C boundary (checked before any CUDA call) and in
the Python functions."""
import ctypes

import pytest
import torch

from jaxrwkv_b200 import _lib
from jaxrwkv_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
from jaxrwkv_b200.group_norm import group_norm_act

P = ctypes.c_void_p
A = P(1 << 12)                             # never dereferenced: the checks come first
ODD = P((1 << 12) + 1)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def fwd(lib, dtype=1, gate=0, B=1, T=4, C=8, x=A, f=A, s0=A, length=None, ns=None, y=A, s_out=A, residual=None, nbytes=0):
    return lib.b200wkv_gated_fwd(None, dtype, gate, B, T, C, x, T * C, C, f, T * C, C, s0, length, ns, y, s_out, residual, nbytes)


def test_recurrence_forward(lib):
    assert fwd(lib, dtype=2) == -1
    assert fwd(lib, gate=2) == -6
    for bad in (dict(B=0), dict(T=0), dict(C=0), dict(B=1 << 20, T=1 << 20), dict(B=1 << 16, C=1 << 16), dict(C=(1 << 22) + 1), dict(T=(1 << 30) + 1)):
        assert fwd(lib, **bad) == -2, bad
    for name in ("x", "f", "y", "s_out"):
        assert fwd(lib, **{name: None}) == -3, name
        assert fwd(lib, **{name: ODD}) == -6, name
    assert lib.b200wkv_gated_fwd(None, 1, 0, 1, 4, 8, A, 32, 8, A, 32, -8, A, None, None, A, A, None, 0) == -2
    assert fwd(lib, s0=ODD) == -6 and fwd(lib, length=P((1 << 12) + 2)) == -6
    assert fwd(lib, residual=A, nbytes=lib.b200wkv_gated_residual_bytes(1, 4, 8) - 1) == -4


def test_recurrence_backward(lib):
    need = lib.b200wkv_gated_residual_bytes(2, 100, 8)
    assert need > 0 and lib.b200wkv_gated_residual_bytes(0, 100, 8) == 0

    def bwd(dtype=1, gate=0, C=8, res=A, nbytes=need, dx=A, gy=None):
        return lib.b200wkv_gated_bwd(None, dtype, gate, 2, 100, C, A, 100 * C, C, A, 100 * C, C, None, None, gy, None, res, nbytes, dx, A, A)
    assert bwd(dtype=5) == -1 and bwd(gate=-1) == -6 and bwd(C=0) == -2
    assert bwd(res=None) == -3 and bwd(dx=None) == -3 and bwd(nbytes=need - 1) == -4 and bwd(gy=ODD) == -6


def test_step(lib):
    def step(dtype=1, gate=1, B=2, C=8, x=A, s=A, s_out=A):
        return lib.b200wkv_gated_step(None, dtype, gate, B, C, x, C, A, C, s, C, None, None, A, s_out, C)
    assert step(dtype=-1) == -1 and step(gate=7) == -6 and step(B=0) == -2 and step(C=0) == -2
    assert step(x=None) == -3 and step(s=None) == -3 and step(s_out=None) == -3 and step(s=P((1 << 12) + 2)) == -6


def test_group_norm(lib):
    def norm(dtype=1, rows=4, C=64, G=4, act=2, x=A, w=A, pd=1, gate=None, y=A):
        return lib.b200wkv_group_norm_fwd(None, dtype, rows, C, G, 1e-5, act, x, C, w, w, pd, gate, C, y)
    assert norm(dtype=3) == -1 and norm(pd=3) == -1 and norm(act=3) == -6 and norm(act=-1) == -6
    for bad in (dict(rows=0), dict(C=0), dict(G=0), dict(G=5), dict(C=16386, G=2), dict(rows=1 << 31), dict(C=(1 << 24) + 4)):
        assert norm(**bad) == -2, bad
    assert lib.b200wkv_group_norm_fwd(None, 1, 4, 64, 4, 1e-5, 2, A, -64, A, A, 1, None, 64, A) == -2
    assert norm(x=None) == -3 and norm(y=None) == -3 and norm(x=ODD) == -6 and norm(w=ODD) == -6 and norm(gate=ODD) == -6

    need = lib.b200wkv_group_norm_workspace_bytes(4, 64)

    def bwd(gate=A, dgate=A, dw=A, ws=A, nbytes=need):
        return lib.b200wkv_group_norm_bwd(None, 1, 4, 64, 4, 1e-5, 2, A, 64, A, A, 1, gate, 64, A, A, dgate, dw, None, ws, nbytes)
    assert bwd(dgate=None) == -3 and bwd(gate=None) == -3 and bwd(ws=None) == -3 and bwd(nbytes=need - 1) == -4
    assert lib.b200wkv_group_norm_workspace_bytes(0, 64) == 0


def test_python_functions_refuse():
    x, s = torch.zeros(2, 3, 8), torch.zeros(2, 8)
    for call, match in ((lambda: gated_recurrence(x, x, s), "CUDA"), (lambda: gated_recurrence(x, x, s, gate="tanh"), "gate"),
                        (lambda: gated_recurrence_step(s, s, s), "CUDA"), (lambda: gated_recurrence_step(s, s, s, gate=None), "gate"),
                        (lambda: gated_recurrence(s[0], s[0], s[0, 0]), r"\(\.\.\., T, C\)"),
                        (lambda: gated_recurrence_step(s.requires_grad_(), s, s), "gradients"),
                        (lambda: group_norm_act(x, None, None, 2), "CUDA"), (lambda: group_norm_act(x, None, None, 2, activation="relu"), "activation")):
        with pytest.raises(_lib.B200WKVError, match=match):
            call()
