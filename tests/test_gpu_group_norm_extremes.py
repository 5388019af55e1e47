"""GPU tests of the group norm where gates and normalised values are as large as their type holds, or infinite."""
import pytest
import torch

from jaxrwkv_b200.group_norm import group_norm_act
from gated_util import np64, units
from oracle import gated as og

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
# silu is 0 to within this wherever its argument is -87 or less: |z| 2^-126 at most at -87.4, and n below 10
NOTHING = 10 * 88 * 2.0 ** -126


def rows_of(dtype, values, D=64):
    g = torch.Generator().manual_seed(1)
    values = torch.tensor(values + [torch.finfo(dtype).min], dtype=torch.float64).to(dtype)
    x, gy = (torch.randn(len(values), 2 * D, generator=g).to(dtype).cuda() for _ in range(2))
    return x, values[:, None].expand(-1, 2 * D).contiguous().cuda(), gy, torch.randn(2 * D, generator=g).to(dtype).cuda(), torch.randn(2 * D, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 63])
def test_a_closed_silu_gate(dtype, D):
    """Nothing comes through, and no gradient but to the gate's own place, which is nothing too."""
    x, gate, gy, w, b = rows_of(dtype, [-90.0, -128.0, -1e4, -1e20, -1e36, -3e38], D)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, gate)]
    out = group_norm_act(leaves[0], leaves[1], leaves[2], 2, gate=leaves[3])
    dx, dw, db, dgate = torch.autograd.grad(out, leaves, gy)
    for name, t in (("out", out), ("dx", dx), ("dw", dw), ("db", db), ("dgate", dgate)):
        assert (t.double().abs() <= 100 * NOTHING).all(), (name, t.abs().max())


@pytest.mark.parametrize("dtype", DTYPES)
def test_silu_of_far_values(dtype):
    """Without a gate the normalised values themselves, moved by the bias: 0 far below, and the values themselves far above."""
    x, _, gy, w, _ = rows_of(dtype, [0.0] * 5)
    for far in (-100.0, -1e6, -1e36, torch.finfo(dtype).min):
        b = torch.full_like(w, far).requires_grad_(True)
        lx, lw = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out = group_norm_act(lx, lw, b, 2)
        for t in (out, *torch.autograd.grad(out, (lx, lw, b), gy)):
            assert (t.double().abs() <= 100 * NOTHING).all(), (far, t.abs().max())
    b = torch.full_like(w, 1e30)
    with torch.no_grad():
        out = group_norm_act(x, w, b, 2).double() / b.double()
    assert ((out - 1).abs() <= 8 * 2.0 ** -24 + torch.finfo(dtype).eps / 2).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_between(dtype):
    """Where silu leaves the range in which its factors are exact: within the bounds, or nothing."""
    x, gate, gy, w, b = rows_of(dtype, [-89.0, -88.0, -87.5, -87.25, -87.0, -80.0, -50.0, 50.0, 87.0, 88.0, 1e4])
    gate = gate[:-1]
    x, gy = x[:-1], gy[:-1]
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, gate)]
    out = group_norm_act(*leaves[:3], 2, gate=leaves[3])
    dx, dw, db, dgate = torch.autograd.grad(out, leaves, gy)
    k = units(dtype) + 2 * 90               # the exponential's argument is rounded: 1/2 ulp of 90 log2(e)
    ref, bounds = og.group_norm(np64(x), np64(w), np64(b), 2, np64(gate), "silu", 1e-5, np64(gy), units=k)
    half = torch.finfo(dtype).eps / 2
    for got, r, bound in zip((out, dx, dw, db, dgate), ref, bounds):
        off = abs(np64(got) - r)
        assert (off <= bound + half * abs(r) * 1.01 + 100 * NOTHING).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_infinite_gates(dtype, act):
    """-inf closes a gate, as its limit does; +inf opens sigmoid's fully and leaves silu's infinite; what is no number stays."""
    x, gate, _, w, b = rows_of(dtype, [0.0] * 3)
    gate[0], gate[1], gate[2] = float("-inf"), float("inf"), float("nan")
    with torch.no_grad():
        n = group_norm_act(x, w, b, 2, activation="none")
        out = group_norm_act(x, w, b, 2, gate=gate, activation=act)
    assert (out[0].double().abs() <= 100 * NOTHING).all()
    if act == "silu":
        assert torch.equal(out[1], n[1] * float("inf"))
    else:                                   # n is rounded, and n times 1 (off by 2 ulp at most) is
        assert ((out[1] - n[1]).double().abs() <= (torch.finfo(dtype).eps + 8 * 2.0 ** -24) * n[1].double().abs()).all()
    assert out[2].isnan().all() and torch.isfinite(out[3]).all()
