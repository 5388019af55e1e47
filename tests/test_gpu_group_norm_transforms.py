"""GPU tests of the group norm under ``torch.func``: gradients, batching, both."""
import itertools

import pytest
import torch

from jaxrwkv_b200 import _lib
from jaxrwkv_b200.gated_recurrence import gated_recurrence
from jaxrwkv_b200.group_norm import group_norm_act

pytestmark = pytest.mark.gpu


def make(n, rows, C, dtype=torch.float32, seed=1):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g).to(dtype).cuda()
    return rn(n, rows, C), 1 + 0.1 * rn(n, C), 0.1 * rn(n, C), rn(n, rows, C), rn(n, rows, C)


def grads(x, w, b, gate, gy, G=2, act="silu"):
    there = [t for t in (x, w, b, gate) if t is not None]

    def f(*ts):
        it = iter(ts)
        a = [None if t is None else next(it) for t in (x, w, b, gate)]
        return group_norm_act(a[0], a[1], a[2], G, gate=a[3], activation=act)
    out, back = torch.func.vjp(f, *there)
    return (out, *back(gy))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("there", list(itertools.product([False, True], repeat=3)))
def test_vjp_is_autograds(there, dtype):
    x, w, b, gate, gy = (t[0] for t in make(1, 70, 48, dtype))
    w, b, gate = (t if q else None for t, q in zip((w, b, gate), there))
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, gate)]
    out = group_norm_act(leaves[0], leaves[1], leaves[2], 2, gate=leaves[3])
    want = (out, *torch.autograd.grad(out, [t for t in leaves if t is not None], gy))
    for a, r in zip(grads(x, w, b, gate, gy), want):
        assert torch.equal(a, r)
    loss = lambda x: (group_norm_act(x, w, b, 2, gate=gate) * gy).sum()
    assert torch.equal(torch.func.grad(loss)(x), want[1])


@pytest.mark.parametrize("mapped", [m for m in itertools.product([False, True], repeat=5) if any(m)])
def test_vmap_with_any_arguments_mapped(mapped):
    """x, weight, bias, gate and the cotangent, each mapped or shared: an instance's results are its own call's."""
    n = 3
    ts = make(n, 21, 40)
    dims = tuple(0 if m else None for m in mapped)
    got = torch.func.vmap(grads, in_dims=dims)(*[t if m else t[0] for t, m in zip(ts, mapped)])
    for i in range(n):
        for a, r in zip(got, grads(*[t[i] if m else t[0] for t, m in zip(ts, mapped)])):
            assert torch.equal(a[i], r)


def test_vmap_in_other_places_and_nested():
    x, w, b, gate, gy = make(6, 9, 32, torch.bfloat16, seed=2)
    f = lambda x, gate: group_norm_act(x, w[0], b[0], 4, gate=gate, activation="sigmoid")
    want = torch.stack([f(x[i], gate[i]) for i in range(6)])
    assert torch.equal(torch.func.vmap(f, in_dims=(1, 2), out_dims=1)(x.movedim(0, 1), gate.movedim(0, 2)), want.movedim(0, 1))
    lead = lambda t: t.reshape(2, 3, *t.shape[1:])
    assert torch.equal(torch.func.vmap(torch.func.vmap(f))(lead(x), lead(gate)), lead(want))
    assert torch.equal(torch.func.vmap(lambda x: group_norm_act(x, None, None, 4))(x), group_norm_act(x, None, None, 4))
    rows = torch.func.vmap(lambda x: group_norm_act(x, w[0], None, 4))(x[0])                 # one row an instance
    assert torch.equal(rows, group_norm_act(x[0], w[0], None, 4))
    per = torch.func.vmap(torch.func.vmap(lambda *a: grads(*a)[1:], in_dims=(0, None, None, 0, 0)))(lead(x), lead(w)[:, 0], lead(b)[:, 0], lead(gate), lead(gy))
    for i, j in itertools.product(range(2), range(3)):
        for a, r in zip(per, grads(lead(x)[i, j], lead(w)[i, 0], lead(b)[i, 0], lead(gate)[i, j], lead(gy)[i, j])[1:]):
            assert torch.equal(a[i, j], r)


def test_a_mixer_under_transforms():
    """Recurrence and output stage, per-instance gradients of everything against a loop."""
    n, T, C = 3, 33, 24
    g = torch.Generator().manual_seed(3)
    rn = lambda *shape: torch.randn(*shape, generator=g).cuda()
    x, f, s, gate, gy, w, b = rn(n, T, C), rn(n, T, C), rn(n, C), rn(n, T, C), rn(n, T, C), 1 + 0.1 * rn(C), 0.1 * rn(C)

    def loss(x, f, s, gate, w, b, gy):
        s_out, h = gated_recurrence(x, f, s)
        return (group_norm_act(h, w, b, 3, gate=gate) * gy).sum() + s_out.square().sum()
    each = torch.func.grad(loss, argnums=(0, 1, 2, 3, 4, 5))
    got = torch.func.vmap(each, in_dims=(0, 0, 0, 0, None, None, 0))(x, f, s, gate, w, b, gy)
    for i in range(n):
        for a, r in zip(got, each(x[i], f[i], s[i], gate[i], w, b, gy[i])):
            assert torch.equal(a[i], r)


def test_second_order_is_refused():
    x, w, b, gate, gy = (t[0] for t in make(1, 4, 16))
    loss = lambda x: (group_norm_act(x, w, b, 2, gate=gate) * gy).sum()
    with pytest.raises(_lib.B200WKVError, match="second-order"):
        torch.func.grad(lambda x: torch.func.grad(loss)(x).sum())(x)
    with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
        torch.func.jvp(lambda x: group_norm_act(x, w, b, 2), (x,), (x,))
