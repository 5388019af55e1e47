"""GPU tests of the gated recurrence under ``torch.func.vmap`` with only some of its arguments mapped."""
import itertools

import pytest
import torch

from jaxrwkv_b200.gated_recurrence import gated_recurrence
from gated_util import inputs

pytestmark = pytest.mark.gpu
GATES = ["sigmoid", "decay"]


def make(n, T, C, gate, seed=1):
    x, f, s, _, ns, gy, gs = (t.cuda() for t in inputs(n, T, C, gate, torch.float32, seed=seed, starts=0.1))
    return x, f, s, ns, gy, gs


def pick(ts, mapped, i):
    """What instance i has of each tensor; those that are not mapped are the first one's."""
    return [t[i if m else 0] for t, m in zip(ts, mapped)]


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("mapped", [m for m in itertools.product([False, True], repeat=5) if any(m)])
def test_gradients_with_any_arguments_mapped(mapped, gate):
    """x, f, s and the two cotangents, each mapped or shared: every instance's gradients are its own call's."""
    n, T, C = 3, 37, 20
    x, f, s, ns, gy, gs = make(n, T, C, gate)
    ts = (x, f, s, gy, gs)

    def grads(x, f, s, gy, gs):
        _, back = torch.func.vjp(lambda x, f, s: gated_recurrence(x, f, s, None, ns[0], gate=gate), x, f, s)
        return back((gs, gy))
    got = torch.func.vmap(grads, in_dims=tuple(0 if m else None for m in mapped))(*pick_all(ts, mapped))
    for i in range(n):
        for a, b in zip(got, grads(*pick(ts, mapped, i))):
            assert torch.equal(a[i], b)


def pick_all(ts, mapped):
    return [t if m else t[0] for t, m in zip(ts, mapped)]


@pytest.mark.parametrize("which", ["x", "f", "s"])
def test_one_argument_mapped_and_one_gradient(which):
    """The cotangent is shared, and the only gradient is that of an argument that is shared too."""
    n, T, C = 3, 40, 16
    x, f, s, _, gy, _ = make(n, T, C, "sigmoid", seed=2)
    for wanted in range(3):
        def grad(one):
            args = [one if name == which else t[0] for name, t in (("x", x), ("f", f), ("s", s))]
            return torch.func.vjp(lambda q: gated_recurrence(*[q if j == wanted else a for j, a in enumerate(args)])[1], args[wanted])[1](gy[0])[0]
        mapped = {"x": x, "f": f, "s": s}[which]
        got = torch.func.vmap(grad)(mapped)
        for i in range(n):
            assert torch.equal(got[i], grad(mapped[i]))


def test_cotangents_alone_mapped():
    """One forward call, and gradients of several cotangents, as a Jacobian takes them."""
    x, f, s, ns, gy, gs = make(4, 50, 24, "decay", seed=3)
    _, back = torch.func.vjp(lambda *a: gated_recurrence(*a, None, ns[:2], gate="decay"), x[:2], f[:2], s[:2])
    gys, gss = torch.stack([gy[:2], gy[2:], gy[1:3]]), torch.stack([gs[:2], gs[2:], gs[1:3]])
    got = torch.func.vmap(back)((gss, gys))
    for i in range(3):
        for a, b in zip(got, back((gss[i], gys[i]))):
            assert torch.equal(a[i], b)
    nested = torch.func.vmap(torch.func.vmap(back))((torch.stack([gss, gss]), torch.stack([gys, gys])))
    for a, b in zip(nested, got):
        assert torch.equal(a[0], b) and torch.equal(a[1], b)
