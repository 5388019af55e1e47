"""CPU tests of the float64 restatements (oracle/gated.py): gradients against differences and against autograd."""
import numpy as np
import pytest
import torch

from oracle import gated as og


def case(gate, T=23, C=5, seed=3):
    r = np.random.default_rng(seed)
    f = 2 + 1.5 * r.standard_normal((T, C)) if gate == "sigmoid" else -1 + r.standard_normal((T, C))
    starts = r.random(T) < 0.15
    return r.standard_normal((T, C)), f, r.standard_normal(C), starts, r.standard_normal(C), r.standard_normal((T, C))


@pytest.mark.parametrize("gate", ["sigmoid", "decay"])
@pytest.mark.parametrize("length", [0, 1, 11, 23])
def test_recurrence_gradients_against_differences(gate, length):
    x, f, s, starts, gs, gy = case(gate)

    def loss(x, f, s):
        (s_out, h), _ = og.gated(x, f, s, length, starts, gate)
        return (s_out * gs).sum() + (h * gy).sum()

    grads, bounds = og.gated_bwd(x, f, s, length, starts, gate, gs, gy)
    r = np.random.default_rng(5)
    for i, (a, g) in enumerate(zip((x, f, s), grads)):
        assert (bounds[i] >= 0).all() and bounds[i].shape == g.shape
        d, step = r.standard_normal(a.shape), 1e-5
        up, down = [x, f, s], [x, f, s]
        up[i], down[i] = a + step * d, a - step * d
        # a central difference of step 1e-5 of an order-one function: 1e-10 of its third derivative, 1e-11 of cancellation
        assert abs((loss(*up) - loss(*down)) / (2 * step) - (g * d).sum()) < 1e-7


@pytest.mark.parametrize("activation", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("gated", [False, True])
def test_group_norm_gradients_against_autograd(activation, gated):
    r = np.random.default_rng(7)
    rows, C, G = 6, 24, 4
    t = [torch.tensor(r.standard_normal(s), requires_grad=True) for s in ((rows, C), (C,), (C,), (rows, C))]
    x, w, b, gate = t
    gy = r.standard_normal((rows, C))
    act = {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[activation]
    n = torch.nn.functional.group_norm(x, G, w, b, 1e-3)
    out = n * act(gate) if gated else act(n)
    grads = torch.autograd.grad(out, t if gated else t[:3], torch.tensor(gy))
    ref, _ = og.group_norm(*[q.detach().numpy() for q in (x, w, b)], G, gate.detach().numpy() if gated else None, activation, 1e-3, gy)
    np.testing.assert_allclose(ref[0], out.detach().numpy(), atol=1e-12)
    for got, want in zip(ref[1:], grads):
        np.testing.assert_allclose(got, want.numpy(), atol=1e-12)
