"""Inputs and comparisons shared by the tests of the gated recurrence and the group norm."""
import numpy as np
import torch

from oracle import gated as og


def inputs(B, T, C, gate, dtype, seed, starts=0.0, lengths=None):
    """x, f (B, T, C), s (B, C) float32, length (B,), new_starts (B, T), gy, gs: CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g)
    x = rn(B, T, C).to(dtype)
    f = (2.0 + 1.5 * rn(B, T, C) if gate == "sigmoid" else torch.linspace(-6, -1, C) + 0.5 * rn(B, T, C)).to(dtype)
    length = torch.randint(0, T + 1, (B,), generator=g) if lengths is None else torch.tensor(lengths)
    return x, f, rn(B, C), length.to(torch.int32), torch.rand(B, T, generator=g) < starts, rn(B, T, C).to(dtype), rn(B, C)


def np64(t):
    return t.detach().double().cpu().numpy()


def units(dtype):
    return og.UNITS[torch.finfo(dtype).bits // 8]


def within(got, ref, bound, what, least=1e-37):
    """Every element within the bound and half a rounding step of its own type; what is no number in the same places."""
    got_, half = np64(got), torch.finfo(got.dtype).eps / 2
    assert got_.shape == ref.shape, (what, got_.shape, ref.shape)
    np.testing.assert_array_equal(np.isnan(got_), np.isnan(ref), err_msg=what)
    room = bound + half * (np.abs(ref) + bound) + least
    bad = ~(np.abs(got_ - ref) <= room) & ~np.isnan(ref) & ~(got_ == ref)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.abs(got_ - ref) / room)))


def check_gated(got, x, f, s, length, ns, gate, gs=None, gy=None, what=""):
    """got: (s_out, out) or (s_out, out, dx, df, ds) of (B, T, C) operands."""
    B, T, _ = x.shape
    k = units(x.dtype)
    for b in range(B):
        L = min(int(length[b]), T)
        args = (np64(x[b]), np64(f[b]), np64(s[b]), L, ns[b].cpu().numpy())
        (ref, bounds) = og.gated(*args, gate, units=k)
        names = ("s_out", "out")
        if len(got) > 2:
            g, gb = og.gated_bwd(*args, gate, np64(gs[b]), np64(gy[b]), units=k)
            ref, bounds, names = ref + g, bounds + gb, names + ("dx", "df", "ds")
        for one, r, bound, name in zip(got, ref, bounds, names):
            within(one[b], r, bound, f"{what} {name} of sequence {b}")


def check_norm(got, x, weight, bias, groups, gate, activation, eps, gy=None, what=""):
    """got: [out] or [out, dx, dweight, dbias, dgate], those that are None left out of the comparison."""
    o = lambda t: None if t is None else np64(t)
    C = x.shape[-1]
    flat = lambda t: None if t is None else t.reshape(-1, C)
    ref, bounds = og.group_norm(o(flat(x)), o(weight), o(bias), groups, o(flat(gate)), activation, eps, o(flat(gy)), units=units(x.dtype))
    for one, r, bound, name in zip(got, ref, bounds, ("out", "dx", "dweight", "dbias", "dgate")):
        if one is not None:
            within(one.reshape(r.shape), r, bound, f"{what} {name}")
