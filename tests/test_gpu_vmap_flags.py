"""GPU tests of ``torch.func.vmap`` with flags that the sequences of an instance share."""
import pytest
import torch

from jaxrwkv_b200.gated_recurrence import gated_recurrence

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,B", [(3, 2), (2, 2), (2, 3)])
@pytest.mark.parametrize("flags", ["starts mapped", "starts shared", "length mapped", "length shared", "a number", "both mapped", "full", "length mapped last"])
def test_flags_shared_by_an_instances_sequences(n, B, flags):
    """x (B, T, C) per instance, flags that its B sequences share, mapped or not; as many instances as sequences and not."""
    T, C = 29, 12
    g = torch.Generator().manual_seed(n + B)
    x, f = (torch.randn(n, B, T, C, generator=g).cuda() for _ in range(2))
    s, gy, gs = torch.randn(n, B, C, generator=g).cuda(), torch.randn(n, B, T, C, generator=g).cuda(), torch.randn(n, B, C, generator=g).cuda()
    per_instance = (torch.rand(n, T, generator=g) < 0.2).cuda()
    lengths = torch.tensor([5, 0, 40][:n], device="cuda")
    length, length_dim, starts, starts_dim = None, None, None, None
    if flags in ("starts mapped", "both mapped"):
        starts, starts_dim = per_instance, 0
    if flags == "starts shared":
        starts = per_instance[0]
    if flags in ("length mapped", "both mapped"):
        length, length_dim = lengths, 0
    if flags == "length shared":
        length = torch.tensor([7, 11, 2][:B], device="cuda")
    if flags == "a number":
        length = 9
    if flags == "full":
        starts, starts_dim = (torch.rand(n, B, T, generator=g) < 0.2).cuda(), 0
    if flags == "length mapped last":
        length, length_dim = torch.tensor([[5, 0, 40][:n]] * B, device="cuda"), 1

    def grads(x, f, s, gy, gs, length, starts):
        out, back = torch.func.vjp(lambda x, f, s: gated_recurrence(x, f, s, length, starts), x, f, s)
        return (*out, *back((gs, gy)))
    got = torch.func.vmap(grads, in_dims=(0,) * 5 + (length_dim, starts_dim))(x, f, s, gy, gs, length, starts)
    of = lambda t, d, i: t if d is None else t.select(d, i)
    for i in range(n):
        for a, b in zip(got, grads(x[i], f[i], s[i], gy[i], gs[i], of(length, length_dim, i), of(starts, starts_dim, i))):
            assert torch.equal(a[i], b)
