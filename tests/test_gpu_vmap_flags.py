"""GPU tests of ``torch.func.vmap`` with flags that the sequences of an instance share."""
import pytest
import torch

from jaxrwkv_b200 import rwkv4, rwkv6, rwkv7
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


@pytest.mark.parametrize("n,B", [(3, 2), (2, 2)])
@pytest.mark.parametrize("version", [4, 6, 7])
def test_flags_shared_in_the_other_recurrences(version, n, B):
    T, H, N = 20, 2, 64
    g = torch.Generator().manual_seed(version + n)
    rn = lambda *shape: 0.3 * torch.randn(*shape, generator=g).cuda()
    starts, lengths = (torch.rand(n, T, generator=g) < 0.2).cuda(), torch.tensor([5, 0, 40][:n], dtype=torch.int32, device="cuda")
    if version == 4:
        w, u = rn(H * N), rn(H * N)
        args = [rn(n, B, T, H * N), rn(n, B, T, H * N), rn(n, B, 3, H * N)]
        call = lambda k, v, s, length, ns: rwkv4.wkv4_cuda(k, v, w, u, s, length, ns)
    elif version == 6:
        u = rn(H, N, 1)
        args = [rn(n, B, T, H, N) for _ in range(3)] + [-torch.exp(rn(n, B, T, H, N, 1)), rn(n, B, H, N, N)]
        call = lambda r, k, v, w, s, length, ns: rwkv6.CudaRWKV.inner_loop(r, k, v, w, u, s, length, ns)
    else:
        args = [rn(n, B, T, H, N) for _ in range(6)] + [rn(n, B, H, N, N)]
        call = lambda *a: rwkv7.wkv7_cuda(*a)

    def grads(length, ns, *args):
        out, back = torch.func.vjp(lambda *a: call(*a, length, ns), *args)
        return (*out, *back(tuple(torch.ones_like(o) for o in out)))
    for length, length_dim, ns, ns_dim in ((lengths, 0, starts, 0), (9, None, starts[0], None), (lengths, 0, starts[0], None)):
        got = torch.func.vmap(grads, in_dims=(length_dim, ns_dim) + (0,) * len(args))(length, ns, *args)
        full_length = (length[:, None] if length_dim == 0 else torch.tensor(length, device="cuda")).expand(n, B)
        full_ns = (ns[:, None] if ns_dim == 0 else ns).expand(n, B, T)
        for a, r in zip(got, grads(full_length, full_ns, *args)):           # one call with every sequence's own flags
            assert torch.equal(a, r)
