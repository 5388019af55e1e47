"""GPU tests of the group norm over more rows than are at work at once, so that every team goes through its rows in a loop."""
import pytest
import torch

from jaxrwkv_b200.group_norm import group_norm_act

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
PER_SM = 2048                              # threads


def passes(rows, G, lanes):
    """Rows that a team takes at least, however many threads are at work, with at least so many lanes in a team."""
    return rows * G * lanes / (torch.cuda.get_device_properties(0).multi_processor_count * PER_SM)


def run(x, w, b, G, gate, act, gy):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, gate)]
    out = group_norm_act(leaves[0], leaves[1], leaves[2], G, gate=leaves[3], activation=act, eps=1e-3)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], gy)
    return (out, grads[0], *grads[3:]), grads[1:3]


# rows, groups, channels, lanes of a team at least (a piece of 16 bytes each, two where groups have more than 32; eight pairs): pieces three and two
# rows ahead, teams of any size, the cap on partial rows, teams added up within a thread block, whole thread blocks, pairs, single channels
SHAPES = {
    torch.bfloat16: [(12001, 32, 64, 8), (8300, 8, 512, 32), (12001, 20, 80, 10), (42001, 9, 64, 8), (145001, 2, 64, 8), (9001, 2, 1024, 128), (2401, 2, 4096, 512),
                     (30001, 17, 60, 8), (60001, 2, 333, 21), (10001, 33, 61, 8)],
    torch.float32: [(6001, 32, 64, 16), (9000, 8, 256, 32), (8001, 20, 72, 18), (21001, 9, 64, 16), (72001, 2, 64, 16), (4801, 2, 1024, 256), (4301, 1, 4096, 512),
                    (40001, 17, 58, 8), (60001, 2, 333, 21)],
}


# groups that take a whole thread block with 16 channels a thread: in pieces of 16 bytes, pairs and single channels
WIDE = [(torch.bfloat16, 6701, 1, 5120, 320), (torch.float32, 4201, 1, 8192, 512), (torch.bfloat16, 7501, 1, 4098, 288), (torch.float32, 7501, 1, 4097, 288)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,rows,G,D,lanes", [(t, *s) for t, ss in SHAPES.items() for s in ss])
def test_every_row_is_as_by_itself(dtype, rows, G, D, lanes, gated):
    """A row's results do not depend on which pass of a team takes it: the same bits as in calls of so few rows that there is one pass.
    The parameters' gradients are the sum of those calls' (64 bits), up to 15 roundings of a running sum, its own and the results', here and there."""
    check(dtype, rows, G, D, lanes, gated, 17)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,rows,G,D,lanes", WIDE)
def test_every_row_of_the_widest_groups(dtype, rows, G, D, lanes, gated):
    """Their sums of 16 rows are added up without compensation: a rounding each."""
    sums = -(-rows // torch.cuda.get_device_properties(0).multi_processor_count) // 16 + 1
    check(dtype, rows, G, D, lanes, gated, 17 + sums)


def check(dtype, rows, G, D, lanes, gated, roundings):
    assert passes(rows, G, lanes) >= 7
    g = torch.Generator(device="cuda").manual_seed(rows + D)
    rn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    C = G * D
    x, gy, gate = rn(rows, C).to(dtype), rn(rows, C).to(dtype), rn(rows, C).to(dtype) if gated else None
    w, b = 1 + 0.2 * rn(C), 0.2 * rn(C)                        # (32-bit parameters, so that their gradients are not rounded further)
    act = "sigmoid" if D == 64 else "silu"
    got, sums = run(x, w, b, G, gate, act, gy)
    total, size = [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(2)], [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(2)]
    few = 256
    one = lambda t, lo: None if t is None else t[lo:lo + few]
    for lo in range(0, rows, few):
        part, part_sums = run(one(x, lo), w, b, G, one(gate, lo), act, one(gy, lo))
        for a, r in zip(got, part):
            assert torch.equal(a[lo:lo + few], r), lo
        xl = one(x, lo).double().unflatten(1, (G, D))
        xh = ((xl - xl.mean(2, keepdim=True)) * (xl.var(2, correction=0, keepdim=True) + 1e-3).rsqrt()).flatten(1)
        z = (one(gate, lo).double() if gated else xh * w + b).requires_grad_(True)
        p = z * torch.sigmoid(z) if act == "silu" else torch.sigmoid(z)
        dn = one(gy, lo).double() * (p.detach() if gated else torch.autograd.grad(p.sum(), z)[0])
        for i, t in enumerate((dn * xh, dn)):
            total[i] += part_sums[i]
            size[i] += t.abs().sum(0)
    for a, r, m in zip(sums, total, size):
        assert ((a.double() - r).abs() <= 2 * roundings * U * m).all(), ((a.double() - r).abs() / m).max() / U
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, w, b, G, gate=gate, activation=act, eps=1e-3), got[0])
