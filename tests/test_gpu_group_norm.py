"""GPU tests of the group norm with an activation against the float64 restatement, within its bounds."""
import pytest
import torch

from jaxrwkv_b200 import _lib
from jaxrwkv_b200.gated_recurrence import gated_recurrence
from jaxrwkv_b200.group_norm import group_norm_act
from gated_util import check_gated, check_norm, inputs

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
ACTS = ["none", "sigmoid", "silu"]


def make(rows, C, dtype, seed, pdtype=None, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g)
    x = (rn(rows, C) + offset * rn(C)).to(dtype).cuda()
    params = [(1.0 + 0.2 * rn(C)), 0.2 * rn(C)]
    return [x] + [p.to(pdtype or dtype).cuda() for p in params] + [rn(rows, C).to(dtype).cuda(), rn(rows, C).to(dtype).cuda()]


def train(x, w, b, G, gate, act, eps, gy):
    """[out, dx, dweight, dbias, dgate], None for what is not there."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, gate)]
    out = group_norm_act(leaves[0], leaves[1], leaves[2], G, gate=leaves[3], activation=act, eps=eps)
    grads = iter(torch.autograd.grad(out, [t for t in leaves if t is not None], gy))
    return [out] + [None if t is None else next(grads) for t in leaves]


# (rows, groups, channels of a group): teams of one lane up to whole thread blocks, vectors and single channels, teams of one
# group within a block that are added up, more groups than the device has places
SHAPES = [(1, 1, 1), (5, 3, 1), (1, 32, 64), (3, 1, 64), (700, 2, 64), (33, 5, 8), (17, 17, 60), (9, 7, 33), (50, 11, 65), (4, 3, 200), (65, 1, 250),
          (7, 3, 256), (40, 4, 512), (3, 2, 513), (5, 2, 1000), (3, 2, 1024), (2, 1, 2050), (4, 1, 4096), (2, 1, 8192), (2, 1, 8190), (2, 40000, 4),
          (1300, 4, 16)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,G,D", SHAPES)
def test_forward_and_backward(rows, G, D, dtype, gated):
    x, w, b, gate, gy = make(rows, G * D, dtype, seed=rows + G + D)
    gate = gate if gated else None
    got = train(x, w, b, G, gate, "silu", 1e-3, gy)
    check_norm(got, x, w, b, G, gate, "silu", 1e-3, gy)
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, w, b, G, gate=gate, eps=1e-3), got[0])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("there", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype,pdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float32, torch.bfloat16)])
def test_activations_and_parameters(act, gated, there, dtype, pdtype):
    x, w, b, gate, gy = make(70, 192, dtype, seed=3, pdtype=pdtype)
    w, b, gate = w if there[0] else None, b if there[1] else None, gate if gated else None
    check_norm(train(x, w, b, 3, gate, act, 64e-5, gy), x, w, b, 3, gate, act, 64e-5, gy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 63])
def test_rows_where_they_lie(dtype, D):
    """Parts of wider rows, leading axes, shared rows, an address that suits one element only."""
    C = 2 * D
    x, w, b, gate, gy = make(24, C, dtype, seed=4)
    want = train(x, w, b, 2, gate, "silu", 1e-5, gy)
    for pad in (0, 8, 1):
        wide = torch.cat([x, gate, x[:, :pad]], dim=1)
        for got, ref in zip(train(wide[:, :C], w, b, 2, wide[:, C:2 * C], "silu", 1e-5, gy), want):
            if pad == 1 or D == 63:                 # other pieces, other order of the sums
                continue
            assert torch.equal(got, ref)
        check_norm(train(wide[:, :C], w, b, 2, wide[:, C:2 * C], "silu", 1e-5, gy), x, w, b, 2, gate, "silu", 1e-5, gy)
    lead = lambda t: t.reshape(2, 3, 4, C)
    for got, ref in zip(train(lead(x), w, b, 2, lead(gate), "silu", 1e-5, lead(gy)), want):
        assert torch.equal(got.reshape(ref.shape), ref)
    turned = x.reshape(4, 6, C).transpose(0, 1)
    got = train(turned, w, b, 2, None, "silu", 1e-5, gy.reshape(6, 4, C))
    check_norm(got, turned.contiguous(), w, b, 2, None, "silu", 1e-5, gy.reshape(6, 4, C))
    shared = x[:1].expand(24, C)
    check_norm(train(shared, w, b, 2, gate[:1].expand(24, C), "silu", 1e-5, gy), shared, w, b, 2, gate[:1].expand(24, C), "silu", 1e-5, gy)
    odd = torch.empty(24 * C + 1, dtype=dtype, device="cuda")[1:].view(24, C).copy_(x)
    check_norm(train(odd, w, b, 2, gate, "silu", 1e-5, gy), x, w, b, 2, gate, "silu", 1e-5, gy)


def test_constant_and_far_rows():
    """No variance, and a mean of many deviations: the centred squares are taken from the centred values."""
    x, w, b, _, gy = make(6, 256, torch.float32, seed=5)
    x[0] = 3.0
    x[1] = 0.0
    x[2] += 1000.0
    check_norm(train(x, w, b, 4, None, "silu", 1e-5, gy), x, w, b, 4, None, "silu", 1e-5, gy)


def test_what_is_no_number_stays_in_its_group():
    x, w, b, gate, gy = make(40, 128, torch.bfloat16, seed=6)
    want = train(x, w, b, 2, gate, "silu", 1e-5, gy)
    x2 = x.clone()
    x2[7, 3] = float("nan")
    got = train(x2, w, b, 2, gate, "silu", 1e-5, gy)
    keep = torch.ones(40, 128, dtype=torch.bool, device="cuda")
    keep[7, :64] = False
    for i in (0, 1, 4):
        assert torch.equal(got[i][keep], want[i][keep]) and got[i][7, :64].isnan().all()
    assert torch.equal(got[2][64:], want[2][64:]) and got[2][:64].isnan().all()


def test_only_some_gradients():
    x, w, b, gate, gy = make(300, 64, torch.float32, seed=7)
    full = train(x, w, b, 1, gate, "silu", 1e-5, gy)
    for want in ((0,), (1,), (2,), (3,), (0, 3)):
        leaves = [t.detach().requires_grad_(i in want) for i, t in enumerate((x, w, b, gate))]
        out = group_norm_act(*leaves[:3], 1, gate=leaves[3])
        for g, i in zip(torch.autograd.grad(out, [leaves[i] for i in want], gy), want):
            assert torch.equal(g, full[1 + i])


def test_offsets_beyond_32_bits():
    rows, C, apart = 80, 64, 30_000_000
    x, w, b, _, gy = make(rows, C, torch.bfloat16, seed=8)
    wide = torch.empty(apart * (rows - 1) + C, dtype=torch.bfloat16, device="cuda").as_strided((rows, C), (apart, 1))
    wide.copy_(x)
    for a, r in zip(train(wide, w, b, 1, None, "silu", 1e-5, gy)[:4], train(x, w, b, 1, None, "silu", 1e-5, gy)):
        assert torch.equal(a, r)


def test_refusals_on_the_device():
    x, w, b, gate, gy = make(4, 64, torch.float32, seed=9)
    bad = [lambda: group_norm_act(x, w, b, 5), lambda: group_norm_act(x, w, b, 0), lambda: group_norm_act(x, w, b, -1), lambda: group_norm_act(x, w, b, 2.0),
           lambda: group_norm_act(x, w[:63], b, 2), lambda: group_norm_act(x, w, b.bfloat16(), 2), lambda: group_norm_act(x, w.cpu(), None, 2),
           lambda: group_norm_act(x, w, b, 2, gate=gate.bfloat16()), lambda: group_norm_act(x, w, b, 2, gate=gate[:2]),
           lambda: group_norm_act(x.half(), None, None, 2), lambda: group_norm_act(x[:0], w, b, 2), lambda: group_norm_act(x, w.half(), None, 2),
           lambda: group_norm_act(torch.zeros(1, 8193, device="cuda"), None, None, 1)]
    for call in bad:
        with pytest.raises(_lib.B200WKVError):
            call()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(group_norm_act(leaf, w, b, 2).sum(), leaf, create_graph=True)
    with pytest.raises(_lib.B200WKVError, match="second-order"):
        torch.autograd.grad(g.sum(), leaf)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
        group_norm_act(fw.make_dual(x, x), w, b, 2)


def test_python_path_gives_the_same(monkeypatch):
    """The functions behind the native host path, taken where that hands a call back."""
    class Back:
        def __getattr__(self, name):
            return lambda *a: None
    x, w, b, gate, gy = make(9, 64, torch.bfloat16, seed=10)
    rx, rf, rs, length, ns, rgy, rgs = (t.cuda() for t in inputs(2, 70, 24, "decay", torch.bfloat16, seed=11, starts=0.05))

    def recur():
        leaves = [t.detach().requires_grad_(True) for t in (rx, rf, rs)]
        s_out, out = gated_recurrence(*leaves, length, ns, gate="decay")
        return [s_out, out, *torch.autograd.grad((s_out, out), leaves, (rgs, rgy))]
    from jaxrwkv_b200.gated_recurrence import gated_recurrence_step

    def steps():
        state = rs.clone()
        return [*gated_recurrence_step(rx[:, 0], rf[:, 0], state, ns[:, 0], length), *gated_recurrence_step(rx[:, 1], rf[:, 1], state, inplace=True)]
    want = train(x, w, b, 2, gate, "silu", 1e-5, gy) + recur() + steps()
    monkeypatch.setattr(_lib, "host", lambda: Back())
    for a, r in zip(train(x, w, b, 2, gate, "silu", 1e-5, gy) + recur() + steps(), want):
        assert torch.equal(a, r)


def test_captured_and_replayed():
    x, w, b, gate, gy = make(100, 128, torch.bfloat16, seed=12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(x, w, b, 2, gate, "silu", 1e-5, gy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = train(x, w, b, 2, gate, "silu", 1e-5, gy)
    for seed in (13, 14):
        new = make(100, 128, torch.bfloat16, seed=seed)
        for to, frm in zip((x, w, b, gate, gy), new):
            to.copy_(frm)
        graph.replay()
        for a, r in zip(got, train(*new[:3], 2, new[3], "silu", 1e-5, new[4])):
            assert torch.equal(a, r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_mixer_of_both(dtype):
    """Projection, recurrence, output stage, projection, as a layer has them: every stage's results and gradients against the
    restatement of that stage on the tensors that reached it."""
    g = torch.Generator().manual_seed(15)
    B, T, D, C, G = 2, 150, 48, 96, 6
    rn = lambda *shape: torch.randn(*shape, generator=g)
    h, w_in, w_out = rn(B, T, D).to(dtype).cuda(), (rn(D, 3 * C) / D ** 0.5).to(dtype).cuda(), (rn(C, D) / C ** 0.5).to(dtype).cuda()
    weight, bias = (1 + 0.1 * rn(C)).to(dtype).cuda().requires_grad_(True), (0.1 * rn(C)).to(dtype).cuda().requires_grad_(True)
    h.requires_grad_(True)
    s = rn(B, C).cuda().requires_grad_(True)
    ns = (torch.rand(B, T, generator=g) < 0.02).cuda()
    length = torch.tensor([T, 99], dtype=torch.int32, device="cuda")
    proj = h @ w_in
    x, f, gate = proj.split(C, dim=2)
    s_out, y = gated_recurrence(x, f, s, length, ns)
    o = group_norm_act(y, weight, bias, G, gate=gate, eps=64e-5)
    out = o @ w_out
    gout, gs = rn(B, T, D).to(dtype).cuda(), rn(B, C).cuda()
    go, gy, ggate, gw, gb, gx, gf, gs0, gh = torch.autograd.grad((out, s_out), (o, y, gate, weight, bias, x, f, s, h), (gout, gs))
    assert torch.isfinite(gh).all()
    check_gated((s_out, y, gx, gf, gs0), x, f, s, length, ns, "sigmoid", gs, gy, "recurrence")
    check_norm([o, gy, gw, gb, ggate], y, weight, bias, G, gate, "silu", 64e-5, go, "output stage")
    # in place of a training step: decode the next token with the same stages
    from jaxrwkv_b200.gated_recurrence import gated_recurrence_step
    with torch.no_grad():
        state = s_out.detach().clone()
        x1, f1, g1 = (h[:, 0] @ w_in).split(C, dim=1)
        _, y1 = gated_recurrence_step(x1, f1, state, inplace=True)
        o1 = group_norm_act(y1, weight, bias, G, gate=g1, eps=64e-5)
    check_norm([o1], y1, weight, bias, G, g1, "silu", 64e-5)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,G,D", [(37, 7, 24), (301, 2, 24), (60, 9, 40), (9, 20, 80), (333, 1, 72), (700, 3, 48), (41, 3, 20), (50, 5, 44), (19, 13, 76),
                                      (2000, 2, 20), (21, 4, 257), (30, 3, 333), (9, 4, 334), (5, 2, 511), (6, 2, 510), (8, 5, 260), (100, 1, 131)])
def test_teams_of_any_size(rows, G, D, dtype, gated):
    """Groups that take three, five, six, seven, nine, ten and more lanes, and single channels up to the widest that a warp has."""
    x, w, b, gate, gy = make(rows, G * D, dtype, seed=rows + G + D)
    gate = gate if gated else None
    got = train(x, w, b, G, gate, "silu", 1e-3, gy)
    check_norm(got, x, w, b, G, gate, "silu", 1e-3, gy)
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, w, b, G, gate=gate, eps=1e-3), got[0])
