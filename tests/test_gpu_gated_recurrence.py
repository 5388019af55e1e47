"""GPU tests of the gated linear recurrence and its step against the float64 restatement, within its running bounds."""
import pytest
import torch

from jaxrwkv_b200 import _lib
from jaxrwkv_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
from gated_util import check_gated, inputs, np64, within
from oracle import gated as og

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
GATES = ["sigmoid", "decay"]


def cuda(*ts):
    return [t.cuda() for t in ts]


def train(x, f, s, length, ns, gate, gs, gy):
    """(s_out, out, dx, df, ds) of operands that live on the GPU."""
    x, f, s = (t.detach().requires_grad_(True) for t in (x, f, s))
    s_out, out = gated_recurrence(x, f, s, length, ns, gate=gate)
    return (s_out, out) + torch.autograd.grad((s_out, out), (x, f, s), (gs, gy))


# lengths around the sizes of segments, tiles and clusters; channels that pairs and vectors of them do not divide
SHAPES = [(1, 1, 1), (2, 1, 66), (1, 2, 8), (3, 7, 31), (2, 8, 64), (1, 9, 33), (2, 17, 130), (2, 63, 40), (1, 64, 2), (2, 65, 62),
          (3, 129, 96), (2, 257, 264), (1, 600, 127), (2, 1100, 36), (1, 2100, 8)]


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C", SHAPES)
def test_forward_and_backward(B, T, C, dtype, gate):
    x, f, s, length, ns, gy, gs = cuda(*inputs(B, T, C, gate, dtype, seed=B + T + C, starts=0.03))
    check_gated(train(x, f, s, length, ns, gate, gs, gy), x, f, s, length, ns, gate, gs, gy)
    check_gated(gated_recurrence(x, f, s, length, ns, gate=gate), x, f, s, length, ns, gate)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences_and_channels(dtype):
    """More sequences than fit on the device at once, and rows long enough for whole vectors."""
    x, f, s, length, ns, gy, gs = cuda(*inputs(9, 200, 2056, "sigmoid", dtype, seed=1, starts=0.01))
    got = train(x, f, s, length, ns, "sigmoid", gs, gy)
    for b in (0, 4, 8):
        cut = slice(b, b + 1)
        check_gated([t[cut] for t in got], x[cut], f[cut], s[cut], length[cut], ns[cut], "sigmoid", gs[cut], gy[cut])


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C", [(150, 8), (150, 6), (150, 5), (4, 2600)])
def test_a_thread_block_a_sequence(B, C, dtype, gate):
    """So many sequences or channels that none is shared: some of them, over several tiles, in pieces of every size."""
    x, f, s, length, ns, gy, gs = cuda(*inputs(B, 300, C, gate, dtype, seed=C, starts=0.02))
    got = train(x, f, s, length, ns, gate, gs, gy)
    for b in (0, B // 2, B - 1):
        cut, ch = slice(b, b + 1), slice(max(0, C - 40), C)
        check_gated([t[cut][..., ch] for t in got], x[cut][..., ch], f[cut][..., ch], s[cut][..., ch], length[cut], ns[cut], gate, gs[cut][..., ch],
                    gy[cut][..., ch])


def test_more_sequences_than_a_grid_axis():
    B = 70001
    x, f, s, length, ns, gy, gs = cuda(*inputs(B, 2, 2, "sigmoid", torch.bfloat16, seed=3, starts=0.1))
    got = train(x, f, s, length, ns, "sigmoid", gs, gy)
    at = [0, 65534, 65535, 65536, B - 1]
    check_gated([t[at] for t in got], x[at], f[at], s[at], length[at], ns[at], "sigmoid", gs[at], gy[at])


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("lengths", [[0, 0, 0], [1, 130, 64], [65, 63, 128], [300, 1000, 129]])
def test_lengths_and_dense_flags(lengths, gate):
    """The returned state at every kind of place (longer than T is T); flags on almost every token."""
    x, f, s, length, ns, gy, gs = cuda(*inputs(3, 130, 34, gate, torch.float32, seed=2, starts=0.6, lengths=lengths))
    ns[0, 0] = True
    check_gated(train(x, f, s, length, ns, gate, gs, gy), x, f, s, length, ns, gate, gs, gy)


@pytest.mark.parametrize("T", [1, 70])
def test_without_flags_and_with_python_values(T):
    x, f, s, _, _, gy, gs = cuda(*inputs(2, T, 16, "decay", torch.float32, seed=4))
    none = torch.zeros(2, T, dtype=torch.bool, device="cuda")
    full = torch.full((2,), T, dtype=torch.int32, device="cuda")
    want = gated_recurrence(x, f, s, full, none, gate="decay")
    for length, ns in ((None, None), (T, None), (full.long(), none.int()), (torch.tensor(T), False), (full.cpu(), none[0])):
        for a, b in zip(gated_recurrence(x, f, s, length, ns, gate="decay"), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [32, 33])
def test_operands_where_they_lie(dtype, C):
    """Halves of one projection's rows, a transposed batch, shared rows, an address that suits one element only: the same bits as
    dense copies."""
    x, f, s, length, ns, gy, gs = cuda(*inputs(3, 75, C, "sigmoid", dtype, seed=6, starts=0.05))
    want = train(x, f, s, length, ns, "sigmoid", gs, gy)
    both = torch.cat([x, f], dim=2)
    odd = torch.empty(3 * 75 * C + 1, dtype=dtype, device="cuda")[1:].view(3, 75, C).copy_(x)
    s_odd = torch.empty(3 * C + 1, device="cuda")[1:].view(3, C).copy_(s)
    turned = f.transpose(0, 1).contiguous().transpose(0, 1)
    for xx, ff, ss in ((both[..., :C], both[..., C:], s), (odd, f, s_odd), (x, turned, s), (x.mT.contiguous().mT, f, s.t().contiguous().t())):
        for a, b in zip(train(xx, ff, ss, length, ns, "sigmoid", gs, gy), want):
            assert torch.equal(a, b)
    shared = f[:1, :1].expand(3, 75, C)
    for a, b in zip(train(x, shared, s, length, ns, "sigmoid", gs, gy), train(x, shared.contiguous(), s, length, ns, "sigmoid", gs, gy)):
        assert torch.equal(a, b)


def test_strided_and_shared_cotangents():
    x, f, s, length, ns, gy, gs = cuda(*inputs(2, 70, 24, "decay", torch.bfloat16, seed=7))
    want = train(x, f, s, length, ns, "decay", gs[:, :1].expand_as(gs), gy[:, :1].expand_as(gy))
    got = train(x, f, s, length, ns, "decay", gs[:, :1].expand_as(gs).contiguous(), gy[:, :1].expand_as(gy).contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [100, 900])
def test_one_cotangent_alone(T):
    x, f, s, length, ns, gy, gs = cuda(*inputs(2, T, 24, "sigmoid", torch.float32, seed=8, starts=0.02))
    for use_state in (False, True):
        leaves = [t.detach().requires_grad_(True) for t in (x, f, s)]
        s_out, out = gated_recurrence(*leaves, length, ns)
        g = torch.autograd.grad(s_out if use_state else out, leaves, gs if use_state else gy)
        zero = (gs, torch.zeros_like(gy)) if use_state else (torch.zeros_like(gs), gy)
        check_gated((s_out, out) + g, x, f, s, length, ns, "sigmoid", *zero)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_beyond_32_bits(dtype, gate):
    """Rows so far apart that their offsets pass 2^31 elements."""
    T, C, apart = 80, 48, 30_000_001 if dtype == torch.float32 else 30_000_000
    x, f, s, length, ns, gy, gs = cuda(*inputs(1, T, C, gate, dtype, seed=9))
    wide = torch.empty(apart * (T - 1) + C, dtype=dtype, device="cuda").as_strided((1, T, C), (0, apart, 1))
    wide.copy_(x)
    check_gated(train(wide, f, s, length, ns, gate, gs, gy), x, f, s, length, ns, gate, gs, gy)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [1, 8, 40, 64, 129])
def test_a_start_flag_drops_what_is_no_number(at, dtype, gate):
    """Operands, state and cotangents that are no numbers do not pass a flag in either direction."""
    T = 200
    x, f, s, _, ns, gy, gs = cuda(*inputs(2, T, 40, gate, dtype, seed=10))
    length = torch.tensor([T, at], dtype=torch.int32, device="cuda")
    ns[:, at] = True
    clean = train(x, f, s, length, ns, gate, gs, gy)
    for value in (float("nan"), float("inf")):
        x2, f2, s2, gy2 = x.clone(), f.clone(), s.clone(), gy.clone()
        x2[:, :at], s2[:], f2[:, :at, ::2] = value, value, float("nan")
        got = train(x2, f2, s2, length, ns, gate, gs, gy)
        for i in (1, 2, 3):                       # behind the flag: outputs and gradients as if nothing had been there
            assert torch.equal(got[i][:, at:], clean[i][:, at:])
        gy2[:, at:] = value
        got = train(x, f, s, length, ns, gate, gs * torch.tensor([[value], [1.0]], device="cuda"), gy2)
        for i in (2, 3):                          # in front of it: gradients likewise (the second's state ends at the flag)
            assert torch.equal(got[i][:, :at], clean[i][:, :at])
        assert torch.equal(got[4], clean[4])


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("at", [3, 66, 130])
def test_a_gate_that_is_no_number_stays_in_its_channel(at, gate):
    """Behind a flag of its own segment, in every second channel."""
    x, f, s, length, ns, gy, gs = cuda(*inputs(2, 200, 40, gate, torch.bfloat16, seed=20, lengths=[200, 150]))
    s[:] = float("inf")
    ns[:, at - 1] = True
    clean = train(x, f, s, length, ns, gate, gs, gy)
    f2 = f.clone()
    f2[:, at, ::2] = float("nan")
    got = train(x, f2, s, length, ns, gate, gs, gy)
    for i in range(5):
        assert torch.equal(got[i][..., 1::2].nan_to_num(7.0), clean[i][..., 1::2].nan_to_num(7.0))
    assert got[1][:, at:, ::2].isnan().all() and torch.equal(got[1][:, at - 1, ::2], clean[1][:, at - 1, ::2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_gates(dtype):
    """Gates at the ends of their range: exactly 0 and 1, and no gradient that is no number."""
    inf = float("inf")
    values = torch.tensor([-inf, -1e30, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 1e30, inf])
    T = 66
    f = values.repeat(T).reshape(T, -1)[None].clone()
    f[0, ::3] = f[0, ::3].flip(-1)
    g = torch.Generator().manual_seed(11)
    x, s, gy, gs = (torch.randn(*shape, generator=g) for shape in ((1, T, 11), (1, 11), (1, T, 11), (1, 11)))
    x, f, s, gy, gs = x.to(dtype).cuda(), f.to(dtype).cuda(), s.cuda(), gy.to(dtype).cuda(), gs.cuda()
    length, ns = torch.tensor([T], device="cuda"), torch.zeros(1, T, dtype=torch.bool, device="cuda")
    for gate in GATES:
        got = train(x, f, s, length, ns, gate, gs, gy)
        assert all(torch.isfinite(t).all() for t in got)
        # (a gate of e^-90 may be flushed to 0: 1e-38 of the largest state, far below any bound here; the state grows to T |x| at most)
        x64, f64 = np64(x[0]), np64(f[0])
        ref, _ = og.gated(x64, f64, np64(s[0]), T, np64(ns[0]), gate)
        grads, _ = og.gated_bwd(x64, f64, np64(s[0]), T, np64(ns[0]), gate, np64(gs[0]), np64(gy[0]))
        # arguments of up to 90 in the hardware's exponential are off by 107 ulp = 214 U; sums of at most T + 1 terms of at most 5 each,
        # each term with T gates behind it
        worst = (T + 1) * 5 * (T * 250 if dtype == torch.bfloat16 else T * 20) * og.U
        for a, b in zip(got, ref + grads):
            within(a[0], b, worst, gate)


def test_leading_axes_and_vmap():
    x, f, s, length, ns, gy, gs = cuda(*inputs(6, 37, 16, "sigmoid", torch.float32, seed=12, starts=0.05))
    want = train(x, f, s, length, ns, "sigmoid", gs, gy)
    lead = lambda t: t.reshape(2, 3, *t.shape[1:])
    got = train(*[lead(t) for t in (x, f, s, length, ns)], "sigmoid", lead(gs), lead(gy))
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    one = gated_recurrence(x[0], f[0], s[0], length[0], ns[0])
    assert torch.equal(one[1], want[1][0]) and torch.equal(one[0], want[0][0])

    def loss(x, f, s, length, ns, gs, gy):
        s_out, out = gated_recurrence(x, f, s, length, ns)
        return (s_out * gs).sum() + (out * gy).sum()
    g = torch.func.vmap(torch.func.vmap(torch.func.grad(loss, argnums=(0, 1, 2))))(*[lead(t) for t in (x, f, s, length, ns, gs, gy)])
    for a, b in zip(g, want[2:]):
        assert torch.equal(a.reshape(b.shape), b)
    out = torch.func.vmap(lambda x, s: gated_recurrence(x, f[0], s, 37, ns[0]), in_dims=(0, 0))(x, s)
    ref = gated_recurrence(x, f[:1].expand_as(f), s, 37, ns[:1].expand_as(ns))
    for a, b in zip(out, ref):
        assert torch.equal(a, b)


def test_refusals_on_the_device():
    x, f, s, length, ns, gy, gs = cuda(*inputs(2, 9, 16, "sigmoid", torch.float32, seed=13))
    bad = [lambda: gated_recurrence(x, f.bfloat16(), s), lambda: gated_recurrence(x, f[:, :8], s), lambda: gated_recurrence(x, f, s[:1]),
           lambda: gated_recurrence(x, f, s.bfloat16()), lambda: gated_recurrence(x.half(), f.half(), s), lambda: gated_recurrence(x, f, s.cpu()),
           lambda: gated_recurrence(x[:, :0], f[:, :0], s), lambda: gated_recurrence_step(x[:, 0], f[:, 0], s[:1]),
           lambda: gated_recurrence_step(x[:, 0], f[:, 0], s.clone().requires_grad_(True)),
           lambda: gated_recurrence_step(x[:, 0], f[:, 0], s.t().contiguous().t(), inplace=True),
           lambda: gated_recurrence_step(x[:, 0], f[:, 0], s[:1].expand_as(s), inplace=True)]
    for call in bad:
        with pytest.raises(_lib.B200WKVError):
            call()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(gated_recurrence(leaf, f, s)[1].sum(), leaf, create_graph=True)
    with pytest.raises(_lib.B200WKVError, match="second-order"):
        torch.autograd.grad(g.sum(), leaf)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
        gated_recurrence(fw.make_dual(x, x), f, s)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C", [(1, 1), (3, 33), (2, 2048), (300, 70)])
def test_step(B, C, dtype, gate):
    x, f, s, length, ns, _, _ = cuda(*inputs(B, 1, C, gate, dtype, seed=14, starts=0.3))
    s_out, out = gated_recurrence_step(x[:, 0], f[:, 0], s, ns[:, 0], length, gate=gate)
    check_gated((s_out, out[:, None]), x, f, s, length, ns, gate)
    wide = torch.zeros(B, 3, C + 5, device="cuda")
    wide[:, 1, :C] = s
    state = wide[:, 1, :C]
    before = state._version
    same, out2 = gated_recurrence_step(x[:, 0], f[:, 0], state, ns[:, 0], length, gate=gate, inplace=True)
    assert same is state and torch.equal(state, s_out) and torch.equal(out, out2) and state._version > before
    assert wide[:, [0, 2]].eq(0).all() and wide[:, 1, C:].eq(0).all()
    seq = gated_recurrence(x, f, s, length, ns, gate=gate)
    assert torch.equal(seq[0], s_out) and torch.equal(seq[1][:, 0], out)
    column = gated_recurrence_step(x[:, 0], f[:, 0], s, ns, length, gate=gate)      # flags as a sequence of one token has them
    assert torch.equal(column[0], s_out) and torch.equal(column[1], out)
    lead = gated_recurrence_step(x.reshape(1, B, C), f.reshape(1, B, C), s[None], ns.reshape(1, B), length[None], gate=gate)
    assert torch.equal(lead[0][0], s_out) and torch.equal(lead[1][0], out)


@pytest.mark.parametrize("gate", GATES)
def test_steps_continue_a_sequence(gate):
    """A prompt in one call, then token by token: within the bounds of the whole sequence."""
    x, f, s, _, ns, _, _ = cuda(*inputs(2, 90, 48, gate, torch.bfloat16, seed=15, starts=0.02))
    length = torch.tensor([90, 90], dtype=torch.int32, device="cuda")
    state, out = gated_recurrence(x[:, :70], f[:, :70], s, None, ns[:, :70], gate=gate)
    outs = [out]
    for t in range(70, 90):
        state, o = gated_recurrence_step(x[:, t], f[:, t], state, ns[:, t], gate=gate, inplace=True)
        outs.append(o[:, None])
    check_gated((state, torch.cat(outs, 1)), x, f, s, length, ns, gate)


def test_inference_mode():
    """Tensors without a version counter, the state updated where it lies."""
    with torch.inference_mode():
        x, f, s, length, ns, _, _ = cuda(*inputs(2, 70, 48, "sigmoid", torch.bfloat16, seed=19))
        state, out = gated_recurrence(x, f, s, length, ns)
        check_gated((state, out), x, f, s, length, ns, "sigmoid")
        same, o = gated_recurrence_step(x[:, 0], f[:, 0], state, inplace=True)
        assert same is state


def test_two_calls_at_once():
    """On two streams, many times over: nothing is shared between calls."""
    sets = [cuda(*inputs(3, 700, 96, "sigmoid", torch.bfloat16, seed=22 + i, starts=0.02)) for i in range(2)]
    run = lambda q: train(q[0], q[1], q[2], q[3], q[4], "sigmoid", q[6], q[5])
    want = [run(q) for q in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for q, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(run(q))
        torch.cuda.synchronize()
        for one, ref in zip(got, want):
            for a, b in zip(one, ref):
                assert torch.equal(a, b)


def test_another_stream_and_captured_calls():
    """On a side stream; forward and backward captured and replayed on new values, two graphs that take turns."""
    make = lambda seed: cuda(*inputs(2, 150, 64, "sigmoid", torch.bfloat16, seed=seed, starts=0.02))
    x, f, s, length, ns, gy, gs = make(16)
    eager = train(x, f, s, length, ns, "sigmoid", gs, gy)       # a graph of its own lives on while others are captured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(train(x, f, s, length, ns, "sigmoid", gs, gy), eager):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    bufs = [[t.clone() for t in (x, f, s, length, ns, gs, gy)] for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        with torch.cuda.stream(side):
            train(*b[:5], "sigmoid", *b[5:])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(train(*b[:5], "sigmoid", *b[5:]))
        graphs.append(graph)
    for seed in (17, 18):
        fresh = [make(seed + 10 * i) for i in range(2)]
        for (x, f, s, length, ns, gy, gs), b in zip(fresh, bufs):
            for to, frm in zip(b, (x, f, s, length, ns, gs, gy)):
                to.copy_(frm)
        graphs[0].replay()
        graphs[1].replay()
        for (x, f, s, length, ns, gy, gs), got in zip(fresh, outs):
            for a, b in zip(got, train(x, f, s, length, ns, "sigmoid", gs, gy)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,C", [(19, 5), (70, 64), (150, 65), (150, 72), (300, 67), (600, 130)])
def test_rows_that_begin_anywhere(T, C, dtype):
    """Rows at every distance from 16 bytes, by where the tensor begins and by its token stride, amid values that are no numbers."""
    B, gate = 2, "sigmoid"
    x, f, s, length, ns, gy, gs = cuda(*inputs(B, T, C, gate, dtype, seed=T + C, starts=0.03))
    want = train(x, f, s, length, ns, gate, gs, gy)
    check_gated(want, x, f, s, length, ns, gate, gs, gy)

    def placed(t, begin, apart):
        room = torch.full((begin + B * T * apart,), float("nan"), dtype=dtype, device="cuda")
        there = room[begin:].view(B, T, apart)[..., :C]
        return there.copy_(t)

    for begin in range(9):
        px, pf = placed(x, begin, C + begin % 3), placed(f, 8 - begin, C + 7)
        for a, b in zip(train(px, pf, s, length, ns, gate, gs, gy), want):
            assert torch.equal(a, b)
        s_out, out = gated_recurrence(px, pf, s, length, ns, gate=gate)
        check_gated((s_out, out), x, f, s, length, ns, gate)
