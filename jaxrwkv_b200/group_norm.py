"""Group norm of rows of channels with an activation, or times an activated gate: the output stage of RWKV-5, 5.2 and 6
(``group_norm(y) * silu(g)``) and of gated recurrences (:mod:`jaxrwkv_b200.gated_recurrence`).  RWKV-7's, with its bonus
term, is :func:`jaxrwkv_b200.time_mixing.mix_post`.

Host side of ``b200wkv_group_norm_{fwd,bwd}``.  Arrays are CUDA ``torch`` tensors; there is no CPU path.
"""
import torch

from . import _lib
from .gated_recurrence import _rows
from .rwkv7 import _cotangent, _ptr, _stream

ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2}
MAX_GROUP = 8192                # channels of a group


def _check_operands(x, weight, bias, gate, groups):
    ts = [t for t in (x, weight, bias, gate) if t is not None]
    if not all(t.is_cuda for t in ts):
        raise _lib.B200WKVError("group_norm_act: tensors must live on a CUDA device (there is no CPU path)")
    if not all(t.device == x.device for t in ts):
        raise _lib.B200WKVError("group_norm_act: all tensors must live on one device")
    if x.dim() < 1 or x.numel() == 0:
        raise _lib.B200WKVError("group_norm_act: every dimension must be at least 1")
    C = x.shape[-1]
    if C > _lib.INT_MAX:                         # (the library counts them in 32 bits)
        raise _lib.B200WKVError("group_norm_act: more channels than 32 bits count")
    if not (isinstance(groups, int) and groups >= 1 and C % groups == 0 and C // groups <= MAX_GROUP):
        raise _lib.B200WKVError(f"group_norm_act: {C} channels cannot be cut into {groups} groups of at most {MAX_GROUP}")
    if gate is not None and (gate.dtype != x.dtype or gate.shape != x.shape):
        raise _lib.B200WKVError("group_norm_act: the gate must have x's element type and shape")
    params = [p for p in (weight, bias) if p is not None]
    if any(tuple(p.shape) != (C,) for p in params) or len({p.dtype for p in params}) > 1:
        raise _lib.B200WKVError("group_norm_act: weight and bias must be (C,) of one element type")
    return _lib.dtype_code(x.dtype), _lib.dtype_code(params[0].dtype) if params else _lib.F32


def _operands(x, weight, bias, gate):
    C = x.shape[-1]
    rows = x.numel() // C
    xr, gr = _rows(x, (rows, C)), None if gate is None else _rows(gate, (rows, C))
    weight, bias = (None if p is None else p.contiguous() for p in (weight, bias))
    return rows, C, xr, gr, weight, bias


def _front(n, t, dim):
    """``t`` with the mapped axis in front, or shared along it."""
    return None if t is None else t.movedim(dim, 0) if dim is not None else t.expand((n,) + tuple(t.shape))


def _one_by_one(n, ts, dims, call):
    """Results of ``call`` for each of n instances of ``ts``, stacked: what differs between them may be the weights, or be summed over rows."""
    each = [call(*[t if d is None else t.select(d, i) for t, d in zip(ts, dims)]) for i in range(n)]
    return tuple(torch.stack(one) for one in zip(*each))


class _GroupNormBwd(torch.autograd.Function):
    """The backward call as its own function so that it has a batching rule too: dx and, of those that there are and that are wanted, dweight,
    dbias and dgate.  Not differentiable a second time."""

    @staticmethod
    def forward(x, weight, bias, gate, gy, groups, activation, eps, wanted):
        lib = _lib.load()
        code, pcode = _check_operands(x, weight, bias, gate, groups)
        with torch.cuda.device(x.device):
            rows, C, xr, gr, wc, bc = _operands(x, weight, bias, gate)
            gy = _cotangent(gy, x.dtype)
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dgate = None if gate is None else torch.empty_like(dx)
            dw = torch.empty_like(wc) if weight is not None and wanted[0] else None
            db = torch.empty_like(bc) if bias is not None and wanted[1] else None
            wbytes = lib.b200wkv_group_norm_workspace_bytes(rows, C) if dw is not None or db is not None else 0
            room = torch.empty(wbytes, dtype=torch.uint8, device=x.device)
            _lib.check(lib.b200wkv_group_norm_bwd(_stream(), code, rows, C, groups, eps, activation, _ptr(xr), xr.stride(0),
                                                  _ptr(wc), _ptr(bc), pcode, _ptr(gr), 0 if gr is None else gr.stride(0), _ptr(gy),
                                                  _ptr(dx), _ptr(dgate), _ptr(dw), _ptr(db), _ptr(room), wbytes))
        return tuple(t for t in (dx, dw, db, dgate) if t is not None)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *g):
        raise _lib.B200WKVError("group_norm_act: second-order differentiation is not supported")

    @staticmethod
    def vmap(info, in_dims, x, weight, bias, gate, gy, groups, activation, eps, wanted):
        n, ts, dims = info.batch_size, (x, weight, bias, gate, gy), in_dims[:5]
        call = lambda *ts: _GroupNormBwd.apply(*ts, groups, activation, eps, wanted)
        if dims[1] is None and dims[2] is None and not any(wanted):      # rows of one call
            x, gate, gy = (_front(n, t, d) for t, d in zip((x, gate, gy), (dims[0], dims[3], dims[4])))
            out = call(x, weight, bias, gate, gy)
        else:
            out = _one_by_one(n, ts, dims, call)
        return out, (0,) * len(out)


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(x, weight, bias, gate, groups, activation, eps):
        lib = _lib.load()
        code, pcode = _check_operands(x, weight, bias, gate, groups)
        with torch.cuda.device(x.device):
            rows, C, xr, gr, weight, bias = _operands(x, weight, bias, gate)
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            _lib.check(lib.b200wkv_group_norm_fwd(_stream(), code, rows, C, groups, eps, activation, _ptr(xr), xr.stride(0), _ptr(weight),
                                                  _ptr(bias), pcode, _ptr(gr), 0 if gr is None else gr.stride(0), _ptr(out)))
        return out

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, bias, gate, ctx.groups, ctx.activation, ctx.eps = inputs
        ctx.there = [t is not None for t in (weight, bias, gate)]
        empty = x.new_empty(0)
        ctx.save_for_backward(x, *[empty if t is None else t for t in (weight, bias, gate)])

    @staticmethod
    def backward(ctx, gy):
        x, *rest = ctx.saved_tensors
        weight, bias, gate = (t if there else None for t, there in zip(rest, ctx.there))
        wanted = tuple(there and need for there, need in zip(ctx.there, ctx.needs_input_grad[1:3]))
        grads = iter(_GroupNormBwd.apply(x, weight, bias, gate, gy, ctx.groups, ctx.activation, ctx.eps, wanted))
        dx, dw, db, dgate = (next(grads) if there else None for there in (True, *wanted, gate is not None))
        return dx, dw, db, dgate, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, weight, bias, gate, groups, activation, eps):
        n, call = info.batch_size, lambda *ts: _GroupNormAct.apply(*ts, groups, activation, eps)
        if in_dims[1] is None and in_dims[2] is None:                    # rows of one call
            return call(_front(n, x, in_dims[0]), weight, bias, _front(n, gate, in_dims[3])), 0
        return _one_by_one(n, (x, weight, bias, gate), in_dims[:4], lambda *ts: (call(*ts),))[0], 0


def group_norm_act(x, weight, bias, groups, gate=None, activation="silu", eps=1e-5):
    """Differentiable.  ``x`` (..., C) -> (..., C): ``n = (x - mean) / sqrt(var + eps) * weight + bias`` with mean and variance
    over each row's ``groups`` groups of ``C // groups`` consecutive channels (at most 8192), then ``act(n)``, or
    ``n * act(gate)`` where a gate of x's shape is given.

    ``activation`` is "none", "sigmoid" or "silu", which is 0 far below zero and of -inf too: a closed gate lets nothing through.
    ``weight`` and ``bias`` are (C,), float32 or bfloat16, each may be None.
    ``x`` and ``gate`` are read where they lie as long as their channels are adjacent and their rows evenly spaced (parts of
    a projection's rows).  The arithmetic is float32, results are rounded once.

    Under ``torch.func.vmap`` instances that share weight and bias are rows of one call; those that do not, and gradients of weight
    and bias for each instance, are calls one by one.
    """
    if activation not in ACTIVATIONS:
        raise _lib.B200WKVError(f"group_norm_act: activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    code = ACTIVATIONS[activation]
    if x.is_cuda:
        native = _lib.host().group_norm(x, weight, bias, gate, groups, code, float(eps))
        if native is not None:                   # None: a transform such as vmap, or arguments that need a closer look
            return native
    return _GroupNormAct.apply(x, weight, bias, gate, groups, code, float(eps))
