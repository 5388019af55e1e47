"""Gated linear recurrence, one number of state per channel, and its single-token step.

``gated_recurrence`` computes ``h_t = a_t h_{t-1} + u_t`` over sequences of any length, with the conventions of this
package's other recurrences: start flags inside the sequences, a carried state in and out, ``length``, gradients from and
into the state, any number of leading batch axes, ``torch.func.vmap``.  Two gates:

* ``"sigmoid"``: ``a = sigmoid(f)``, ``u = (1 - a) x`` - the state is a running mean that the forget gate ``f`` opens;
* ``"decay"``: ``a = exp(-exp(f))``, ``u = x`` - ``f`` is the raw log-log decay, as RWKV-7's ``w``.

Host side of ``b200wkv_gated_{fwd,bwd,step}``.  Arrays are CUDA ``torch`` tensors; there is no CPU path.
"""
import torch

from . import _lib
from .rwkv7 import _cotangent, _ptr, _stream, _vmap_flags, _vmap_front

GATES = {"sigmoid": 0, "decay": 1}


def _gate_code(gate):
    if gate not in GATES:
        raise _lib.B200WKVError(f"gated_recurrence: gate must be one of {sorted(GATES)}, not {gate!r}")
    return GATES[gate]


def _check_operands(x, f, s, state_shape):
    if not all(t.is_cuda for t in (x, f, s)):
        raise _lib.B200WKVError("gated_recurrence: tensors must live on a CUDA device (there is no CPU path)")
    if not (x.device == f.device == s.device):
        raise _lib.B200WKVError("gated_recurrence: x, f and s must live on one device")
    if x.dtype != f.dtype:
        raise _lib.B200WKVError("gated_recurrence: x and f must share one element type")
    if s.dtype != torch.float32:
        raise _lib.B200WKVError("gated_recurrence: the state is kept in float32")
    if x.shape != f.shape or tuple(s.shape) != tuple(state_shape):
        raise _lib.B200WKVError(f"gated_recurrence: shapes do not fit: x {tuple(x.shape)}, f {tuple(f.shape)}, s {tuple(s.shape)}")
    if x.dim() == 0 or x.numel() == 0:
        raise _lib.B200WKVError("gated_recurrence: there must be channels, and every dimension must be at least 1")
    if x.numel() // x.shape[-1] > _lib.INT_MAX or x.shape[-1] > _lib.INT_MAX:          # (the library counts both in 32 bits)
        raise _lib.B200WKVError("gated_recurrence: more tokens or channels than 32 bits count")
    return _lib.dtype_code(x.dtype)


def _rows(t, shape):
    """``t`` as rows of adjacent channels, where it lies if it can be."""
    t = t.reshape(shape)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _flag_bytes(length, new_starts, lead, tail, device):
    if length is not None:
        length = torch.as_tensor(length, device=device).expand(lead).to(torch.int32).contiguous()
    if new_starts is not None:
        new_starts = torch.as_tensor(new_starts, device=device)
        new_starts = (new_starts if new_starts.dtype == torch.bool else new_starts.to(torch.uint8)).expand(lead + tail).contiguous()
    return length, new_starts


def _dims(x):
    lead = tuple(x.shape[:-2])
    B = 1
    for d in lead:
        B *= d
    return lead, B, x.shape[-2], x.shape[-1]


class _GatedBwd(torch.autograd.Function):
    """The backward call as its own function so that it has a batching rule too.  Not differentiable a second time."""

    @staticmethod
    def forward(x, f, length, new_starts, residual, gs, gy, gate):
        lib = _lib.load()
        lead, B, T, C = _dims(x)
        with torch.cuda.device(x.device):
            xr, fr = _rows(x, (B, T, C)), _rows(f, (B, T, C))
            length, new_starts = _flag_bytes(length, new_starts, lead, (T,), x.device)
            gs = None if gs is None else gs.to(torch.float32).contiguous()
            gy, residual = _cotangent(gy, x.dtype), _cotangent(residual, torch.uint8)
            if residual.numel() != lib.b200wkv_gated_residual_bytes(B, T, C):
                raise _lib.B200WKVError("gated_recurrence: the residual is another call's")
            dx, df = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
            ds = torch.empty(lead + (C,), dtype=torch.float32, device=x.device)
            _lib.check(lib.b200wkv_gated_bwd(_stream(), _lib.dtype_code(x.dtype), gate, B, T, C, _ptr(xr), xr.stride(0), xr.stride(1),
                                             _ptr(fr), fr.stride(0), fr.stride(1), _ptr(length), _ptr(new_starts), _ptr(gy), _ptr(gs),
                                             _ptr(residual), residual.numel(), _ptr(dx), _ptr(df), _ptr(ds)))
        return dx, df, ds

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *g):
        raise _lib.B200WKVError("gated_recurrence: second-order differentiation is not supported")

    @staticmethod
    def vmap(info, in_dims, x, f, length, new_starts, residual, gs, gy, gate):
        length, new_starts = _vmap_flags(length, new_starts, in_dims[2:4], _rank(x, in_dims[0]))
        x, f, residual, gs, gy = _batched(info.batch_size, (x, f, residual, gs, gy), in_dims[:2] + in_dims[4:7])
        return _GatedBwd.apply(x, f, length, new_starts, residual, gs, gy, gate), (0, 0, 0)


def _rank(x, dim):
    """Leading axes of an instance's x (..., T, C)."""
    return x.dim() - 2 - (dim is not None)


def _batched(n, xs, dims):
    """Every argument with the new axis in front, those without one shared along it."""
    return _vmap_front(n, xs, dims, (False,) * len(xs))


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(x, f, s, length, new_starts, gate):
        lib = _lib.load()
        lead, B, T, C = _dims(x)
        code = _check_operands(x, f, s, lead + (C,))
        with torch.cuda.device(x.device):
            xr, fr, sr = _rows(x, (B, T, C)), _rows(f, (B, T, C)), s.contiguous()
            length, new_starts = _flag_bytes(length, new_starts, lead, (T,), x.device)
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            s_out = torch.empty(lead + (C,), dtype=torch.float32, device=x.device)
            rbytes = lib.b200wkv_gated_residual_bytes(B, T, C)
            # by sequences, so that a call under vmap hands each instance its own, and a backward call sees whose they are
            residual = torch.empty(lead + (rbytes // B,), dtype=torch.uint8, device=x.device)
            _lib.check(lib.b200wkv_gated_fwd(_stream(), code, gate, B, T, C, _ptr(xr), xr.stride(0), xr.stride(1), _ptr(fr), fr.stride(0),
                                             fr.stride(1), _ptr(sr), _ptr(length), _ptr(new_starts), _ptr(out), _ptr(s_out),
                                             _ptr(residual), rbytes))
        return s_out, out, residual

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, f, s, length, new_starts, gate = inputs
        ctx.gate = gate
        ctx.flags = [t is not None for t in (length, new_starts)]
        empty = x.new_empty(0)
        ctx.save_for_backward(x, f, *[empty if t is None else torch.as_tensor(t) for t in (length, new_starts)], output[2])
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(output[2])

    @staticmethod
    def backward(ctx, gs, gy, _gres):
        x, f, length, new_starts, residual = ctx.saved_tensors
        length, new_starts = (t if there else None for t, there in zip((length, new_starts), ctx.flags))
        dx, df, ds = _GatedBwd.apply(x, f, length, new_starts, residual, gs, gy, ctx.gate)
        return dx, df, ds, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, f, s, length, new_starts, gate):
        length, new_starts = _vmap_flags(length, new_starts, in_dims[3:5], _rank(x, in_dims[0]))
        x, f, s = _batched(info.batch_size, (x, f, s), in_dims[:3])
        s_out, out, residual = _Gated.apply(x, f, s, length, new_starts, gate)
        return (s_out, out, residual), (0, 0, 0)


def gated_recurrence(x, f, s, length=None, new_starts=None, gate="sigmoid"):
    """Differentiable.  ``x`` and ``f`` (..., T, C) of one element type, the state ``s`` (..., C) in float32; returns
    ``(s_out, out)``, ``out`` like ``x``.

    ``h_t = a_t h_{t-1} + u_t`` from ``s``, ``out_t = h_t``; a start flag (``new_starts`` (..., T)) drops the state in front
    of its token, whatever it holds; ``s_out`` is the state after token ``length - 1`` (``s`` for length 0), while ``out`` is
    computed for all T tokens.  ``length`` (...) and ``new_starts`` may be shared by the leading axes; None: T everywhere, no
    starts.  ``x`` and ``f`` are read where they lie as long as their channels are adjacent (halves of a projection's rows).
    The arithmetic is float32, ``out`` is rounded once.
    """
    code = _gate_code(gate)
    if x.is_cuda:
        native = _lib.host().gated(x, f, s, length, new_starts, code)
        if native is not None:                   # None: a transform such as vmap, or arguments that need a closer look
            return native
    if x.dim() < 2:
        raise _lib.B200WKVError("gated_recurrence: x must be (..., T, C)")
    s_out, out, _ = _Gated.apply(x, f, s, length, new_starts, code)
    return s_out, out


def gated_recurrence_step(x, f, s, new_starts=None, length=None, gate="sigmoid", inplace=False):
    """One token of :func:`gated_recurrence` without autograd: ``x``, ``f`` and the float32 state ``s`` are (..., C),
    ``length`` (...), ``new_starts`` (...) or (..., 1).  Returns ``(s_out, out)``; a row of length 0 keeps its state and has its output all the same.  With
    ``inplace`` the state is updated where it lies (rows of a wider container may have any distance) and ``s_out`` is ``s``.
    There is no batching rule for ``torch.func.vmap``: leading axes are what it takes instead.
    """
    code = _gate_code(gate)
    if x.is_cuda:
        native = _lib.host().gated_step(x, f, s, new_starts, length, code, bool(inplace))
        if native is not None:                   # None: arguments that need a closer look
            return native
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, f, s)):
        raise _lib.B200WKVError("gated_recurrence_step: has no gradients; call gated_recurrence")
    dtype = _check_operands(x, f, s, x.shape)
    lib = _lib.load()
    lead, C = tuple(x.shape[:-1]), x.shape[-1]
    B = x.numel() // C
    with torch.cuda.device(x.device):
        xr, fr = _rows(x, (B, C)), _rows(f, (B, C))
        if inplace:
            if not (s.is_contiguous() or s.dim() == 2 and (s.stride(1) == 1 or C == 1) and (s.stride(0) >= C or B == 1)):
                raise _lib.B200WKVError("gated_recurrence_step: a state updated in place must be rows of adjacent channels")
            sr = s.view(B, C)
        else:
            sr = _rows(s, (B, C))
        s_out = s if inplace else torch.empty(s.shape, dtype=torch.float32, device=s.device)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if isinstance(new_starts, torch.Tensor) and new_starts.dim() == len(lead) + 1 and new_starts.shape[-1] == 1:
            new_starts = new_starts.squeeze(-1)
        length, new_starts = _flag_bytes(length, new_starts, lead, (), x.device)
        _lib.check(lib.b200wkv_gated_step(_stream(), dtype, code, B, C, _ptr(xr), xr.stride(0), _ptr(fr), fr.stride(0), _ptr(sr), sr.stride(0),
                                          _ptr(length), _ptr(new_starts), _ptr(out), _ptr(s_out), sr.stride(0) if inplace else C))
    if inplace and not s.is_inference():
        torch.autograd.graph.increment_version(s)
    return s_out, out
