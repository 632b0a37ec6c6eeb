"""``Rotary``: rotary positions on queries and keys (adaptq_rotary_* of adaptq.h).

    rotary = Rotary(128, base=500000.0)
    q, k = rotary(positions, q, k)         # [tokens, heads, dim] or [batch, tokens, heads, dim]

Device tensors of fp32, fp16 or bf16, rotated in one launch on torch's current
stream, in fp32 and rounded once.  Differentiable in q and k, backward and forward (dual
tensors of torch.autograd.forward_ad; the transforms of torch.func are refused).  Calls
may be captured into a graph, which the Rotary has to outlive, a backward pass only
together with its forward, on leaves that no graph outside the capture holds (as torch
wants it of any operator).  Tracing (torch.jit.trace, make_fx, torch.export) is refused;
torch.compile runs the calls between its graphs.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import adaptq_py

# ADAPTQ_IO_* and ADAPTQ_ROTARY_* in adaptq.h
IO_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SCALINGS = {None: 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


# torch's current stream of a device as an address; without the Stream object around it where
# torch has that call (0.1 us instead of 1.7, of 8 to 11 that a small call takes the host)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device: torch.device) -> int:
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


# Bound here, as _raw_stream is, for a small call's host time: a check of both costs 0.1 us.
tracing_state = torch._C._get_tracing_state
dispatch_modes = torch._C._len_torch_dispatch_stack
increment_version = torch._C._increment_version  # of a sequence of tensors


def refuse_tracing(what: str) -> None:
    """Called where tracing_state() or dispatch_modes() is set.  A call goes to the library by
    address, past torch's dispatcher: a program traced through it would hold the output's
    allocation alone and return memory that nobody wrote."""
    if tracing_state() is None:
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if get_proxy_mode() is None:
            return
    raise RuntimeError(f"{what} cannot be traced; leave its calls out of the traced program")


class Rotary:
    """Rotation of the first ``dim`` channels of a row: pairs (i, i + dim/2), or
    (2i, 2i + 1) with ``interleaved``, by position * base^(-2i/dim).

    scaling, for contexts longer than a model was trained on:

    - "linear": every angle divided by ``factor``;
    - "ntk": base * factor^(dim/(dim-2)) in place of base;
    - "bands": pairs that turn more than ``fast`` (4) times over ``context``
      positions stay, those below ``slow`` (1) are divided by factor, linear between;
    - "yarn": the same with the ramp over the pairs' numbers and ``fast`` 32, and
      cosine and sine times 0.1 ln(factor) + 1.

    ``amplitude`` replaces the factor on cosine and sine (1, but for "yarn").  The
    object lives on ``device`` (the current one).
    """

    def __init__(self, dim: int, *, base: float = 10000.0, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, context: int = 0,
                 slow: float | None = None, fast: float | None = None,
                 amplitude: float | None = None, device=None):
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {list(SCALINGS)}, got {scaling!r}")
        for name, x in (("slow", slow), ("fast", fast), ("amplitude", amplitude)):
            if x is not None and not x > 0:
                raise ValueError(f"{name} must be positive, got {x}")
        self.dim = dim
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise ValueError(f"Rotary lives on a GPU, got device {self.device}")
        with torch.cuda.device(self.device):
            self.device = torch.device("cuda", torch.cuda.current_device())
            self._handle = adaptq_py.Rotary(dim, interleaved, base, SCALINGS[scaling], factor,
                                            context, slow or 0.0, fast or 0.0, amplitude or 0.0)

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, *,
                 inplace: bool = False):
        """Rotated q, or (q, k).  positions: int32 [tokens] or [batch, tokens]; q, k: [tokens,
        heads, dim] or [batch, tokens, heads, dim] of one type, any strides with rows side by
        side.  inplace: writes into q and k (not where they need gradients)."""
        if _differentiated(q, k):
            if inplace:
                raise ValueError("inplace rotation of tensors that need gradients")
            out = _Rotate.apply(self, positions, False, q, k)
        else:
            out = self._rotate(positions, q, k, inplace, False)
        return out if k is not None else out[0]

    def _turn(self, positions, q, k, backward):
        if _differentiated(q, k):
            return _Rotate.apply(self, positions, backward, q, k)
        return self._rotate(positions, q, k, False, backward)

    def _rotate(self, positions, q, k, inplace, backward):
        if tracing_state() is not None or dispatch_modes():
            refuse_tracing("Rotary")
        if positions.dtype != torch.int32:
            raise TypeError(f"positions must be int32, got {positions.dtype}")
        io = IO_TYPES.get(q.dtype)
        if io is None:
            raise TypeError(f"rows must be float32, float16 or bfloat16, got {q.dtype}")
        n = q.dim()
        if n != 3 and n != 4:
            raise ValueError("rows must be [tokens, heads, dim] or [batch, tokens, heads, dim], "
                             f"got {tuple(q.shape)}")
        shape = q.shape
        batch, tokens, dim = (shape[0] if n == 4 else 1), shape[-3], shape[-1]
        if positions.dim() == 1:
            ok, stride = positions.shape[0] == tokens, 0
        else:
            ok = n == 4 and positions.shape in ((batch, tokens), (1, tokens))
            stride = positions.stride(0) if ok and positions.shape[0] > 1 else 0
        if not ok:
            raise ValueError(f"positions of shape {tuple(positions.shape)} do not fit rows of "
                             f"shape {tuple(shape)}")
        if tokens > 1 and positions.stride(-1) != 1 or stride and stride < tokens:
            positions, stride = positions.contiguous(), tokens if stride else 0
        if q.device != self.device or positions.device != self.device:
            raise ValueError(f"tensors must be on {self.device}")
        args = []
        outs = []
        for x in (q, k):
            if x is None:
                outs.append(None)
                continue
            if x is k and (x.dtype != q.dtype or x.device != q.device or x.dim() != n or
                           x.shape[:-2] != shape[:-2] or x.shape[-1] != dim):
                raise ValueError(f"k {tuple(x.shape)} {x.dtype} does not go with q "
                                 f"{tuple(shape)} {q.dtype}")
            if x.numel() and x.stride(-1) != 1:
                if inplace:
                    raise ValueError("inplace needs rows whose values lie side by side")
                x = x.contiguous()
            y = x if inplace else torch.empty_like(x)
            if y is not x and y.numel() and y.stride(-1) != 1:
                y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            outs.append(y)
            size = x.element_size()
            s, t = x.stride(), y.stride()
            args += (x.data_ptr(), y.data_ptr(), x.shape[-2], s[-2] * size, s[-3] * size,
                     s[0] * size if n == 4 else 0, t[-2] * size, t[-3] * size,
                     t[0] * size if n == 4 else 0)
        if q.numel() == 0 or k is not None and k.numel() == 0:
            if q.numel() or k is not None and k.numel():
                raise ValueError("q and k must both have heads")
            return tuple(outs)
        self._handle.rotate(positions.data_ptr(), stride, batch, tokens, dim, io, backward,
                            stream_of(self.device), *args)
        if inplace:  # a graph that saved them sees that they changed, as torch's own writes do
            increment_version([x for x in (q, k) if x is not None])
        return tuple(outs)


def _differentiated(q, k) -> bool:
    """Whether a call on q and k (or None) is to be differentiated, backward or forward."""
    if (q.requires_grad or k is not None and k.requires_grad) and torch.is_grad_enabled():
        return True
    return forward_ad._current_level >= 0 and any(
        x is not None and forward_ad.unpack_dual(x).tangent is not None for x in (q, k))


class _Rotate(torch.autograd.Function):
    """The rotation.  It is linear: the gradient is the transposed rotation of the outputs'
    gradients, the tangents of the outputs are the rotated tangents (both themselves
    differentiable)."""

    @staticmethod
    def forward(ctx, rotary, positions, backward, q, k):
        ctx.rotary, ctx.backward_ = rotary, backward
        ctx.shapes = q.shape, None if k is None else k.shape
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.set_materialize_grads(False)
        out = rotary._rotate(positions, q, k, False, backward)
        needs = ctx.needs_input_grad
        if not (needs[3] and needs[4]) and forward_ad._current_level < 0:
            ctx.mark_non_differentiable(*(y for y, need in zip(out, needs[3:])
                                          if y is not None and not need))
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        _, _, _, needs_q, needs_k = ctx.needs_input_grad
        return None, None, None, *_Rotate._each(ctx, dq if needs_q else None,
                                                dk if needs_k else None, not ctx.backward_)

    @staticmethod
    def jvp(ctx, _rotary, _positions, _backward, tq, tk):
        dtype = (tk if tq is None else tq).dtype
        zeros = (t if t is not None or shape is None else
                 torch.zeros(shape, dtype=dtype, device=ctx.rotary.device)
                 for t, shape in zip((tq, tk), ctx.shapes))  # an output's tangent may not be None
        return _Rotate._each(ctx, *zeros, ctx.backward_)

    @staticmethod
    def _each(ctx, a, b, backward):
        (positions,) = ctx.saved_tensors
        if a is not None:
            return ctx.rotary._turn(positions, a, b, backward)
        if b is not None:
            return None, ctx.rotary._turn(positions, b, None, backward)[0]
        return None, None
