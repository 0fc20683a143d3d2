"""The norms around a block, fused with its gate and the residual sum.

The reference norms with x * rsqrt(mean(x^2) + eps) * weight (src/norm.py:15-17) and adds each block's
output to the stream it read (src/layers.py:202).  ``block_norm`` does the end of one block and the
start of the next in one pass (csrc/norm.hip): the block's output, normed and gated where asked, added to
the scaled stream, and the sum's norm.  ``rms_norm`` is the norm alone, in front of the first block.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import _DTYPE_CODE, call_on, ptr, stream_of
from .kernels import _plain_eager, _refuse_tangents, _require, custom_op

__all__ = ["block_norm", "rms_norm"]

MAX_WIDTH = 16384
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_NO_GATE, _CHANNEL, _ROW, _ELEMENT = range(4)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (weight [D], default ones): x [..., D]
    in bf16, fp16 or fp32, at most 16384 wide; squares and sums in fp32, the result rounded once to x's
    dtype.  Differentiable (once, in reverse mode) in x and weight."""
    _check(x, None, weight, None, None, None)
    return _call(x, None, weight, None, None, None, 1.0, eps)[0]


def block_norm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               residual_scale: float | torch.Tensor | None = None, eps: float = 1e-6):
    """The end of a block and the norm in front of the next, with norm(v) = v / sqrt(mean(v^2) + eps):

      new_residual = residual_scale * residual + gate * u,  u = norm(y) * post_weight, or y without post_weight
      normed       = norm(new_residual) * weight

    y [..., D] is the block's output, residual the stream of the same shape in y's dtype or fp32 (bf16, fp16
    or fp32, D at most 16384).  weight, post_weight: [D].  gate: [D], [..., 1] or y's shape (this one in y's
    dtype).  residual_scale: a number, or a tensor of one value or [D].  The vectors may have any of the three types.
    Returns (normed in y's dtype, new_residual in residual's).

    Computed in fp32 and each output rounded once: the norm is that of the sum before its rounding.
    Differentiable (once, in reverse mode) in every tensor, gradients in their dtype, bit-identical from call to call.
    The backward keeps the inputs and two words a row, forms the sum again, and works in up to 12 D bytes a workgroup."""
    _require(residual is not None, "residual must be a tensor (rms_norm takes none)")
    if residual_scale is None:
        scale, value = None, 1.0
    elif isinstance(residual_scale, torch.Tensor):
        scale, value = residual_scale, 1.0
    else:
        scale, value = None, float(residual_scale)
    _check(y, residual, weight, post_weight, gate, scale)
    return _call(y, residual, weight, post_weight, gate, scale, value, eps)[:2]


def _check(y, residual, weight, post_weight, gate, scale):
    _require(y.is_cuda, "Input must be on CUDA")
    shape, dt, dev = y.shape, y.dtype, y.device
    _require(len(shape) >= 1 and 1 <= shape[-1] <= MAX_WIDTH, "the last dimension must be in [1, 16384]")
    _require(dt in _DTYPES, "y must be bf16, fp16 or fp32")
    D = shape[-1]
    if residual is not None:
        _require(residual.shape == shape and residual.device == dev, "residual must have y's shape and device")
        _require(residual.dtype == dt or residual.dtype == torch.float32, "residual must have y's dtype or fp32")
    for t in (weight, post_weight):
        if t is not None:
            _require(t.ndim == 1 and t.shape[0] == D and t.device == dev and t.dtype in _DTYPES,
                     "weight and post_weight must be [D] on y's device, in bf16, fp16 or fp32")
    if gate is not None:
        kind = _gate_kind(gate, y)
        _require(kind != _NO_GATE and gate.device == dev and gate.dtype in _DTYPES,
                 "gate must be [D], [..., 1] or of y's shape, on y's device")
        _require(kind != _ELEMENT or gate.dtype == dt, "a gate of y's shape must have y's dtype")
    if scale is not None:
        _require((scale.numel() == 1 or scale.shape == (D,)) and scale.device == dev and scale.dtype in _DTYPES,
                 "residual_scale must be a number, or one value or [D] on y's device")


def _gate_kind(gate, y):
    """[D] is a gate of channels, whatever else it could be."""
    if gate is None:
        return _NO_GATE
    if gate.ndim == 1 and gate.shape[0] == y.shape[-1]:
        return _CHANNEL
    if gate.shape == (*y.shape[:-1], 1):
        return _ROW
    return _ELEMENT if gate.shape == y.shape else _NO_GATE


def _call(y, residual, weight, post_weight, gate, scale, value, eps):
    tensors = [t for t in (y, residual, weight, post_weight, gate, scale) if t is not None]
    _refuse_tangents(*tensors)
    if _plain_eager() and all(type(t) in _PLAIN for t in tensors):
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
            return _BlockNorm.apply(y, residual, weight, post_weight, gate, scale, value, float(eps))
        return _launch(y, residual, weight, post_weight, gate, scale, value, float(eps), False)
    return _norm_op(y, residual, weight, post_weight, gate, scale, value, float(eps))


def _rows(t, D):
    """(what holds t's rows of adjacent elements, their address, the elements between them)"""
    if t.is_contiguous():
        return t, t.data_ptr(), D
    t = t if t.ndim == 2 else t.reshape(-1, D)
    if t.stride(1) != 1 or t.stride(0) < D:
        t = t.contiguous()
    return t, t.data_ptr(), max(t.stride(0), D)


def _vector(t):
    """(what holds the vector, its address, its type's code)"""
    if t is None:
        return None, 0, 0
    t = t if t.is_contiguous() else t.contiguous()
    return t, t.data_ptr(), _DTYPE_CODE[t.dtype]


def _inputs(y, residual, weight, post_weight, gate, scale, value):
    """(what must live until the launch, the arguments both directions share)"""
    D = y.shape[-1]
    T = y.numel() // D
    code = _DTYPE_CODE[y.dtype]
    kind = _NO_GATE if gate is None else _gate_kind(gate, y)
    if kind == _NO_GATE:
        gp = gcode = ldg = 0
    else:
        gcode = _DTYPE_CODE[gate.dtype]
        if kind == _ELEMENT:
            gate, gp, ldg = _rows(gate, D)
        else:
            if kind == _ROW:
                gate = gate.reshape(-1)
            if kind == _CHANNEL or gate.stride(0) < 1:
                gate = gate.contiguous()
            gp, ldg = gate.data_ptr(), max(gate.stride(0), 1)  # (one expanded value stays as it is, with 0)
    y, yp, ldy = _rows(y, D)
    if residual is None:
        rp, rcode, ldr = 0, code, D
    else:
        rcode = _DTYPE_CODE[residual.dtype]
        residual, rp, ldr = _rows(residual, D)
    weight, wp, wcode = _vector(weight)
    post_weight, pp, pcode = _vector(post_weight)
    scale, sp, scode = _vector(scale)
    # (a scale of one value stays one where D is 1 too)
    skind = 0 if scale is None else 1 if scale.numel() == 1 else 2
    return (y, residual, weight, post_weight, gate, scale), (yp, code, ldy, rp, rcode, ldr, T, D, wp, wcode, pp, pcode, gp, gcode,
                                                             kind, ldg, sp, scode, skind, value)


_T, _KIND = 6, 14  # of the arguments


def _launch(y, residual, weight, post_weight, gate, scale, value, eps, train=True):
    """(normed, new residual or None, what the backward needs of the rows or None)"""
    held, args = _inputs(y, residual, weight, post_weight, gate, scale, value)
    n = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    x = None if residual is None else torch.empty(y.shape, dtype=residual.dtype, device=y.device)
    stats = torch.empty(2 * args[_T], dtype=torch.float32, device=y.device) if train else None
    call_on(n, "cin_block_norm", *args, eps, n.data_ptr(), ptr(x), ptr(stats), stream_of(n))
    return n, x, stats


@functools.lru_cache(maxsize=256)
def _workspace(T, D, device):
    with torch.cuda.device(device):  # (the device's CUs decide)
        return _lib.load().cin_block_norm_workspace(T, D)


def _launch_backward(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs):
    """Gradients of the six tensors, None where not needed."""
    held, args = _inputs(y, residual, weight, post_weight, gate, scale, value)
    T, D = args[_T], args[_T + 1]
    dev = y.device
    grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if need and t is not None else None
             for t, need in zip((y, residual, weight, post_weight, gate, scale), needs)]
    if T == 0:  # sums over no rows
        return [g if g is None else g.zero_() for g in grads]
    gn, gnp, ldgn = (None, 0, 0) if gn is None else _rows(gn, D)
    gx, gxp, ldgx = (None, 0, 0) if gx is None else _rows(gx, D)
    dy, dr, dw, dpw, dgate, dscale = grads
    ws, work = 0, None
    if dw is not None or dpw is not None or dscale is not None or (dgate is not None and args[_KIND] == _CHANNEL):
        ws = _workspace(T, D, y.get_device())
        work = torch.empty(ws, dtype=torch.uint8, device=dev)
    call_on(y, "cin_block_norm_backward", *args, stats.data_ptr(), gnp, ldgn, gxp, ldgx, ptr(dy), ptr(dr), ptr(dw), ptr(dpw),
            ptr(dgate), ptr(dscale), ptr(work), ws, stream_of(y))
    return grads


class _BlockNorm(torch.autograd.Function):
    """block_norm in eager mode, its launches called directly."""

    @staticmethod
    def forward(ctx, y, residual, weight, post_weight, gate, scale, value, eps):
        n, x, stats = _launch(y, residual, weight, post_weight, gate, scale, value, eps)
        ctx.save_for_backward(y, residual, weight, post_weight, gate, scale, stats)
        ctx.value = value
        ctx.set_materialize_grads(False)
        return n, x

    @staticmethod
    def backward(ctx, gn, gx):
        # (the wrapper costs 4 us of host time a call; only a graph of the gradient needs it)
        f = _gradients if not torch.is_grad_enabled() else once_differentiable(_gradients)
        return f(ctx, gn, gx)


def _gradients(ctx, gn, gx):
    if gn is None and gx is None:
        return (None,) * 8
    _refuse_tangents(gn, gx)
    return (*_launch_backward(gn, gx, *ctx.saved_tensors, ctx.value, ctx.needs_input_grad), None, None)


@custom_op("block_norm", "(Tensor y, Tensor? residual, Tensor? weight, Tensor? post_weight, Tensor? gate, Tensor? scale, "
           "float value, float eps) -> (Tensor, Tensor, Tensor)")
def _norm_op(y, residual, weight, post_weight, gate, scale, value, eps):
    # without a residual the second output is an empty placeholder
    n, x, stats = _launch(y, residual, weight, post_weight, gate, scale, value, eps)
    return n, x if x is not None else y.new_empty((0,)), stats


@_norm_op.register_fake
def _(y, residual, weight, post_weight, gate, scale, value, eps):
    rows = 1
    for n in y.shape[:-1]:
        rows = rows * n
    return (y.new_empty(y.shape), y.new_empty((0,)) if residual is None else residual.new_empty(y.shape),
            y.new_empty((2 * rows,), dtype=torch.float32))


@custom_op("block_norm_backward", "(Tensor? gn, Tensor? gx, Tensor y, Tensor? residual, Tensor? weight, Tensor? post_weight, "
           "Tensor? gate, Tensor? scale, Tensor stats, float value, bool[6] needs) -> (Tensor, Tensor, Tensor, Tensor, Tensor, "
           "Tensor)")
def _norm_bwd_op(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs):
    # a gradient not asked for comes back as an empty placeholder
    grads = _launch_backward(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs)
    return tuple(g if g is not None else y.new_empty((0,)) for g in grads)


@_norm_bwd_op.register_fake
def _(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs):
    return tuple(t.new_empty(t.shape) if need and t is not None else y.new_empty((0,))
                 for t, need in zip((y, residual, weight, post_weight, gate, scale), needs))


def _setup(ctx, inputs, output):
    *tensors, value, _eps = inputs
    stats = output[2]
    ctx.mark_non_differentiable(*((stats,) if tensors[1] is not None else output[1:]))
    ctx.save_for_backward(*tensors, stats)
    ctx.value = value


def _backward(ctx, gn, gx, _gstats):
    *tensors, stats = ctx.saved_tensors
    _refuse_tangents(gn, gx, *tensors)
    needs = [bool(n) and t is not None for n, t in zip(ctx.needs_input_grad[:6], tensors)]
    grads = _norm_bwd_op(gn, gx if tensors[1] is not None else None, *tensors, stats, ctx.value, needs)
    return (*(g if need else None for g, need in zip(grads, needs)), None, None)


_norm_op.register_autograd(_backward, setup_context=_setup)
