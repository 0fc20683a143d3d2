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
from ._lib import call_on, dtype_code, ptr, stream_of
from .kernels import _plain_eager, _require, custom_op

__all__ = ["block_norm", "rms_norm"]

MAX_WIDTH = 16384
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_NO_GATE, _CHANNEL, _ROW, _ELEMENT = range(4)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (weight [D], default ones): x [..., D]
    in bf16, fp16 or fp32, at most 16384 wide; squares and sums in fp32, the result rounded once to x's
    dtype.  Differentiable (once) in x and weight."""
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
    Differentiable (once) in every tensor, gradients in their dtype, bit-identical from call to call.  The backward
    keeps the inputs and two words a row, forms the sum again, and works in up to 16 D bytes a workgroup."""
    _require(residual is not None, "residual must be a tensor (rms_norm takes none)")
    scale, value = (residual_scale, 1.0) if torch.is_tensor(residual_scale) else \
        (None, 1.0 if residual_scale is None else float(residual_scale))
    _check(y, residual, weight, post_weight, gate, scale)
    return _call(y, residual, weight, post_weight, gate, scale, value, eps)[:2]


def _check(y, residual, weight, post_weight, gate, scale):
    _require(y.is_cuda, "Input must be on CUDA")
    _require(y.ndim >= 1 and 1 <= y.shape[-1] <= MAX_WIDTH, f"the last dimension must be in [1, {MAX_WIDTH}]")
    _require(y.dtype in _DTYPES, "y must be bf16, fp16 or fp32")
    D, dev = y.shape[-1], y.device
    if residual is not None:
        _require(residual.shape == y.shape and residual.device == dev, "residual must have y's shape and device")
        _require(residual.dtype == y.dtype or residual.dtype == torch.float32, "residual must have y's dtype or fp32")
    for name, t in (("weight", weight), ("post_weight", post_weight)):
        if t is not None:
            _require(t.shape == (D,) and t.device == dev and t.dtype in _DTYPES,
                     f"{name} must be [D] on y's device, in bf16, fp16 or fp32")
    if gate is not None:
        kind = _gate_kind(gate, y)
        _require(kind != _NO_GATE and gate.device == dev and gate.dtype in _DTYPES,
                 "gate must be [D], [..., 1] or of y's shape, on y's device")
        _require(kind != _ELEMENT or gate.dtype == y.dtype, "a gate of y's shape must have y's dtype")
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
    args = (y, residual, weight, post_weight, gate, scale)
    tensors = [t for t in args if t is not None]
    if _plain_eager() and all(type(t) in _PLAIN for t in tensors):
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
            return _BlockNorm.apply(*args, value, float(eps))
        return _launch(*args, value, float(eps), False)
    n, x, stats = _norm_op(*args, value, float(eps))
    return n, x, stats


def _rows(t):
    """(t as rows of adjacent elements, elements between them)"""
    D = t.shape[-1]
    t2 = t if t.ndim == 2 else t.reshape(-1, D)
    if not t2.is_contiguous() and (t2.stride(1) != 1 or t2.stride(0) < D):
        t2 = t2.contiguous()
    return t2, max(t2.stride(0), D)


def _side(t):
    """(what holds the rows, the arguments of one tensor [.., D]: pointer, type, stride)"""
    if t is None:
        return None, (0, 0, 0)
    rows, ld = _rows(t)
    return rows, (rows.data_ptr(), dtype_code(rows), ld)


def _inputs(y, residual, weight, post_weight, gate, scale, value):
    """(what must live until the launch, the arguments both directions share)"""
    y2, ya = _side(y)
    r2, ra = _side(residual)
    if residual is None:
        ra = (0, ya[1], ya[2])
    w = None if weight is None else weight.contiguous()
    pw = None if post_weight is None else post_weight.contiguous()
    kind = _gate_kind(gate, y)
    ldg, g = 0, gate
    if kind == _ELEMENT:
        g, ldg = _rows(gate)
    elif kind == _ROW:
        g = gate.reshape(-1)
        ldg = g.stride(0)
        if ldg < 1:
            g, ldg = g.contiguous(), 1
    elif kind == _CHANNEL:
        g = gate.contiguous()
    s = None if scale is None else scale.contiguous()
    # (a scale of one value stays one where D is 1 too)
    skind = 0 if s is None else 1 if s.numel() == 1 else 2
    code = lambda t: 0 if t is None else dtype_code(t)  # noqa: E731
    return (y2, r2, w, pw, g, s), (*ya, *ra, y2.shape[0], y2.shape[1], ptr(w), code(w), ptr(pw), code(pw), ptr(g), code(g),
                                   kind, ldg, ptr(s), code(s), skind, value)


def _launch(y, residual, weight, post_weight, gate, scale, value, eps, train=True):
    """(normed, new residual or None, what the backward needs of the rows or None)"""
    keep, args = _inputs(y, residual, weight, post_weight, gate, scale, value)
    n = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    x = None if residual is None else torch.empty(y.shape, dtype=residual.dtype, device=y.device)
    stats = torch.empty(2 * args[6], dtype=torch.float32, device=y.device) if train else None
    call_on(y, "cin_block_norm", *args, eps, n.data_ptr(), ptr(x), ptr(stats), stream_of(y))
    return n, x, stats


@functools.lru_cache(maxsize=256)
def _workspace(T, D, device):
    with torch.cuda.device(device):  # (the device's CUs decide)
        return _lib.load().cin_block_norm_workspace(T, D)


def _launch_backward(gn, gx, y, residual, weight, post_weight, gate, scale, stats, value, needs):
    """Gradients of the six tensors, None where not needed."""
    keep, args = _inputs(y, residual, weight, post_weight, gate, scale, value)
    T, D = args[6:8]
    grads = [torch.empty(t.shape, dtype=t.dtype, device=y.device) if need and t is not None else None
             for t, need in zip((y, residual, weight, post_weight, gate, scale), needs)]
    if T == 0:  # sums over no rows
        return [g if g is None else g.zero_() for g in grads]
    gn2, gna = _side(gn)
    gx2, gxa = _side(gx)
    sums = any(g is not None for g in (grads[2], grads[3], grads[5])) or (grads[4] is not None and args[14] == _CHANNEL)
    ws = _workspace(T, D, y.device) if sums else 0
    work = torch.empty(ws, dtype=torch.uint8, device=y.device) if sums else None
    call_on(y, "cin_block_norm_backward", *args, stats.data_ptr(), gna[0], gna[2], gxa[0], gxa[2], *(ptr(g) for g in grads),
            ptr(work), ws, stream_of(y))
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
    return (*_launch_backward(gn, gx, *ctx.saved_tensors, ctx.value, ctx.needs_input_grad[:6]), None, None)


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
    needs = [bool(n) and t is not None for n, t in zip(ctx.needs_input_grad[:6], tensors)]
    grads = _norm_bwd_op(gn, gx if tensors[1] is not None else None, *tensors, stats, ctx.value, needs)
    return (*(g if need else None for g, need in zip(grads, needs)), None, None)


_norm_op.register_autograd(_backward, setup_context=_setup)
