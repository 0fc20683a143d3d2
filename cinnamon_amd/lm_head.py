"""The output projection and the softmax cross entropy over a large vocabulary in one operator.

The reference keeps lm_head out of FP8 (src/kernels.py:863-867) and trains on
cross_entropy(lm_head(x), targets) for the main and the MTP heads (src/train.py:355-372), which
writes the logits [n_tokens, vocabulary], their log-softmax and its gradient.
``linear_cross_entropy`` computes loss and gradients by pieces of the vocabulary on bf16, fp16 or
fp32 matrix units (csrc/lm_head.hip) without ever keeping the logits.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import call_on, dtype_code, ptr, stream_of
from .kernels import _cdiv, _plain_eager, _require, custom_op

__all__ = ["linear_cross_entropy"]

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """cross_entropy(x @ weight.T, target) without the logits: x [..., D], weight [V, D] of the same
    dtype (bf16, fp16 or fp32), target [...] integers.  Returns fp32: the mean over the rows whose
    target is not ignore_index (NaN without one, as torch's), their sum, or with reduction "none"
    each row's loss (0 for an ignored one).  A target outside [0, V) gives NaN, in the gradients too.

    Differentiable in x and weight (once), gradients in their dtype.  Products are summed in fp32;
    the gradient of the logits enters the two gradient products rounded to the inputs' dtype.
    fp32 inputs are multiplied as three bf16 parts each, to the accuracy of fp32 products.
    Results do not vary from call to call.  The backward recomputes the logits piece by piece:
    beside the inputs it keeps one copy of the rows that count (fp32: 1.5 times their size, and the
    weight's; a weight whose width is no multiple of 64: a padded copy) and a few words a row, and
    works in up to about 1 GiB for a piece of the logits' gradient plus fp32 sums of x's."""
    _require(x.is_cuda and weight.is_cuda and target.is_cuda, "Inputs must be on CUDA")
    _require(x.device == weight.device == target.device, "Inputs must be on one device")
    _require(weight.ndim == 2 and x.ndim >= 1 and x.shape[-1] == weight.shape[1], "x must be [..., D] and weight [V, D]")
    _require(target.shape == x.shape[:-1], "target must have x's shape without its last dimension")
    _require(x.dtype in _DTYPES and x.dtype == weight.dtype,
             "x and weight must share one dtype of bf16, fp16 and fp32 (cast one of them)")
    _require(not target.dtype.is_floating_point and not target.dtype.is_complex and target.dtype != torch.bool,
             "target must hold integers")
    _require(weight.shape[0] >= 1 and weight.shape[1] >= 1, "weight must not be empty")
    _require(reduction in ("mean", "sum", "none"), "reduction must be 'mean', 'sum' or 'none'")
    x2 = x.reshape(-1, x.shape[-1])
    y = target.reshape(-1).to(torch.int64)
    mode = {"none": 0, "sum": 1, "mean": 2}[reduction]
    if _plain_eager(x2, weight, y):
        if torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad):
            loss = _LinearCE.apply(x2, weight, y, int(ignore_index), mode)
        else:
            loss = _launch_forward(x2, weight, y, int(ignore_index), mode)[0]
    else:
        loss = _forward_op(x2, weight, y, int(ignore_index), mode)[0]
    return loss.view(target.shape) if mode == 0 else loss


def _padded(D):
    """D rounded up to whole K steps of the products."""
    return _cdiv(D, 64) * 64


def _operand_shapes(x, V):
    """Shapes of the compacted rows and of the weight's copy, and their dtype: fp32 operands are three
    bf16 planes (csrc/lm_head.hip), others the rows padded to whole K steps; no copy of a 16-bit
    weight whose width needs no padding."""
    T, D = x.shape
    Dp = _padded(D)
    if x.dtype == torch.float32:
        return (3 * T, Dp), (3 * V, Dp), torch.bfloat16
    return (T, Dp), (V if Dp != D else 0, Dp), x.dtype


def _rows(t):
    """Rows of adjacent elements that do not overlap."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _weight_rows(w):
    """The weight as the products read it where its width needs no padding: rows on 16 bytes."""
    if w.stride(1) == 1 and w.stride(0) >= w.shape[1] and w.stride(0) * w.element_size() % 16 == 0 \
            and w.data_ptr() % 16 == 0 and w.stride(0) <= 1 << 20:
        return w
    return w.contiguous() if not w.is_contiguous() else w.clone()


def _workspace(name, backward, T, D, V, dtype, device):
    n = _lib.load().cin_linear_ce_workspace(dtype_code(dtype), T, D, V, backward)
    if n < 0:
        raise ValueError(f"{name}: {_lib.last_error()}")
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def _launch_forward(x, weight, target, ignore_index, mode):
    """(loss, compacted rows, padded weight or empty, int state, float state)"""
    (T, D), V = x.shape, weight.shape[0]
    dev = x.device
    x = _rows(x)
    xc, wp, dtype = _operand_shapes(x, V)
    pad = wp[0] > 0
    w = _rows(weight) if pad else _weight_rows(weight)
    target = target.contiguous()
    xc = torch.empty(xc, dtype=dtype, device=dev)
    wp = torch.empty(wp, dtype=dtype, device=dev)
    si = torch.empty(4 + 3 * T, dtype=torch.int32, device=dev)
    sf = torch.empty(2 * T, dtype=torch.float32, device=dev)
    rows = torch.empty(T, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev) if mode else rows
    ws = _workspace("linear_cross_entropy", 0, T, D, V, x.dtype, dev)
    call_on(x, "cin_linear_ce_forward", ptr(x), dtype_code(x), T, D, x.stride(0), ptr(w), V, w.stride(0), ptr(target),
            ignore_index, int(mode == 2), ptr(xc), ptr(wp) if pad else 0, ptr(si), ptr(sf), ptr(rows),
            ptr(loss) if mode else 0, ptr(ws), ws.numel(), stream_of(x))
    return loss, xc, wp, si, sf


def _launch_backward(grad, xc, weight, si, sf, D, dtype, mode, need_x, need_w):
    """(dx, dw) of dtype, None where not needed; weight: its copy where there is one."""
    T, V = sf.shape[0] // 2, weight.shape[0] // (3 if dtype == torch.float32 else 1)
    dev = xc.device
    dx = torch.empty((T, D), dtype=dtype, device=dev) if need_x else None
    if T == 0:
        return dx, torch.zeros((V, D), dtype=dtype, device=dev) if need_w else None
    dw = torch.empty((V, D), dtype=dtype, device=dev) if need_w else None
    w = _weight_rows(weight)
    ws = _workspace("linear_cross_entropy", 1, T, D, V, dtype, dev)
    call_on(xc, "cin_linear_ce_backward", ptr(xc), dtype_code(dtype), T, D, ptr(w), V, w.stride(0), ptr(si), ptr(sf),
            ptr(grad), 0 if mode else grad.stride(0), int(mode == 2), ptr(dx), ptr(dw), ptr(ws), ws.numel(),
            stream_of(xc))
    return dx, dw


class _LinearCE(torch.autograd.Function):
    """linear_cross_entropy in eager mode, its launches called directly."""

    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, mode):
        loss, xc, wp, si, sf = _launch_forward(x, weight, target, ignore_index, mode)
        ctx.save_for_backward(xc, wp if wp.shape[0] else weight, si, sf)
        ctx.options = x.shape[1], x.dtype, mode
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        dx, dw = _launch_backward(grad, *ctx.saved_tensors, *ctx.options, *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None


@custom_op("linear_ce_forward", "(Tensor x, Tensor weight, Tensor target, int ignore_index, int mode) -> "
           "(Tensor, Tensor, Tensor, Tensor, Tensor)")
def _forward_op(x, weight, target, ignore_index, mode):
    return _launch_forward(x, weight, target, ignore_index, mode)


@_forward_op.register_fake
def _(x, weight, target, ignore_index, mode):
    T = x.shape[0]
    xc, wp, dtype = _operand_shapes(x, weight.shape[0])
    return (x.new_empty(() if mode else (T,), dtype=torch.float32), x.new_empty(xc, dtype=dtype),
            x.new_empty(wp, dtype=dtype), x.new_empty((4 + 3 * T,), dtype=torch.int32),
            x.new_empty((2 * T,), dtype=torch.float32))


@custom_op("linear_ce_backward", "(Tensor grad, Tensor xc, Tensor weight, Tensor si, Tensor sf, int D, ScalarType dtype, "
           "int mode) -> (Tensor, Tensor)")
def _backward_op(grad, xc, weight, si, sf, D, dtype, mode):
    return _launch_backward(grad, xc, weight, si, sf, D, dtype, mode, True, True)


@_backward_op.register_fake
def _(grad, xc, weight, si, sf, D, dtype, mode):
    V = weight.shape[0] // (3 if dtype == torch.float32 else 1)
    return xc.new_empty((sf.shape[0] // 2, D), dtype=dtype), xc.new_empty((V, D), dtype=dtype)


def _setup(ctx, inputs, output):
    x, weight, _target, _ignore, mode = inputs
    loss, xc, wp, si, sf = output
    ctx.mark_non_differentiable(xc, wp, si, sf)
    copied = x.dtype == torch.float32 or _padded(x.shape[1]) != x.shape[1]
    ctx.save_for_backward(xc, wp if copied else weight, si, sf)
    ctx.options = x.shape[1], x.dtype, mode


def _backward(ctx, grad, *_):
    dx, dw = _backward_op(grad, *ctx.saved_tensors, *ctx.options)
    return dx, dw, None, None, None


_forward_op.register_autograd(_backward, setup_context=_setup)
