"""The vocabulary's end of the model: the output projection with its cross entropy, and the verification of
drafted tokens.

The reference keeps lm_head out of FP8 (src/kernels.py:863-867) and trains on
cross_entropy(lm_head(x), targets) for the main and the MTP heads (src/train.py:355-372), which
writes the logits [n_tokens, vocabulary], their log-softmax and its gradient.
``linear_cross_entropy`` computes loss and gradients by pieces of the vocabulary on bf16, fp16 or
fp32 matrix units (csrc/lm_head.hip); only those of few rows of a wide model, fewer bytes than the
weight, are ever kept.

The reference trains heads that predict further tokens (MTP, src/layers.py:215-241).  ``verify_drafts`` is the step
that uses them: drafted tokens are kept or replaced so that the result is distributed as the target's
(csrc/verify.hip).
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call_on, dtype_code, ptr, stream_of
from .kernels import _cdiv, _plain_eager, _refuse_tangents, _require, _run, custom_op

__all__ = ["linear_cross_entropy", "verify_drafts"]

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_MODES = {"none": 0, "sum": 1, "mean": 2}
_DIRECT_ROWS = 128  # up to which fp32 is multiplied as it is (csrc/lm_head.hip kDirectRows)
_KEEP_ROWS = 128    # up to which the logits may be kept for the backward
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """cross_entropy(x @ weight.T, target) without the logits: x [..., D], weight [V, D] of the same
    dtype (bf16, fp16 or fp32), target [...] integers.  Returns fp32: the mean over the rows whose
    target is not ignore_index (NaN without one, as torch's), their sum, or with reduction "none"
    each row's loss (0 for an ignored one).  A target outside [0, V) gives NaN, in the gradients too.

    Differentiable in x and weight (once), gradients in their dtype.  Products are summed in fp32;
    the gradient of the logits enters the two gradient products rounded to the inputs' dtype, but for the
    targets' entries: what rounding takes off them is added back.
    fp32 inputs are multiplied as three bf16 parts each, to the accuracy of fp32 products (up to 128
    rows as they are, 32 products to a sum).
    Results do not vary from call to call.  The backward recomputes the logits piece by piece (those of
    up to 128 rows are kept where they are at most half the weight's bytes): beside the inputs it keeps
    one copy of the rows that count (fp32 of more than 128 rows: 1.5 times their size, and the weight's;
    a weight whose width is no multiple of 64: a padded copy) and a few words a row, and works in up to
    about 1 GiB for a piece of the logits' gradient plus fp32 sums of x's."""
    _require(x.is_cuda and weight.is_cuda and target.is_cuda, "Inputs must be on CUDA")
    _require(x.device == weight.device == target.device, "Inputs must be on one device")
    _require(weight.ndim == 2 and x.ndim >= 1 and x.shape[-1] == weight.shape[1], "x must be [..., D] and weight [V, D]")
    _require(target.shape == x.shape[:-1], "target must have x's shape without its last dimension")
    _require(x.dtype in _DTYPES and x.dtype == weight.dtype,
             "x and weight must share one dtype of bf16, fp16 and fp32 (cast one of them)")
    _require(not target.dtype.is_floating_point and not target.dtype.is_complex and target.dtype != torch.bool,
             "target must hold integers")
    _require(weight.shape[0] >= 1 and weight.shape[1] >= 1, "weight must not be empty")
    _require(reduction in _MODES, "reduction must be 'mean', 'sum' or 'none'")
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    y = target if target.ndim == 1 else target.reshape(-1)
    if y.dtype != torch.int64:
        y = y.to(torch.int64)
    mode = _MODES[reduction]
    _refuse_tangents(x2, weight)
    # (a layer's own Parameter is a plain tensor to the autograd Function)
    if _plain_eager(y) and type(x2) in _PLAIN and type(weight) in _PLAIN:
        if torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad):
            loss = _LinearCE.apply(x2, weight, y, int(ignore_index), mode)
        else:
            loss = _launch_forward(x2, weight, y, int(ignore_index), mode, False)[0]
    else:
        loss = _forward_op(x2, weight, y, int(ignore_index), mode)[0]
    return loss.view(target.shape) if mode == 0 and target.ndim != 1 else loss


def _keeps(T, D, dtype):
    """Whether the backward reads logits that the forward kept: where writing and reading them, 8 T bytes a
    column, moves no more than reading the weight again (131072 columns, bf16, forward and gradients: 128 x 128
    169 us kept and 152 formed again, 128 x 512 188 and 188, 128 x 1024 334 and 351, 16 x 512 143 and 156; fp32 gains
    up to there and loses 4% at most beyond: 128 x 128 252 and 261, 128 x 1024 908 and 1129)."""
    return T <= _KEEP_ROWS and 8 * T <= D * dtype.itemsize


def _layout(T, D, V, dtype):
    """Bytes of the state that the forward leaves: its rows that count, the weight's copy, integers
    and floats (csrc/lm_head.hip), for few rows the logits, each from a multiple of 256 on.  Operands are padded to whole K
    steps of 64; fp32 ones are three bf16 planes (for few rows as they are); a weight in one plane
    whose width needs no padding is not copied.  Returns (offsets of the five, total, whether the weight is copied)."""
    Dp = _cdiv(D, 64) * 64
    planes = 3 if dtype == torch.float32 and T > _DIRECT_ROWS else 1
    es = 4 if dtype == torch.float32 and T <= _DIRECT_ROWS else 2
    copied = planes == 3 or Dp != D
    offsets, at = [], 0
    for n in (planes * T * Dp * es, planes * V * Dp * es if copied else 0, 4 * (4 + 3 * T), 12 * T,
              4 * T * _cdiv(V, 64) * 64 if _keeps(T, D, dtype) else 0):
        offsets.append(at)
        at += _cdiv(n, 256) * 256
    return offsets, at, copied


@functools.lru_cache(maxsize=256)
def _sizes(T, D, V, dtype):
    """_layout's, and the workspaces' bytes of the forward and the backward."""
    ws = [_lib.load().cin_linear_ce_workspace(dtype_code(dtype), T, D, V, back) for back in (0, 1)]
    if min(ws) < 0:
        raise ValueError(f"linear_cross_entropy: {_lib.last_error()}")
    return (*_layout(T, D, V, dtype), *ws)


def _rows(t):
    """Rows of adjacent elements that do not overlap (_pitch apart)."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _pitch(t):
    """Elements between rows; a single row's stride says nothing."""
    return max(t.stride(0), t.shape[1])


def _weight_rows(w):
    """The weight as the products read it where its width needs no padding: rows on 16 bytes."""
    if w.stride(1) == 1 and w.stride(0) >= w.shape[1] and w.stride(0) * w.element_size() % 16 == 0 \
            and w.data_ptr() % 16 == 0 and w.stride(0) <= 1 << 20:
        return w
    return w.contiguous() if not w.is_contiguous() else w.clone(memory_format=torch.contiguous_format)


def _launch_forward(x, weight, target, ignore_index, mode, keep=True):
    """(loss, state for the backward; not keep: for none)"""
    (T, D), V = x.shape, weight.shape[0]
    x = _rows(x)
    (xc, wp, si, sf, sz), total, copied, ws, _ = _sizes(T, D, V, x.dtype)
    w = _rows(weight) if copied else _weight_rows(weight)
    target = target.contiguous()
    state = torch.empty(total if keep else sz, dtype=torch.uint8, device=x.device)
    work = torch.empty(ws, dtype=torch.uint8, device=x.device)
    rows = x.new_empty(T, dtype=torch.float32)
    loss = x.new_empty((), dtype=torch.float32) if mode else rows
    at = state.data_ptr()
    call_on(x, "cin_linear_ce_forward", x.data_ptr(), dtype_code(x), T, D, _pitch(x), w.data_ptr(), V, _pitch(w),
            target.data_ptr(), ignore_index, mode == 2, at + xc, at + wp if copied else 0, at + si, at + sf,
            rows.data_ptr(), loss.data_ptr() if mode else 0, work.data_ptr(), ws, at + sz if keep and _keeps(T, D, x.dtype) else 0,
            stream_of(x))
    return loss, state


def _launch_backward(grad, state, weight, T, mode, need_x, need_w):
    """(dx, dw), None where not needed."""
    V, D = weight.shape
    dtype = weight.dtype
    dx = weight.new_empty((T, D)) if need_x else None
    if T == 0:
        return dx, weight.new_zeros((V, D)) if need_w else None
    dw = weight.new_empty((V, D)) if need_w else None
    (xc, wp, si, sf, sz), _, copied, _, ws = _sizes(T, D, V, dtype)
    at = state.data_ptr()
    if copied:
        w, ldw = at + wp, _cdiv(D, 64) * 64
    else:
        weight = _weight_rows(weight)
        w, ldw = weight.data_ptr(), _pitch(weight)
    work = torch.empty(ws, dtype=torch.uint8, device=weight.device)
    call_on(weight, "cin_linear_ce_backward", at + xc, dtype_code(dtype), T, D, w, V, ldw, at + si, at + sf, grad.data_ptr(),
            0 if mode else grad.stride(0), mode == 2, ptr(dx), ptr(dw), work.data_ptr(), ws, at + sz if _keeps(T, D, dtype) else 0, stream_of(weight))
    return dx, dw


class _LinearCE(torch.autograd.Function):
    """linear_cross_entropy in eager mode, its launches called directly."""

    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, mode):
        loss, state = _launch_forward(x, weight, target, ignore_index, mode)
        ctx.save_for_backward(state, weight)
        ctx.options = x.shape[0], mode
        return loss

    @staticmethod
    def backward(ctx, grad):
        # (the wrapper costs 4 us of host time a call; only a graph of the gradient needs it)
        f = _gradients if not torch.is_grad_enabled() else once_differentiable(_gradients)
        return f(ctx, grad)


def _gradients(ctx, grad):
    _refuse_tangents(grad)
    dx, dw = _launch_backward(grad, *ctx.saved_tensors, *ctx.options, *ctx.needs_input_grad[:2])
    return dx, dw, None, None, None


@custom_op("linear_ce_forward", "(Tensor x, Tensor weight, Tensor target, int ignore_index, int mode) -> (Tensor, Tensor)")
def _forward_op(x, weight, target, ignore_index, mode):
    return _launch_forward(x, weight, target, ignore_index, mode)


@_forward_op.register_fake
def _(x, weight, target, ignore_index, mode):
    (T, D), V = x.shape, weight.shape[0]
    return (x.new_empty(() if mode else (T,), dtype=torch.float32),
            x.new_empty((_layout(T, D, V, x.dtype)[1],), dtype=torch.uint8))


@custom_op("linear_ce_backward", "(Tensor grad, Tensor state, Tensor weight, int T, int mode, bool need_x, bool need_w) -> "
           "(Tensor, Tensor)")
def _backward_op(grad, state, weight, T, mode, need_x, need_w):
    # a gradient not asked for comes back as an empty placeholder
    dx, dw = _launch_backward(grad, state, weight, T, mode, need_x, need_w)
    return dx if need_x else weight.new_empty((0,)), dw if need_w else weight.new_empty((0,))


@_backward_op.register_fake
def _(grad, state, weight, T, mode, need_x, need_w):
    return (weight.new_empty((T, weight.shape[1]) if need_x else (0,)),
            weight.new_empty(weight.shape if need_w else (0,)))


def _setup(ctx, inputs, output):
    x, weight, _target, _ignore, mode = inputs
    _loss, state = output
    ctx.mark_non_differentiable(state)
    ctx.save_for_backward(state, weight)
    ctx.options = x.shape[0], mode


def _backward(ctx, grad, _state):
    need_x, need_w = ctx.needs_input_grad[:2]
    _refuse_tangents(grad, *ctx.saved_tensors)
    dx, dw = _backward_op(grad, *ctx.saved_tensors, *ctx.options, need_x, need_w)
    return dx if need_x else None, dw if need_w else None, None, None, None


_forward_op.register_autograd(_backward, setup_context=_setup)


# ---------------------------------------------------------------------------
# Drafted tokens
# ---------------------------------------------------------------------------
MAX_DRAFTS = 63


def verify_drafts(draft_tokens: torch.Tensor, draft_probs: torch.Tensor | None, target_probs: torch.Tensor,
                  uniforms: torch.Tensor, n_drafts: torch.Tensor | None = None):
    """Drafted tokens against the target's probabilities, from given random numbers: (tokens int64
    [B, K + 1], accepted int64 [B]), distributed as tokens drawn from target_probs one by one.

    draft_tokens [B, K] integers, drawn from draft_probs [B, K, V]; target_probs [B, K + 1, V], the target's
    at each draft's position and after the last; bf16, fp16 or fp32, one type for both.  uniforms [B, K + 1] in
    [0, 1), fp32 or fp64.  n_drafts [B] integers: sequence b has that many drafts (default K, clamped to
    [0, K]); its row n_drafts[b] of target_probs is the one after the last.  draft_probs None: the drafts were certain of
    their tokens (a greedy draft).  K may be 0: a draw from target_probs[:, 0].

    Position i keeps its token x while uniforms[i] * draft_probs[i, x] < target_probs[i, x] (a token
    outside [0, V) is not kept).  With n = accepted tokens kept, tokens[n] is drawn by uniforms[K] from
    max(target_probs[n] - draft_probs[n], 0), or from target_probs[n] past the last draft or where nothing is left:
    the first token at which the running sum exceeds uniforms[K] times the whole.  Behind it tokens is -1; it is
    -1 itself where the sum is not positive and finite.  Products, differences and sums are in 64 bits; rows need not
    sum to one.  No gradient."""
    dev = target_probs.device
    _require(target_probs.is_cuda and draft_tokens.device == dev and uniforms.device == dev
             and (draft_probs is None or draft_probs.device == dev) and (n_drafts is None or n_drafts.device == dev),
             "Inputs must be on one CUDA device")
    _require(draft_tokens.ndim == 2 and target_probs.ndim == 3, "draft_tokens must be [B, K] and target_probs [B, K + 1, V]")
    (B, K), V = draft_tokens.shape, target_probs.shape[2]
    _require(K <= MAX_DRAFTS, "at most 63 drafts")
    _require(target_probs.shape == (B, K + 1, V) and V >= 1, "target_probs must be [B, K + 1, V]")
    _require(target_probs.dtype in _DTYPES, "probabilities must be bf16, fp16 or fp32")
    _require(draft_probs is None or (draft_probs.shape == (B, K, V) and draft_probs.dtype == target_probs.dtype),
             "draft_probs must be [B, K, V] in target_probs' dtype")
    _require(uniforms.shape == (B, K + 1) and uniforms.dtype in (torch.float32, torch.float64),
             "uniforms must be [B, K + 1] in fp32 or fp64")
    draft_tokens = _integers(draft_tokens)
    if n_drafts is not None:
        _require(n_drafts.shape == (B,), "n_drafts must be [B]")
        n_drafts = _integers(n_drafts)
    return _run(_verify_op, draft_tokens, draft_probs, target_probs, uniforms, n_drafts)


def _integers(t):
    """int64, of integers."""
    if t.dtype == torch.int64:
        return t
    _require(not t.dtype.is_floating_point and not t.dtype.is_complex and t.dtype != torch.bool,
             "draft_tokens and n_drafts must hold integers")
    return t.to(torch.int64)


@functools.lru_cache(maxsize=256)
def _verify_workspace(B, K, V, device):
    with torch.cuda.device(device):  # (the device's CUs decide)
        n = _lib.load().cin_verify_drafts_workspace(B, K, V)
    if n < 0:
        raise ValueError(f"verify_drafts: {_lib.last_error()}")
    return n


def _channels(t):
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@custom_op("verify_drafts", "(Tensor tokens, Tensor? draft, Tensor target, Tensor uniforms, Tensor? counts) -> (Tensor, Tensor)")
def _verify_op(tokens, draft, target, uniforms, counts):
    draft, target = _channels(draft), _channels(target)
    (B, K), V = tokens.shape, target.shape[2]
    out = tokens.new_empty((B, K + 1))
    accepted = tokens.new_empty((B,))
    ws = _verify_workspace(B, K, V, target.device)
    work = torch.empty(ws, dtype=torch.uint8, device=target.device)
    q = (0, 0, 0) if draft is None else (draft.data_ptr(), draft.stride(0), draft.stride(1))
    call_on(target, "cin_verify_drafts", tokens.data_ptr(), tokens.stride(0), tokens.stride(1), *q, target.data_ptr(),
            target.stride(0), target.stride(1), dtype_code(target), B, K, V, uniforms.data_ptr(),
            uniforms.dtype == torch.float64, uniforms.stride(0), uniforms.stride(1), ptr(counts),
            0 if counts is None else counts.stride(0), out.data_ptr(), accepted.data_ptr(), work.data_ptr(), ws, stream_of(target))
    return out, accepted


@_verify_op.register_fake
def _(tokens, draft, target, uniforms, counts):
    return tokens.new_empty((tokens.shape[0], tokens.shape[1] + 1)), tokens.new_empty((tokens.shape[0],))
