"""Rotary positions for queries and keys (reference src/attention.py:9-128).

``rotary_tables`` makes the cosines and sines of a context once, in 64 bits, with the
frequencies scaled for long contexts where asked; ``apply_rotary`` turns the channel pairs of
queries and keys in one launch (csrc/rotary.hip) and is differentiable in both.  It goes in
front of kernels.indexer_scores_fp8 and of attention.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from ._lib import call_on, dtype_code, ptr, stream_of
from .kernels import _plain_eager, _refuse_tangents, _require, custom_op

__all__ = ["rotary_tables", "apply_rotary"]

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def rotary_tables(rot: int, length: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                  original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                  attention_factor: float | None = None, device=None):
    """(cos, sin), fp32 [length, rot / 2] each: position p times frequency base^(-2i / rot), taken
    in 64 bits (an fp32 product is 0.03 rad off at position 10^6) and rounded once.

    scaling None, or for contexts ``factor`` times the original_length (default length / factor):
      "linear"  positions divided by factor;
      "ntk"     base raised to base * factor^(rot / (rot - 2)): the fastest frequency stays, the
                slowest is divided by factor;
      "yarn"    frequencies that turn more than beta_fast times in original_length stay, those
                that turn less than beta_slow times are divided by factor, a linear ramp over the
                index between; both tables times attention_factor, by default 0.1 ln(factor) + 1."""
    _require(rot >= 2 and rot % 2 == 0, "rot must be even and at least 2")
    _require(length >= 0, "length must not be negative")
    _require(scaling in (None, "linear", "ntk", "yarn"), "scaling must be None, 'linear', 'ntk' or 'yarn'")
    _require(base > 1 and factor >= 1, "base must be above 1 and factor at least 1")
    _require(scaling != "ntk" or rot > 2, "ntk scaling needs rot > 2")
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    freq = base ** (-2 * i / rot)
    scale = 1.0 if attention_factor is None else float(attention_factor)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        n = original_length if original_length is not None else length / factor
        _require(n > 0 and beta_fast > beta_slow > 0, "yarn scaling needs original_length > 0 and beta_fast > beta_slow > 0")

        def index_of(turns):  # the index whose frequency turns that often in n positions
            return rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(index_of(beta_fast)), 0)
        hi = min(math.ceil(index_of(beta_slow)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)  # 0: stays, 1: divided
        freq = freq * (1 - ramp) + freq / factor * ramp
        if attention_factor is None and factor > 1:
            scale = 0.1 * math.log(factor) + 1
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return (angle.cos() * scale).to(torch.float32), (angle.sin() * scale).to(torch.float32)


def apply_rotary(q: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, interleaved: bool = True, start: int = 0):
    """q [B, L, H, D] (or [B, L, D]: one head), and k [B, L, Hk, D] if given, with the pairs of
    channels [start, start + rot) turned by the angle of their position; the other channels are
    copied.  Returns q's result, or (q's, k's); new tensors in the inputs' dtype (bf16, fp16 or
    fp32), each value computed in fp32 and rounded once.

    cos, sin: fp32 [P, rot / 2] (rotary_tables), no gradient.  positions: integer [L] or [B, L];
    default 0 .. L - 1.  A token at a negative position is copied as it is (padding); one at P or
    beyond gives NaN in its rotated channels.  interleaved: pairs (2i, 2i + 1), else
    (i, i + rot / 2).  Any strides (x.transpose(1, 2) takes [B, H, L, D])."""
    _require(q.ndim in (3, 4) and (k is None or k.ndim in (3, 4)), "q and k must be [B, L, H, D] or [B, L, D]")
    for t in (q, k):
        if t is None:
            continue
        _require(t.is_cuda, "Input must be on CUDA")
        _require(t.dtype in _DTYPES, "q and k must be bf16, fp16 or fp32")
        _require(t.device == q.device and t.dtype == q.dtype, "q and k must share device and dtype")
        _require(t.shape[:2] == q.shape[:2] and t.shape[-1] == q.shape[-1], "q and k must share B, L and D")
    _require(cos.ndim == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32,
             "cos and sin must be fp32 [P, rot / 2]")
    _require(cos.device == q.device and sin.device == q.device, "cos and sin must be on q's device")
    _require(not (cos.requires_grad or sin.requires_grad) or not torch.is_grad_enabled(),
             "cos and sin carry no gradient: detach them")
    (P, half), L = cos.shape, q.shape[1]
    _require(half >= 1 and start >= 0 and start + 2 * half <= q.shape[-1],
             "the rotated channels [start, start + rot) must lie within the head")
    if positions is None:
        _require(L <= P, "more tokens than the tables hold positions")
    else:
        _require(positions.device == q.device and not positions.dtype.is_floating_point
                 and not positions.dtype.is_complex and positions.dtype != torch.bool,
                 "positions must be integers on q's device")
        _require(tuple(positions.shape) in ((L,), (q.shape[0], L)), "positions must be [L] or [B, L]")
        if positions.dtype != torch.int64:
            positions = positions.to(torch.int64)
    args = (q, k, cos, sin, positions, bool(interleaved), int(start))
    _refuse_tangents(*args)
    if _plain_eager(*args):
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            out = _Rotary.apply(*args)
        else:
            out = _launch(*args, False)
    else:
        out = _rotary_op(*args, False)
    return out[0] if k is None else out


def _rows(t):
    """t with adjacent channels and token and head strides that fit in 32 bits."""
    if t.is_contiguous() or (t.stride(-1) == 1 and max(t.stride()[1:-1]) < 1 << 31):
        return t
    return t.contiguous()


def _empty(x):
    """An output like x, its channels adjacent."""
    out = torch.empty_like(x)
    return out if out.stride(-1) == 1 else torch.empty_like(x, memory_format=torch.contiguous_format)


_NO_SIDE = (0,) * 9


def _side(t):
    """(output, the arguments of one tensor: both pointers, their batch, token and head strides,
    the heads)"""
    if t.is_contiguous():
        out = torch.empty_like(t)
        shape = t.shape
        H = shape[2] if len(shape) == 4 else 1
        D = shape[-1]
        l = H * D
        b = shape[1] * l
        return out, (t.data_ptr(), b, l, D, out.data_ptr(), b, l, D, H)
    t = _rows(t)
    out = _empty(t)

    def strides(x):
        return (x.stride(0), x.stride(1), x.stride(2) if x.ndim == 4 else 0)

    return out, (t.data_ptr(), *strides(t), out.data_ptr(), *strides(out), t.shape[2] if t.ndim == 4 else 1)


def _launch(q, k, cos, sin, positions, interleaved, start, inverse):
    """(q's result, k's); a tensor that is None gives None."""
    oq, sq = (None, _NO_SIDE) if q is None else _side(q)
    ok, sk = (None, _NO_SIDE) if k is None else _side(k)
    t = q if q is not None else k
    shape = t.shape
    cos, sin = cos.contiguous(), sin.contiguous()
    P, half = cos.shape
    spb, spl = (0, 0) if positions is None else (positions.stride(0) if positions.ndim == 2 else 0, positions.stride(-1))
    call_on(t, "cin_rotary", *sq, *sk, dtype_code(t), shape[0], shape[1], shape[-1], cos.data_ptr(), sin.data_ptr(), P,
            half, 2 * half, start, ptr(positions), spb, spl, interleaved, inverse, stream_of(t))
    return oq, ok


class _Rotary(torch.autograd.Function):
    """apply_rotary in eager mode: its gradient is the turn back by the same angles."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, start):
        ctx.save_for_backward(cos, sin, positions)
        ctx.options = interleaved, start
        ctx.set_materialize_grads(False)
        return _launch(q, k, cos, sin, positions, interleaved, start, False)

    @staticmethod
    def backward(ctx, gq, gk):
        # (the wrapper costs 4 us of host time a call; only a graph of the gradient needs it)
        f = _rotary_turn_back if not torch.is_grad_enabled() else once_differentiable(_rotary_turn_back)
        return f(ctx, gq, gk)


def _rotary_turn_back(ctx, gq, gk):
    need_q, need_k = ctx.needs_input_grad[:2]
    gq, gk = gq if need_q else None, gk if need_k else None
    if gq is None and gk is None:
        return (None,) * 7
    _refuse_tangents(gq, gk)
    return (*_launch(gq, gk, *ctx.saved_tensors, *ctx.options, True), None, None, None, None, None)


@custom_op("rotary", "(Tensor q, Tensor? k, Tensor cos, Tensor sin, Tensor? positions, bool interleaved, int start, "
           "bool inverse) -> (Tensor, Tensor)")
def _rotary_op(q, k, cos, sin, positions, interleaved, start, inverse):
    # without k the second output is an empty placeholder
    oq, ok = _launch(q, k, cos, sin, positions, interleaved, start, inverse)
    return oq, ok if ok is not None else q.new_empty((0,))


@_rotary_op.register_fake
def _(q, k, cos, sin, positions, interleaved, start, inverse):
    return _empty(_rows(q)), _empty(_rows(k)) if k is not None else q.new_empty((0,))


def _rotary_setup(ctx, inputs, output):
    _q, k, cos, sin, positions, interleaved, start, inverse = inputs
    ctx.save_for_backward(cos, sin, positions)
    ctx.options = interleaved, start, inverse
    ctx.with_k = k is not None


def _rotary_backward(ctx, gq, gk):
    cos, sin, positions = ctx.saved_tensors
    interleaved, start, inverse = ctx.options
    _refuse_tangents(gq, gk)
    dq, dk = _rotary_op(gq, gk if ctx.with_k else None, cos, sin, positions, interleaved, start, not inverse)
    return dq, dk if ctx.with_k else None, None, None, None, None, None, None


_rotary_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)
