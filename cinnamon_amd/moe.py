"""Device-side MoE dispatch and combine around the FP8 grouped experts.

Counterpart of the permute -> grouped experts -> unpermute block of the reference's
MoE.forward (src/layers.py:126-157):

  reference                                      here
  sigmoid, bias, top-k, renormalized weights     moe_gate: one launch, and one for the gradient
  expanded_idx.sort(), token_indices, bincount,  moe_route: stable counting sort on the
  cumsum, max_expert_tokens = .item()            device, int64 expert ranges, no host sync
  sorted_x = flat_x[token_indices] (bf16),       moe_gather_quantize: the 1x128 quantizer
  then the experts quantize it                   reads x rows through the permutation
  sorted_out * sorted_scores, scatter_add_       moe_combine: per-token sum in sorted order

``routed_experts`` chains those after moe_gate with layers.experts_forward/backward; its gradients reach
x, the expert weights and the routing scores.  ``moe_decode`` is the whole layer, router and shared expert
included, for the few tokens of a generation step (csrc/moe_decode.hip).  Every launch is a cinnamon_amd:: torch
operator (torch.compile traces through it).  The sort is stable, so within an expert the
rows keep token order (the reference's unstable sort may order them differently; each
row's result does not depend on its position, and the combine adds a token's terms in
sorted position order, the order of a sequential scatter_add_).
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib, layers
from ._lib import call, call_on, dtype_code, ptr, stream_of
from .kernels import _cdiv, _plain_eager, _refuse_tangents, _require, _run_detached, _scale_buf, custom_op

_ROUTE_CHUNK = 1024  # assignments per route workgroup (csrc/moe.hip kChunk)
MAX_EXPERTS = 4096
MAX_TOP_K = 16
MAX_GROUPS = 64
MAX_DECODE_TOKENS = 128
MAX_DECODE_EXPERTS = 1024

__all__ = ["moe_gate", "moe_route", "moe_gather_quantize", "moe_gather_sum", "moe_combine",
           "moe_combine_backward", "RoutedExpertsFunction", "routed_experts", "moe_decode"]


# ---------------------------------------------------------------------------
# The gate (reference src/layers.py:122-126)
# ---------------------------------------------------------------------------
_SCORES = {"sigmoid": 0, "softmax": 1}
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def moe_gate(logits: torch.Tensor, top_k: int, bias: torch.Tensor | None = None, score: str = "sigmoid",
             n_groups: int = 1, top_groups: int | None = None, group_top: int = 2, renormalize: bool = True,
             scale: float = 1.0, return_scores: bool = False):
    """The chosen experts of each token and their weights, from the router's logits [n_tokens, E]
    (bf16, fp16 or fp32): (top_idx int64 [n_tokens, top_k], top_scores fp32 [n_tokens, top_k]) for
    routed_experts, and with return_scores all scores fp32 [n_tokens, E] (for a balance loss).

      scores = sigmoid(logits) or softmax(logits); choice = scores + bias (fp32 [E], only chooses);
      with n_groups > 1, E / n_groups neighbouring experts form a group, a group counts by the sum of
      its group_top (1 or 2) largest choices, and only the best top_groups groups stay;
      top_idx: the top_k largest choices left, falling, ties to the lowest index; choices are
      compared in 64 bits; NaN counts as the greatest, as in torch.topk;
      top_scores = scale * scores[top_idx], divided by (their sum + 1e-9) with renormalize.

    Differentiable in logits, through top_scores and scores; no gradient reaches bias."""
    _require(logits.is_cuda, "Input must be on CUDA")
    _require(logits.ndim == 2, "logits must be [n_tokens, n_experts]")
    _require(logits.dtype in (torch.bfloat16, torch.float16, torch.float32), "logits must be bf16, fp16 or fp32")
    E = logits.shape[1]
    _require(1 <= E <= MAX_EXPERTS, f"n_experts must be in [1, {MAX_EXPERTS}]")
    _require(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _require(1 <= n_groups <= MAX_GROUPS and E % n_groups == 0, f"n_groups must divide n_experts and be in [1, {MAX_GROUPS}]")
    top_groups = n_groups if top_groups is None else top_groups
    _require(1 <= top_groups <= n_groups, "top_groups must be in [1, n_groups]")
    _require(group_top in (1, 2), "group_top must be 1 or 2")
    _require(1 <= top_k <= min(MAX_TOP_K, top_groups * (E // n_groups)),
             f"top_k must be in [1, {MAX_TOP_K}] and within the experts of the kept groups")
    if bias is not None:
        _require(bias.shape == (E,) and bias.device == logits.device, "bias must be [n_experts] on logits' device")
        _require(bias.dtype == torch.float32, "bias must be fp32")
        bias = bias.detach()
    options = (int(top_k), _SCORES[score], int(n_groups), int(top_groups), int(group_top), bool(renormalize),
               float(scale), bool(return_scores))
    _refuse_tangents(logits)
    if _plain_eager(logits, bias):
        if torch.is_grad_enabled() and logits.requires_grad:
            out = _MoeGate.apply(logits, bias, *options)
        else:
            out = _launch_gate(logits, bias, *options)
    else:
        out = _gate_op(logits, bias, *options)
    return out if return_scores else out[:2]


def _gate_rows(logits):
    return logits if logits.is_contiguous() or (logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1]) \
        else logits.contiguous()


def _launch_gate(logits, bias, top_k, score, n_groups, top_groups, group_top, renormalize, scale, return_scores):
    """(idx, weights, scores or None)"""
    lg = _gate_rows(logits)
    T, E = lg.shape
    idx = lg.new_empty((T, top_k), dtype=torch.int64)
    w = lg.new_empty((T, top_k), dtype=torch.float32)
    scores = lg.new_empty((T, E), dtype=torch.float32) if return_scores else None
    bias = None if bias is None else bias.contiguous()
    call_on(lg, "cin_moe_gate", lg.data_ptr(), dtype_code(lg), max(lg.stride(0), E), ptr(bias), T, E, top_k, score,
            n_groups, top_groups, group_top, renormalize, scale, idx.data_ptr(), w.data_ptr(), ptr(scores), stream_of(lg))
    return idx, w, scores


def _launch_gate_backward(logits, idx, gw, gs, score, renormalize, scale):
    """Gradient of the logits; gw or gs may be None."""
    lg = _gate_rows(logits)
    T, E = lg.shape
    out = lg.new_empty((T, E))
    gw = None if gw is None else gw.contiguous()
    gs = None if gs is None else gs.contiguous()
    call_on(lg, "cin_moe_gate_backward", ptr(lg), dtype_code(lg), max(lg.stride(0), E), T, E, idx.shape[1], score,
            renormalize, scale, idx.data_ptr(), ptr(gw), ptr(gs), out.data_ptr(), stream_of(lg))
    return out


class _MoeGate(torch.autograd.Function):
    """moe_gate in eager mode, its two launches called directly."""

    @staticmethod
    def forward(ctx, logits, bias, *options):
        idx, w, scores = _launch_gate(logits, bias, *options)
        ctx.save_for_backward(logits, idx)
        ctx.options = options
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(idx)
        return idx, w, scores

    @staticmethod
    def backward(ctx, *grads):
        # (the wrapper costs 4 us of host time a call; only a graph of the gradient needs it)
        f = _gate_gradient if not torch.is_grad_enabled() else once_differentiable(_gate_gradient)
        return f(ctx, *grads)


def _gate_gradient(ctx, _gidx, gw, gs):
    if gw is None and gs is None:
        return (None,) * 10
    _refuse_tangents(gw, gs)
    _k, score, _g, _tg, _gt, renormalize, scale, _rs = ctx.options
    return (_launch_gate_backward(*ctx.saved_tensors, gw, gs, score, renormalize, scale),) + (None,) * 9


@custom_op("moe_gate", "(Tensor logits, Tensor? bias, int top_k, int score, int n_groups, int top_groups, int group_top, "
           "bool renormalize, float scale, bool return_scores) -> (Tensor, Tensor, Tensor)")
def _gate_op(logits, bias, *options):
    # without return_scores the last output is an empty placeholder
    idx, w, scores = _launch_gate(logits, bias, *options)
    return idx, w, scores if scores is not None else logits.new_empty((0,), dtype=torch.float32)


@_gate_op.register_fake
def _(logits, bias, top_k, score, n_groups, top_groups, group_top, renormalize, scale, return_scores):
    T, E = logits.shape
    return (logits.new_empty((T, top_k), dtype=torch.int64), logits.new_empty((T, top_k), dtype=torch.float32),
            logits.new_empty((T, E) if return_scores else (0,), dtype=torch.float32))


@custom_op("moe_gate_backward", "(Tensor logits, Tensor idx, Tensor gw, Tensor? gs, int score, bool renormalize, "
           "float scale) -> Tensor")
def _gate_bwd_op(logits, idx, gw, gs, score, renormalize, scale):
    return _launch_gate_backward(logits, idx, gw, gs, score, renormalize, scale)


@_gate_bwd_op.register_fake
def _(logits, idx, gw, gs, score, renormalize, scale):
    return logits.new_empty(logits.shape)


def _gate_setup(ctx, inputs, output):
    logits, _bias, _k, score, _g, _tg, _gt, renormalize, scale, return_scores = inputs
    idx, _w, scores = output
    ctx.save_for_backward(logits, idx)
    ctx.mark_non_differentiable(*((idx,) if return_scores else (idx, scores)))
    ctx.options = score, renormalize, scale, return_scores


def _gate_backward(ctx, _gidx, gw, gs):
    logits, idx = ctx.saved_tensors
    _refuse_tangents(gw, gs, logits)
    score, renormalize, scale, return_scores = ctx.options
    dz = _gate_bwd_op(logits, idx, gw, gs if return_scores else None, score, renormalize, scale)
    return (dz,) + (None,) * 9


_gate_op.register_autograd(_gate_backward, setup_context=_gate_setup)


# ---------------------------------------------------------------------------
# Routing (reference src/layers.py:133-148)
# ---------------------------------------------------------------------------
def moe_route(top_idx: torch.Tensor, n_experts: int):
    """Stable sort of the flattened top-k ids on the device.

    top_idx [T, k] integer expert ids -> (perm int64 [T*k], inv int32 [T*k], counts,
    starts, ends int64 [E]).  perm[r] = t*k + j of the assignment at sorted position r
    (the reference's sort_order; token_indices = perm // k), inv its inverse.  Ids
    outside [0, E) are dropped: inv -1, and perm -1 at the positions past the kept ones.
    """
    _require(top_idx.is_cuda, "Input must be on CUDA")
    _require(top_idx.ndim == 2, "top_idx must be [n_tokens, top_k]")
    _require(1 <= n_experts <= MAX_EXPERTS, f"n_experts must be in [1, {MAX_EXPERTS}]")
    return _run_detached(_route_op, top_idx.to(torch.int64).contiguous(), int(n_experts))


@custom_op("moe_route", "(Tensor idx, int n_experts) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
def _route_op(idx, n_experts):
    T, k = idx.shape
    A = T * k
    dev = idx.device
    perm = torch.empty(A, dtype=torch.int64, device=dev)
    inv = torch.empty(A, dtype=torch.int32, device=dev)
    counts = torch.empty(n_experts, dtype=torch.int64, device=dev)
    starts = torch.empty(n_experts, dtype=torch.int64, device=dev)
    ends = torch.empty(n_experts, dtype=torch.int64, device=dev)
    nws = max(1, 2 * _cdiv(A, _ROUTE_CHUNK) * n_experts)
    ws = torch.empty(nws, dtype=torch.int32, device=dev)
    call("cin_moe_route", ptr(idx), T, k, n_experts, ptr(perm), ptr(inv), ptr(counts), ptr(starts),
         ptr(ends), ptr(ws), nws, stream_of(idx))
    return perm, inv, counts, starts, ends


@_route_op.register_fake
def _(idx, n_experts):
    A = idx.shape[0] * idx.shape[1]
    i64 = torch.int64
    return (idx.new_empty((A,), dtype=i64), idx.new_empty((A,), dtype=torch.int32),
            idx.new_empty((n_experts,), dtype=i64), idx.new_empty((n_experts,), dtype=i64),
            idx.new_empty((n_experts,), dtype=i64))


# ---------------------------------------------------------------------------
# Gather fused into the 1x128 quantization, and its backward (reference :139-141)
# ---------------------------------------------------------------------------
def moe_gather_quantize(x: torch.Tensor, perm: torch.Tensor, top_k: int, round_scale: bool = False,
                        inv: torch.Tensor | None = None, col_scales: bool = False):
    """quantize_fp8_rowwise(x[perm // top_k]) bit for bit, without the gathered rows:
    (codes float8_e4m3fn [A, D], scales fp32 [A, ceil(D/128)]); rows where perm is -1 get the
    quantization of a zero row.  With ``inv`` (moe_route's inverse map) each token row is
    quantized once and written to its top_k sorted rows (one read of x instead of top_k);
    without it each sorted row reads its token row."""
    _require(x.is_cuda and perm.is_cuda, "Input must be on CUDA")
    _require(x.ndim == 2 and perm.ndim == 1, "x must be [n_tokens, d] and perm 1-D")
    _require(top_k >= 1, "top_k must be >= 1")
    if inv is not None:
        _require(inv.numel() == x.shape[0] * top_k, "inv must hold n_tokens * top_k entries")
        return _run_detached(_scatter_quant_op, x, perm.to(torch.int64), inv.to(torch.int32), int(top_k),
                             bool(round_scale), bool(col_scales))
    return _run_detached(_gather_quant_op, x, perm.to(torch.int64), int(top_k), bool(round_scale), bool(col_scales))


def _codes_rows8(A, D, like):
    """[A, D] e4m3 codes whose rows start 8 bytes apart at least (the quantizer stores 8 codes
    at a time): a view of a buffer with rows padded to a multiple of 8 when D is not."""
    Dp = _cdiv(D, 8) * 8
    buf = like.new_empty((A, Dp), dtype=torch.float8_e4m3fn)
    return buf if Dp == D else buf[:, :D]


@custom_op("moe_gather_quant_rowwise",
           "(Tensor x, Tensor perm, int top_k, bool round_scale, bool col_scales) -> (Tensor, Tensor)")
def _gather_quant_op(x, perm, top_k, round_scale, col_scales):
    x = _x_rows16(x)
    A = perm.numel()
    T, D = x.shape
    pm = perm.contiguous()
    q = _codes_rows8(A, D, x)
    s = _scale_buf(x, A, _cdiv(D, 128), col_scales)
    call("cin_moe_gather_quant_rowwise", ptr(x), dtype_code(x), T, D, x.stride(0), ptr(pm), A, top_k,
         int(round_scale), ptr(q), q.stride(0), ptr(s), s.stride(0), s.stride(1), stream_of(x))
    return q, s


@_gather_quant_op.register_fake
def _(x, perm, top_k, round_scale, col_scales):
    A, D = perm.shape[0], x.shape[1]
    return _codes_rows8(A, D, x), _scale_buf(x, A, _cdiv(D, 128), col_scales)


def _x_rows16(x):
    """x with unit column stride and 16-byte aligned rows (the quantizer loads 16 bytes at a
    time): x itself when it qualifies, else a copy whose rows are padded to 16 bytes (the
    padding is never read: the kernel loads the last chunk of a row element by element)."""
    es = x.element_size()
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (x.stride(0) * es) % 16 == 0:
        return x
    T, D = x.shape
    per = 16 // es
    buf = x.new_empty((T, _cdiv(max(D, 1), per) * per))
    buf[:, :D].copy_(x)
    return buf[:, :D]


@custom_op("moe_scatter_quant_rowwise",
           "(Tensor x, Tensor perm, Tensor inv, int top_k, bool round_scale, bool col_scales) -> "
           "(Tensor, Tensor)")
def _scatter_quant_op(x, perm, inv, top_k, round_scale, col_scales):
    x = _x_rows16(x)
    A = perm.numel()
    T, D = x.shape
    pm, iv = perm.contiguous(), inv.contiguous()
    q = _codes_rows8(A, D, x)
    s = _scale_buf(x, A, _cdiv(D, 128), col_scales)
    if col_scales:
        # a token's scales go once into a token-major table, then to its sorted rows with
        # stores that run along the rows (308 -> 252 us at config 3; with row-major scales
        # the stores the kernel makes itself are faster, 263 against 326 us)
        ws = torch.empty(T * _cdiv(D, 128), dtype=torch.float32, device=x.device)
        call("cin_moe_scatter_quant_rowwise_ws", ptr(x), dtype_code(x), T, D, x.stride(0), ptr(iv),
             top_k, ptr(pm), A, int(round_scale), ptr(q), q.stride(0), ptr(s), s.stride(0), s.stride(1),
             ptr(ws), stream_of(x))
    else:
        call("cin_moe_scatter_quant_rowwise", ptr(x), dtype_code(x), T, D, x.stride(0), ptr(iv), top_k,
             ptr(pm), A, int(round_scale), ptr(q), q.stride(0), ptr(s), s.stride(0), s.stride(1),
             stream_of(x))
    return q, s


@_scatter_quant_op.register_fake
def _(x, perm, inv, top_k, round_scale, col_scales):
    A, D = perm.shape[0], x.shape[1]
    return _codes_rows8(A, D, x), _scale_buf(x, A, _cdiv(D, 128), col_scales)


def moe_gather_sum(g: torch.Tensor, inv: torch.Tensor, top_k: int,
                   out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Gradient of x[perm // top_k]: out[t] = sum of g[r] over token t's sorted positions r,
    in increasing r, fp32 sums -> [T, D] in out_dtype (T = inv.numel() // top_k)."""
    _require(g.is_cuda and inv.is_cuda, "Input must be on CUDA")
    _require(1 <= top_k <= MAX_TOP_K, f"top_k must be in [1, {MAX_TOP_K}]")
    _require(inv.numel() % top_k == 0, "inv must hold n_tokens * top_k entries")
    return _run_detached(_gather_sum_op, g, inv.to(torch.int32), int(top_k), out_dtype)


@custom_op("moe_gather_sum", "(Tensor g, Tensor inv, int top_k, ScalarType out_dtype) -> Tensor")
def _gather_sum_op(g, inv, top_k, out_dtype):
    gc = g if g.stride(1) == 1 else g.contiguous()
    iv = inv.contiguous()
    T = iv.numel() // top_k
    A, D = gc.shape
    out = torch.empty((T, D), dtype=out_dtype, device=g.device)
    call("cin_moe_gather_sum", ptr(gc), dtype_code(gc), gc.stride(0), ptr(iv), T, top_k, A, D,
         ptr(out), dtype_code(out), out.stride(0), stream_of(gc))
    return out


@_gather_sum_op.register_fake
def _(g, inv, top_k, out_dtype):
    return g.new_empty((inv.shape[0] // top_k, g.shape[1]), dtype=out_dtype)


# ---------------------------------------------------------------------------
# Weighted combine and its backward (reference :151-154)
# ---------------------------------------------------------------------------
def moe_combine(sorted_out: torch.Tensor, top_scores: torch.Tensor, inv: torch.Tensor) -> torch.Tensor:
    """routed_out [T, D] fp32 = sum over token t's assignments of sorted_out[r] *
    top_scores[t, j], added in increasing sorted position r (sorted_out fp32, fp16 or bf16,
    widened exactly)."""
    _require(sorted_out.is_cuda and top_scores.is_cuda and inv.is_cuda, "Input must be on CUDA")
    _require(top_scores.ndim == 2 and 1 <= top_scores.shape[1] <= MAX_TOP_K,
             f"top_scores must be [n_tokens, top_k] with top_k <= {MAX_TOP_K}")
    _require(inv.numel() == top_scores.numel(), "inv must hold n_tokens * top_k entries")
    _require(sorted_out.dtype in (torch.float32, torch.float16, torch.bfloat16),
             "sorted_out must be fp32, fp16 or bf16 (the experts' output)")
    return _run_detached(_combine_op, sorted_out, top_scores, inv.to(torch.int32))


@custom_op("moe_combine", "(Tensor y, Tensor scores, Tensor inv) -> Tensor")
def _combine_op(y, scores, inv):
    yc = y if y.stride(1) == 1 else y.contiguous()
    sc = scores if scores.stride(1) == 1 else scores.contiguous()
    iv = inv.contiguous()
    T, k = sc.shape
    A, D = yc.shape
    out = torch.empty((T, D), dtype=torch.float32, device=y.device)
    call("cin_moe_combine", ptr(yc), dtype_code(yc), yc.stride(0), ptr(sc), dtype_code(sc), sc.stride(0),
         ptr(iv), T, k, A, D, ptr(out), out.stride(0), stream_of(yc))
    return out


@_combine_op.register_fake
def _(y, scores, inv):
    return y.new_empty((scores.shape[0], y.shape[1]), dtype=torch.float32)


def moe_combine_backward(dout: torch.Tensor, sorted_out: torch.Tensor, top_scores: torch.Tensor,
                         perm: torch.Tensor, inv: torch.Tensor, dy_dtype: torch.dtype | None = None):
    """Gradients of moe_combine: (d sorted_out [A, D], d top_scores [T, k] fp32).

    d sorted_out is the fp32 product dout * score rounded (RNE) to dy_dtype, by default
    sorted_out's dtype (the dtype autograd gives the gradient of a tensor).  For fp16 sorted
    outputs, dy_dtype=torch.bfloat16 keeps tiny gradients: a loss averaged over many tokens
    gives row gradients of 1e-6 and below, which fp16 holds only as subnormals (and flushes
    below 6e-8), while bf16 keeps fp32's range at the same traffic; RoutedExpertsFunction
    asks for it."""
    _require(dout.is_cuda and sorted_out.is_cuda, "Input must be on CUDA")
    if dy_dtype is None:
        dy_dtype = sorted_out.dtype
    _require(dy_dtype in (torch.float32, torch.bfloat16, torch.float16), "dy_dtype must be fp32, bf16 or fp16")
    return _run_detached(_combine_bwd_op, dout.float(), sorted_out, top_scores, perm.to(torch.int64),
                         inv.to(torch.int32), dy_dtype)


@custom_op("moe_combine_backward",
           "(Tensor dout, Tensor y, Tensor scores, Tensor perm, Tensor inv, ScalarType dy_dtype)"
           " -> (Tensor, Tensor)")
def _combine_bwd_op(dout, y, scores, perm, inv, dy_dtype):
    dc = dout if dout.stride(1) == 1 else dout.contiguous()
    yc = y if y.stride(1) == 1 else y.contiguous()
    sc = scores if scores.stride(1) == 1 else scores.contiguous()
    pm, iv = perm.contiguous(), inv.contiguous()
    T, k = sc.shape
    A, D = yc.shape
    dy = torch.empty((A, D), dtype=dy_dtype, device=y.device)
    ds = torch.empty((T, k), dtype=torch.float32, device=y.device)
    call("cin_moe_combine_backward", ptr(dc), dc.stride(0), ptr(yc), dtype_code(yc), yc.stride(0),
         ptr(sc), dtype_code(sc), sc.stride(0), ptr(pm), ptr(iv), T, k, A, D, ptr(dy), dtype_code(dy),
         dy.stride(0), ptr(ds), stream_of(yc))
    return dy, ds


@_combine_bwd_op.register_fake
def _(dout, y, scores, perm, inv, dy_dtype):
    return (y.new_empty(y.shape, dtype=dy_dtype),
            y.new_empty(scores.shape, dtype=torch.float32))


# ---------------------------------------------------------------------------
# Autograd and the routed-experts block
# ---------------------------------------------------------------------------
class RoutedExpertsFunction(torch.autograd.Function):
    """The routed block as one autograd node: gather-quantize -> FP8 SwiGLU experts ->
    weighted combine, with gradients for x, the expert weights and the routing scores.

    The sorted expert outputs [A, D] are stored in fp16: the reference's routed experts
    return fp16 GEMM results (src/layers.py:69-75), and fp16 halves the traffic of the down
    GEMM's output, the combine and its backward.  They stay inside this node, so their
    gradient is not cast back to fp16 by autograd: the combine backward writes it in bf16
    (fp32's range) for the experts' backward, and the sorted-row input gradients come back
    in bf16 too, each token's sum added in fp32 and rounded once to x's dtype."""

    @staticmethod
    def forward(ctx, x, w12, w3, top_scores, perm, inv, starts, ends, top_k, weights_fp8=None):
        ys, saved = RoutedExpertsFunction.experts(x, w12, w3, perm, inv, starts, ends, top_k, weights_fp8)
        ctx.save_for_backward(*saved, ys, top_scores, perm, inv)
        ctx.top_k = top_k
        ctx.x_dtype = x.dtype
        ctx.w_dtypes = (w12.dtype, w3.dtype)
        return moe_combine(ys, top_scores, inv)

    @staticmethod
    def backward(ctx, dout):
        *saved, ys, top_scores, perm, inv = ctx.saved_tensors
        dy, ds = moe_combine_backward(dout, ys, top_scores, perm, inv,
                                      dy_dtype=torch.float32 if ys.dtype == torch.float32 else torch.bfloat16)
        dx, dw12, dw3 = RoutedExpertsFunction.experts_backward(tuple(saved), dy, inv, ctx.top_k, ctx.x_dtype)
        return (dx, dw12.to(ctx.w_dtypes[0]), dw3.to(ctx.w_dtypes[1]), ds.to(top_scores.dtype),
                None, None, None, None, None, None)

    @staticmethod
    def experts(x, w12, w3, perm, inv, starts, ends, top_k, weights_fp8=None):
        """Sorted expert outputs (fp16 [A, D]) and the tensors their backward needs."""
        xq, xs = moe_gather_quantize(x, perm, top_k, inv=inv, col_scales=True)
        return layers.experts_forward(xq, xs, w12, w3, starts, ends, x.dtype, weights_fp8,
                                      out_dtype=torch.float16)

    @staticmethod
    def experts_backward(saved, dy, inv, top_k, x_dtype):
        """(dx, dw12, dw3) from the sorted outputs' gradient dy [A, D] (bf16 or fp32)."""
        dxs, dw12, dw3 = layers.experts_backward(saved, dy, torch.bfloat16)
        return moe_gather_sum(dxs, inv, top_k, x_dtype), dw12, dw3


def routed_experts(experts: layers.GroupedExperts, x: torch.Tensor, top_idx: torch.Tensor,
                   top_scores: torch.Tensor):
    """The routed part of MoE.forward (reference src/layers.py:126-157) on the device.

    x [n_tokens, d_model] (bf16/fp16/fp32), top_idx [n_tokens, k] expert ids, top_scores
    [n_tokens, k] gate weights.  Returns (routed_out [n_tokens, d_model] fp32, expert_counts
    int64 [E]) -- the reference's routed_out (before the view) and the bincount it feeds to
    the expert-bias update.  Autograd reaches x, experts.w12 / w3 and top_scores.
    """
    _require(x.is_cuda, "Input must be on CUDA")
    _require(top_idx.shape == top_scores.shape and top_idx.shape[0] == x.shape[0],
             "top_idx and top_scores must be [n_tokens, top_k]")
    k = top_idx.shape[1]
    _require(1 <= k <= MAX_TOP_K, f"top_k must be in [1, {MAX_TOP_K}]")
    perm, inv, counts, starts, ends = moe_route(top_idx, experts.n_experts)
    out = RoutedExpertsFunction.apply(x, experts.w12, experts.w3, top_scores, perm, inv, starts, ends, k,
                                      experts.quantized_weights())
    return out, counts


# ---------------------------------------------------------------------------
# The whole layer for a few tokens (reference src/layers.py:113-157 at generation)
# ---------------------------------------------------------------------------
def moe_decode(x: torch.Tensor, router_weight: torch.Tensor, experts, top_k: int, bias: torch.Tensor | None = None,
               score: str = "sigmoid", n_groups: int = 1, top_groups: int | None = None, group_top: int = 2,
               renormalize: bool = True, scale: float = 1.0, shared=None, return_routing: bool = False):
    """The mixture-of-experts layer of a generation step: x [n_tokens, D] (bf16, fp16 or fp32, at most 128
    tokens) -> out of the same shape and dtype,

      top_idx, top_scores = moe_gate(x @ router_weight.T, top_k, bias, score, n_groups, ...)
      out_t = sum_j top_scores[t, j] * expert_{top_idx[t, j]}(x_t) + shared(x_t)
      expert(v) = W3 (silu(W1 v) * (W2 v))

    and with return_routing (out, top_idx int64, top_scores fp32 [n_tokens, top_k]).

    router_weight [E, D] in bf16, fp16 or fp32 (E at most 1024), the other options as in moe_gate; the logits are summed
    and the experts chosen in 64 bits.  experts: a layers.GroupedExperts, whose FP8 weights are used (kept between
    calls with its weight cache, else quantized in every call), or (w12, w12_scales, w3, w3_scales): w12
    [E, 2 H, D] (W1 above W2) and w3 [E, D, H], either e4m3 codes with fp32 scales of 128 x 128 blocks
    ([E, ceil(2 H / 128), ceil(D / 128)] and [E, ceil(D / 128), ceil(H / 128)], as
    layers.quantize_expert_weights returns them) or bf16 with None for the scales.  shared: None or such a tuple of one
    expert, without E and with an H of its own.  D and H are multiples of 16.  Weights and scales that are not contiguous, or
    whose first element is not on 16 bytes, are copied whole in every call.

    Only the chosen experts' weights are read.  Unlike in routed_experts activations are not quantized: x is exact in the
    products, silu(W1 v) * (W2 v) keeps 24 bits, products are summed in fp32 and the result is rounded once.
    Bit-identical from call to call.  Inference only: where x, a weight (also of a GroupedExperts), a scale or the bias
    requires a gradient, the backward is refused (under torch.compile, which forms it at once, the call is); torch.no_grad()
    saves the host work of that."""
    _require(x.is_cuda, "Input must be on CUDA")
    _require(x.ndim == 2 and x.shape[0] <= MAX_DECODE_TOKENS, "x must be [n_tokens, D] with at most 128 tokens")
    _require(x.dtype in _DTYPES, "x must be bf16, fp16 or fp32")
    dev, D = x.device, x.shape[1]
    _require(router_weight.ndim == 2 and router_weight.shape[1] == D and router_weight.device == dev
             and router_weight.dtype in _DTYPES, "router_weight must be [E, D] on x's device, in bf16, fp16 or fp32")
    E = router_weight.shape[0]
    _require(1 <= E <= MAX_DECODE_EXPERTS, "n_experts must be in [1, 1024]")
    _require(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _require(1 <= n_groups <= MAX_GROUPS and E % n_groups == 0, "n_groups must divide n_experts and be in [1, 64]")
    top_groups = n_groups if top_groups is None else top_groups
    _require(1 <= top_groups <= n_groups, "top_groups must be in [1, n_groups]")
    _require(group_top in (1, 2), "group_top must be 1 or 2")
    _require(1 <= top_k <= min(MAX_TOP_K, top_groups * (E // n_groups)),
             "top_k must be in [1, 16] and within the experts of the kept groups")
    if bias is not None:
        _require(bias.shape == (E,) and bias.device == dev and bias.dtype == torch.float32,
                 "bias must be fp32 [n_experts] on x's device")
        bias = _without_grad(bias)
    trained = None
    if isinstance(experts, layers.GroupedExperts):
        _require(experts.n_experts == E and experts.d_model == D, "the router and the experts differ in number or width")
        _require(D % 128 == 0 and experts.hidden_dim % 64 == 0, "GroupedExperts' FP8 blocks need D in multiples of 128, H of 64")
        w12, w3 = experts.w12.detach(), experts.w3.detach()
        H = experts.hidden_dim
        if torch.is_grad_enabled():  # (their codes record no graph)
            trained = next((w for w in (experts.w12, experts.w3) if w.requires_grad), None)
        q = experts.quantized_weights()
        (w12q, _, w12s), (w3q, _, w3s) = q if q is not None else layers.quantize_expert_weights(w12, w3)
        experts = (w12q.view(E, 2 * H, D), w12s.view(E, 2 * H // 128, -1), w3q.view(E, D, H), w3s.view(E, D // 128, -1))
    weights = _decode_weights(experts, x, (E,))
    extra = (None,) * 4
    if shared is not None:
        extra = _decode_weights(shared, x, ())
        _require(extra[0].dtype == weights[0].dtype, "the shared expert's weights must have the experts' type")
    out = _run_detached(_decode_op, x, router_weight, bias, *weights, *extra, int(top_k), _SCORES[score], int(n_groups),
                        int(top_groups), int(group_top), bool(renormalize), float(scale), trained)
    return out if return_routing else out[0]


def _decode_weights(weights, x, lead):
    """The four tensors of stacked experts (lead (E,)) or of one (()), checked."""
    _require(isinstance(weights, (tuple, list)) and len(weights) == 4, "expert weights must be (w12, w12_scales, w3, w3_scales)")
    w12, s12, w3, s3 = weights
    D, dev, dt = x.shape[1], x.device, w12.dtype
    H = w3.shape[-1] if w3.ndim else 0
    _require(w12.shape == (*lead, 2 * H, D) and w3.shape == (*lead, D, H), "w12 must be [E, 2 H, D] and w3 [E, D, H]")
    _require(D >= 16 and H >= 16 and D % 16 == 0 and H % 16 == 0 and D <= 65536 and H <= 65536,
             "D and H must be multiples of 16 up to 65536")
    _require(dt == w3.dtype and w12.device == dev and w3.device == dev, "weights must share one dtype, on x's device")
    if dt == torch.bfloat16:
        _require(s12 is None and s3 is None, "bf16 weights have no scales")
        return _without_grad(w12), None, _without_grad(w3), None
    _require(dt == torch.float8_e4m3fn, "weights must be e4m3 codes or bf16")
    _require(s12 is not None and s3 is not None and s12.dtype == torch.float32 and s3.dtype == torch.float32
             and s12.device == dev and s3.device == dev and s12.shape == (*lead, _cdiv(2 * H, 128), _cdiv(D, 128))
             and s3.shape == (*lead, _cdiv(D, 128), _cdiv(H, 128)), "codes need fp32 scales of their 128 x 128 blocks, on x's device")
    return w12, _without_grad(s12), w3, _without_grad(s3)


def _without_grad(t):
    """A plain tensor; but what records a graph stays, so that the operator refuses its backward."""
    # (detach costs 0.6 us of host time each)
    if t.requires_grad:
        return t if torch.is_grad_enabled() else t.detach()
    return t if type(t) is torch.Tensor else t.detach()


@functools.lru_cache(maxsize=256)
def _decode_workspace(dtype, *sizes):
    n = _lib.load().cin_moe_decode_workspace(dtype_code(dtype), *sizes)
    if n < 0:
        raise ValueError(f"moe_decode: {_lib.last_error()}")
    return n


def _on16(t):
    """(contiguous, its first element on 16 bytes; its address)"""
    if t is None:
        return None, 0
    at = t.data_ptr()
    if at % 16 or not t.is_contiguous():
        t = t.clone(memory_format=torch.contiguous_format)
        at = t.data_ptr()
    return t, at


@custom_op("moe_decode", "(Tensor x, Tensor router, Tensor? bias, Tensor w12, Tensor? s12, Tensor w3, Tensor? s3, Tensor? shared_w12, "
           "Tensor? shared_s12, Tensor? shared_w3, Tensor? shared_s3, int top_k, int score, int n_groups, int top_groups, "
           "int group_top, bool renormalize, float scale, Tensor? trained=None) -> (Tensor, Tensor, Tensor)")
def _decode_op(x, router, bias, w12, s12, w3, s3, sw12, ss12, sw3, ss3, top_k, score, n_groups, top_groups, group_top, renormalize,
               scale, trained=None):
    # trained: a weight behind the codes that records a graph, for the refusal of its backward alone
    x, router = _gate_rows(x), _gate_rows(router)
    T, D = x.shape
    E, H = router.shape[0], w3.shape[-1]
    Hs = 0 if sw3 is None else sw3.shape[-1]
    held, p = zip(*[_on16(t) for t in (w12, s12, w3, s3, sw12, ss12, sw3, ss3)])
    bias = None if bias is None else bias.contiguous()
    out = x.new_empty((T, D))
    idx = x.new_empty((T, top_k), dtype=torch.int64)
    weights = x.new_empty((T, top_k), dtype=torch.float32)
    ws = _decode_workspace(x.dtype, T, D, E, top_k, H, Hs)
    work = torch.empty(ws, dtype=torch.uint8, device=x.device)
    call_on(x, "cin_moe_decode", x.data_ptr(), dtype_code(x), max(x.stride(0), D), T, D, router.data_ptr(), dtype_code(router),
            max(router.stride(0), D), E, ptr(bias), top_k, score, n_groups, top_groups, group_top, renormalize, scale,
            w12.dtype == torch.float8_e4m3fn, *p[:4], H, *p[4:], Hs, out.data_ptr(), idx.data_ptr(), weights.data_ptr(),
            work.data_ptr(), ws, stream_of(x))
    return out, idx, weights


@_decode_op.register_fake
def _(x, router, bias, w12, s12, w3, s3, sw12, ss12, sw3, ss3, top_k, *options):
    T, D = x.shape
    return (x.new_empty((T, D)), x.new_empty((T, top_k), dtype=torch.int64), x.new_empty((T, top_k), dtype=torch.float32))
