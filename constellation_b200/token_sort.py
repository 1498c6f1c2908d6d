"""Tokens sorted by expert and back, with gradients.

The dispatch and the combine around expert products that take rows grouped by expert
(``dispatch_topk_experts`` / ``combine_outputs_torch``, ``server/moe_layer_runtime.py:111-167``), for a
whole batch and without a host synchronisation::

    order = sort_routes(topk_idx, n_experts)                  # (expert, token, k)
    rows = sort_tokens(x, order)                              # [T * K, H], expert e at offsets[e]
    y = ...                                                   # products of the rows, e.g. grouped_int4
    out = unsort_tokens(y, order, topk_weight, residual=h)    # out[t] = sum_k w[t, k] y[row_of[t, k]] + h[t]

Shapes depend on ``T`` and ``K`` alone: routes to experts held elsewhere leave rows behind
``offsets[-1]``, which are zero.  Sums run in fp32 in the order of ``k`` and are rounded once, so
results repeat bit for bit.

``sort_tokens`` and ``unsort_tokens`` record their gradients where an input asks for one (not twice
differentiable; forward-mode tangents are refused).  Under CUDA graph capture autograd is refused, on
both passes: a capture calls ``sort_tokens_backward`` and ``unsort_tokens_backward``, which are plain
launches.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check
from .context import _MOST_ROWS, _empty, _no_tangent, _on, _ptr, _rows, _stream, dtype_code


@dataclass(frozen=True)
class TokenOrder:
    """Routes in the order (expert, token, k), as ``sort_routes`` makes it: contiguous int32 on one device."""

    row_of: torch.Tensor    # [T, K] row of a route, -1 where its expert is held elsewhere
    route_of: torch.Tensor  # [T * K] t * K + k of a row, -1 behind the last expert's rows
    offsets: torch.Tensor   # [n_experts + 1] first row of each expert; the last entry: rows in use

    def __post_init__(self):
        r, q, o = self.row_of, self.route_of, self.offsets
        if r.dim() != 2 or q.dim() != 1 or o.dim() != 1 or q.shape[0] != r.numel() or o.shape[0] < 2 \
                or q.shape[0] > _MOST_ROWS:
            raise RuntimeError("not an order: row_of [T, K], route_of [T * K] and offsets [n_experts + 1] are expected")
        dev = r.device
        for t in (r, q, o):
            if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
                raise RuntimeError("an order is contiguous int32 on one device")


def _made(row_of, route_of, offsets) -> TokenOrder:
    """A ``TokenOrder`` of tensors that were made as one, without the checks of one that a caller makes."""
    order = object.__new__(TokenOrder)
    order.__dict__.update(row_of=row_of, route_of=route_of, offsets=offsets)
    return order


def sort_routes(topk_idx: torch.Tensor, n_experts: int, *, first_expert: int = 0) -> TokenOrder:
    """The order of ``topk_idx`` (``[T, K]`` int32 or int64) over the experts ``[first_expert,
    first_expert + n_experts)``, at most 1024; any other id, -1 among them, is a route to an expert
    held elsewhere.  A token may name an expert twice; each route has its own row."""
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dim() != 2 or not topk_idx.is_cuda:
        raise TypeError("sort_routes expects a 2-D CUDA tensor")
    if topk_idx.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_idx must be int32 or int64, got {topk_idx.dtype}")
    T, K = topk_idx.shape
    n = T * K
    if n > _MOST_ROWS:
        raise RuntimeError(f"sort_routes takes at most 2^30 routes, got {n}")
    dev = topk_idx.device
    topk_idx = topk_idx.contiguous()
    n_experts = int(n_experts)
    if not 1 <= n_experts <= 1024:
        raise ValueError(f"n_experts must be in [1, 1024], got {n_experts}")
    if not 0 <= first_expert < 1 << 31:
        raise ValueError(f"first_expert must be in [0, 2^31), got {first_expert}")
    row_of = _empty(T, K, torch.int32, dev)
    route_of = torch.empty_strided((n,), (1,), dtype=torch.int32, device=dev)
    offsets = torch.empty_strided((n_experts + 1,), (1,), dtype=torch.int32, device=dev)
    with _on(dev):
        check(_lib.lib.cst_sort_routes(topk_idx.data_ptr(), topk_idx.element_size(), T, K, n_experts,
                                       int(first_expert), row_of.data_ptr(), route_of.data_ptr(), offsets.data_ptr(),
                                       _stream(dev)))
    return _made(row_of, route_of, offsets)


def _check_order(order: TokenOrder, dev: torch.device) -> None:
    if order.row_of.device != dev:
        raise RuntimeError(f"device mismatch: rows={dev} order={order.row_of.device}")


def _matrix(name: str, t: torch.Tensor, rows: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or not t.is_cuda:
        raise TypeError(f"{name} must be a 2-D CUDA tensor")
    if t.shape[0] != rows or not 1 <= t.shape[1] <= 1 << 30:
        raise RuntimeError(f"{name} must be [{rows}, H] with H in [1, 2^30], got {tuple(t.shape)}")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors])


def _refuse_capture(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: autograd is not supported under CUDA graph capture; call the operators on "
                           "detached tensors and sort_tokens_backward / unsort_tokens_backward")


def _end(order: TokenOrder) -> int:
    """Address of the rows in use (the last of the offsets)."""
    return order.offsets.data_ptr() + 4 * (order.offsets.shape[0] - 1)


def _sort(x, order, scale):
    T, K = order.row_of.shape
    H, dev = x.shape[1], x.device
    x, ld = _rows(x)
    size = x.element_size()
    rows = _empty(T * K, H, x.dtype, dev)
    rows_scale, n_scale, ld_scale = None, 0, 0
    if scale is not None:
        scale, ld_scale = _rows(scale)
        n_scale = scale.shape[1]
        rows_scale = _empty(T * K, n_scale, torch.float32, dev)
    with _on(dev):
        check(_lib.lib.cst_sort_rows(x.data_ptr(), H * size, ld * size, _ptr(scale), n_scale, ld_scale, T, K,
                                     order.row_of.data_ptr(), _end(order), rows.data_ptr(), _ptr(rows_scale),
                                     _stream(dev)))
    return rows, rows_scale


def _unsort(rows, order, weight, residual, out_dtype):
    T, K = order.row_of.shape
    H, dev = rows.shape[1], rows.device
    rows, ld = _rows(rows)
    rt, ldr = 0, 0
    if residual is not None:
        residual, ldr = _rows(residual)
        rt = dtype_code(residual.dtype)
    out = _empty(T, H, out_dtype, dev)
    with _on(dev):
        check(_lib.lib.cst_unsort_rows(rows.data_ptr(), dtype_code(rows.dtype), ld, order.row_of.data_ptr(),
                                       _ptr(weight), T, K, H, _ptr(residual), rt, ldr, out.data_ptr(),
                                       dtype_code(out_dtype), _stream(dev)))
    return out


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.save_for_backward(order.row_of, order.route_of, order.offsets)
        return _sort(x, order, None)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_capture("sort_tokens")
        return sort_tokens_backward(grad, _made(*ctx.saved_tensors)), None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, residual, order, out_dtype):
        ctx.residual_dtype = None if residual is None else residual.dtype
        ctx.weighted = weight is not None
        saved = [order.row_of, order.route_of, order.offsets]
        need_rows = ctx.weighted and weight.requires_grad
        ctx.rows_dtype, ctx.has_rows = rows.dtype, need_rows
        saved += ([weight] if ctx.weighted else []) + ([rows] if need_rows else [])
        ctx.save_for_backward(*saved)
        return _unsort(rows, order, weight, residual, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_capture("unsort_tokens")
        _no_tangent("unsort_tokens' gradient", grad)
        saved = ctx.saved_tensors
        order = _made(*saved[:3])
        weight = saved[3] if ctx.weighted else None
        rows = saved[4] if ctx.has_rows else None
        d_rows, d_weight = _unsort_grad(grad, rows, ctx.rows_dtype, order, weight, ctx.needs_input_grad[0],
                                        ctx.needs_input_grad[1])
        d_residual = grad.to(ctx.residual_dtype) if ctx.needs_input_grad[2] else None
        return d_rows, d_weight, d_residual, None, None


def sort_tokens(x: torch.Tensor, order: TokenOrder, *, scale: torch.Tensor | None = None):
    """``rows[row_of[t, k]] = x[t]``, ``[T * K, H]``; rows behind ``order.offsets[-1]`` are zero.

    ``x`` is fp16, bf16, fp32, or e4m3; with ``scale`` (fp32 ``[T, n]``, the row scales of e4m3 rows) the
    scales are sorted with them and ``(rows, rows_scale)`` is returned.  The gradient of ``x`` is the sum
    of its rows' gradients in fp32, rounded once."""
    T = order.row_of.shape[0]
    _matrix("x", x, T)
    _check_order(order, x.device)
    if x.dtype != torch.float8_e4m3fn:
        dtype_code(x.dtype)
    _no_tangent("sort_tokens", x, scale)
    if scale is not None:
        _matrix("scale", scale, T)
        if scale.dtype != torch.float32 or scale.device != x.device:
            raise RuntimeError("scale must be fp32 on the device of x")
        if _wants_grad(scale, x):
            raise RuntimeError("rows with scales have no gradient")
        return _sort(x, order, scale)
    if _wants_grad(x):
        if x.dtype == torch.float8_e4m3fn:
            raise RuntimeError("e4m3 rows have no gradient")
        _refuse_capture("sort_tokens")
        return _SortTokens.apply(x, order)
    return _sort(x, order, None)[0]


def unsort_tokens(rows: torch.Tensor, order: TokenOrder, weight: torch.Tensor | None = None, *,
                  residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``out[t] = sum_k weight[t, k] * rows[row_of[t, k]] (+ residual[t])``, ``[T, H]`` in ``out_dtype`` (that of
    ``rows`` if None).

    ``rows`` and ``residual`` are fp16, bf16 or fp32, each in its own type; ``weight`` is fp32 ``[T, K]`` or
    None (ones).  A route held elsewhere adds nothing, whatever its weight, and its weight's gradient is
    zero; so are the gradients of rows behind ``order.offsets[-1]``."""
    T, K = order.row_of.shape
    _matrix("rows", rows, T * K)
    _check_order(order, rows.device)
    dtype_code(rows.dtype)
    out_dtype = out_dtype or rows.dtype
    dtype_code(out_dtype)
    if weight is not None:
        if weight.dtype != torch.float32 or weight.shape != (T, K) or weight.device != rows.device:
            raise RuntimeError(f"weight must be fp32 [{T}, {K}] on the device of rows")
        weight = weight.contiguous()
    if residual is not None:
        _matrix("residual", residual, T)
        dtype_code(residual.dtype)
        if residual.shape[1] != rows.shape[1] or residual.device != rows.device:
            raise RuntimeError("residual must be [T, H] on the device of rows")
    _no_tangent("unsort_tokens", rows, weight, residual)
    if _wants_grad(rows, weight, residual):
        _refuse_capture("unsort_tokens")
        return _UnsortTokens.apply(rows, weight, residual, order, out_dtype)
    return _unsort(rows, order, weight, residual, out_dtype)


def sort_tokens_backward(grad_rows: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """The gradient of ``sort_tokens``'s ``x`` for ``grad_rows`` (``[T * K, H]``): ``unsort_tokens`` without weights."""
    T, K = order.row_of.shape
    _matrix("grad_rows", grad_rows, T * K)
    _check_order(order, grad_rows.device)
    _no_tangent("sort_tokens_backward", grad_rows)
    return _unsort(grad_rows.detach(), order, None, None, grad_rows.dtype)


def unsort_tokens_backward(grad: torch.Tensor, rows: torch.Tensor, order: TokenOrder,
                           weight: torch.Tensor | None = None):
    """The gradients ``(d_rows, d_weight)`` of ``unsort_tokens`` for ``grad`` (``[T, H]``); ``d_weight`` is None
    without ``weight``.  ``d_rows`` has the type of ``rows``."""
    T, K = order.row_of.shape
    _matrix("grad", grad, T)
    _matrix("rows", rows, T * K)
    _check_order(order, rows.device)
    dtype_code(rows.dtype)
    if grad.shape[1] != rows.shape[1] or grad.device != rows.device:
        raise RuntimeError("grad must be [T, H] on the device of rows")
    if weight is not None:
        if weight.dtype != torch.float32 or weight.shape != (T, K) or weight.device != rows.device:
            raise RuntimeError(f"weight must be fp32 [{T}, {K}] on the device of rows")
    _no_tangent("unsort_tokens_backward", grad, rows, weight)
    if weight is not None:
        weight = weight.detach().contiguous()
    return _unsort_grad(grad.detach(), rows.detach(), rows.dtype, order, weight, True, weight is not None)


def _unsort_grad(grad, rows, rows_dtype, order, weight, need_rows, need_weight):
    T, K = order.row_of.shape
    H, dev = grad.shape[1], grad.device
    grad, ld_grad = _rows(grad)
    ld_rows = 0
    if rows is not None:
        rows, ld_rows = _rows(rows)
    d_rows = _empty(T * K, H, rows_dtype, dev) if need_rows else None
    d_weight = _empty(T, K, torch.float32, dev) if need_weight else None
    with _on(dev):
        check(_lib.lib.cst_unsort_rows_grad(grad.data_ptr(), dtype_code(grad.dtype), ld_grad, _ptr(rows),
                                            dtype_code(rows_dtype), ld_rows, order.row_of.data_ptr(), _ptr(weight),
                                            _end(order), T, K, H, _ptr(d_rows), _ptr(d_weight), _stream(dev)))
    return d_rows, d_weight
