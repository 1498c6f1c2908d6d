"""Experts held in 4 bits: weights with group scales, their grouped products, and the layer over them.

``Int4Weight`` holds ``E`` weights ``[N, K]`` as 4-bit integers with one scale (and optionally one zero
point) for 32, 64 or 128 consecutive ``k``; ``grouped_int4`` multiplies rows sorted by expert with them
(``cst_grouped_int4``); ``Int4Experts`` is the compute object of a sparse layer over such experts, with
the routing, residency and layer calls of ``ExpertContext`` that ``MoEStack`` and ``ExpertParallelMoE`` use.
An expert takes 0.53 of its FP8 size at groups of 128, and a decode step streams that much less.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import CST_DTYPE_E4M3, check
from .context import (ExpertContext, MoEConfig, _empty, _no_grad, _on, _ptr, _rows, _stream, dtype_code)
from .fp8_utils import dequant_fp8_weight_blockwise
from .token_sort import sort_routes, sort_tokens, unsort_tokens


def quantize_int4(w: torch.Tensor, group: int = 128, *, symmetric: bool = True,
                  scale_dtype: torch.dtype = torch.float16):
    """``w [..., N, K]`` to 4 bits with one scale for ``group`` consecutive ``k``, rounded to nearest; returns
    ``(q, scale, zero)`` as ``Int4Weight`` takes them.  Symmetric: ``scale = max |w| / 7``, ``zero`` None
    (8); otherwise the group's range, widened to hold 0, over 15 steps and a zero point."""
    if group not in (32, 64, 128) or w.dim() < 2 or w.shape[-1] % group:
        raise ValueError(f"group must be 32, 64 or 128 and divide K={w.shape[-1] if w.dim() else 0}, got {group}")
    v = w.detach().float().unflatten(-1, (-1, group))
    if symmetric:
        step, zero = v.abs().amax(-1) / 7, None
    else:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        step = (hi - lo) / 15
    # the quotients are taken with the scale as it is stored
    scale = torch.where(step > 0, step, torch.ones_like(step)).to(scale_dtype)
    scale = torch.where(scale == 0, torch.full_like(scale, torch.finfo(scale_dtype).tiny), scale)
    if not symmetric:
        zero = torch.round(-lo / scale.float()).clamp(0, 15)
    q = torch.round(v / scale.float().unsqueeze(-1)) + (8.0 if zero is None else zero.unsqueeze(-1))
    q = q.clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale, None if zero is None else zero.to(torch.uint8)


class Int4Weight:
    """``E`` weights ``[N, K]`` in 4 bits, in the kernels' layout, laid out once.

    ``q`` is uint8 ``[E, N, K / 2]`` (two values a byte, the lower ``k`` in the lower half), ``scale``
    ``[E, N, K / group]`` in fp16, bf16 or fp32 and ``zero`` uint8 ``[E, N, K / group]`` in 0..15 or None
    (8): ``W = scale * (q - zero)``.  The leading dimension may be left out (one weight).  With ``swiglu``
    the rows are the "up" half, then the "gate" half, and products return ``silu(gate) * up``."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None, *,
                 swiglu: bool = False):
        for name, t in (("q", q), ("scale", scale), ("zero", zero)):
            if t is not None and (not isinstance(t, torch.Tensor) or t.dim() not in (2, 3) or not t.is_cuda):
                raise TypeError(f"{name} must be a 2-D or 3-D CUDA tensor")
        if q.dim() == 2:
            q, scale = q[None], scale[None] if scale.dim() == 2 else scale
            zero = zero[None] if zero is not None and zero.dim() == 2 else zero
        E, N, K = q.shape[0], q.shape[1], 2 * q.shape[2]
        if scale.dim() != 3 or scale.shape[:2] != (E, N) or not scale.shape[2] or K % scale.shape[2]:
            raise RuntimeError(f"scale must be [{E}, {N}, {K} / group], got {tuple(scale.shape)}")
        self._init(E, N, K, K // scale.shape[2], scale.dtype, zero is not None, swiglu, q.device)
        self._pack(0, E, q, scale, zero)

    @classmethod
    def empty(cls, n_experts: int, n: int, k: int, *, group: int = 128, scale_dtype: torch.dtype = torch.float16,
              zero_points: bool = False, swiglu: bool = False, device="cuda") -> "Int4Weight":
        """Room for ``n_experts`` weights; one that is not loaded is all zero."""
        w = cls.__new__(cls)
        w._init(n_experts, n, k, group, scale_dtype, zero_points, swiglu, torch.device(device))
        return w

    def _init(self, E, N, K, group, scale_dtype, has_zero, swiglu, device):
        if device.type != "cuda":
            raise RuntimeError(f"Int4Weight needs a CUDA device, got {device}")
        self._c = _lib.CstInt4Weight(int(E), int(N), int(K), int(group), dtype_code(scale_dtype), int(has_zero),
                                     int(bool(swiglu)))
        self._ref = ctypes.byref(self._c)
        size = ctypes.c_int64()
        check(_lib.lib.cst_int4_bytes(self._ref, ctypes.byref(size)))
        self.n_experts, self.n, self.k, self.group = int(E), int(N), int(K), int(group)
        self.scale_dtype, self.zero_points, self.swiglu = scale_dtype, bool(has_zero), bool(swiglu)
        self.out_features = self.n // 2 if swiglu else self.n
        self.data = torch.zeros(size.value, dtype=torch.uint8, device=device)
        self.device = self.data.device
        self._sizes: dict = {}  # bytes of a workspace by x's type and rows

    def load(self, expert: int, q: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None) -> None:
        """Lay expert ``expert``'s ``q [N, K / 2]``, ``scale`` and ``zero`` ``[N, K / group]`` out (stream-ordered)."""
        if not 0 <= expert < self.n_experts:
            raise IndexError(f"expert {expert} outside [0, {self.n_experts})")
        self._pack(int(expert), 1, q[None], scale[None], None if zero is None else zero[None])

    def _pack(self, first, count, q, scale, zero):
        G = self.k // self.group
        _no_grad("Int4Weight", scale)
        if (zero is not None) != self.zero_points:
            raise RuntimeError("zero points are given for all experts of a weight or for none")
        for name, t, shape, dtype in (("q", q, (count, self.n, self.k // 2), torch.uint8),
                                      ("scale", scale, (count, self.n, G), self.scale_dtype),
                                      ("zero", zero, (count, self.n, G), torch.uint8)):
            if t is not None and (tuple(t.shape) != shape or t.dtype != dtype or t.device != self.device):
                raise RuntimeError(f"{name} must be {dtype} {list(shape)} on {self.device}, got {t.dtype} "
                                   f"{list(t.shape)} on {t.device}")
        q, scale = q.contiguous(), scale.contiguous()
        zero = zero.contiguous() if zero is not None else None
        with _on(self.device):
            check(_lib.lib.cst_int4_pack(self._ref, first, count, q.data_ptr(), scale.data_ptr(), _ptr(zero),
                                         self.data.data_ptr(), _stream(self.device)))

    def _workspace(self, xt: int, R: int) -> int:
        size = self._sizes.get((xt, R))
        if size is None:
            got = ctypes.c_int64()
            check(_lib.lib.cst_int4_workspace(self._ref, xt, R, ctypes.byref(got)))
            if len(self._sizes) >= 64:
                self._sizes.clear()
            size = self._sizes[(xt, R)] = got.value
        return size

    def device_error(self) -> None:
        """Wait for the current stream and raise if a product's bounded device-side wait gave up."""
        with _on(self.device):
            check(_lib.lib.cst_int4_device_error(self._ref, self.data.data_ptr(), _stream(self.device)))


def grouped_int4(x: torch.Tensor, w: Int4Weight, offsets: torch.Tensor | None = None, *,
                 x_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[r] = W[e] x[r]`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of each expert; rows outside are zero.

    ``x [R, K]`` is fp16, bf16, or e4m3 with ``x_scale`` fp32 ``[R, ceil(K / 128)]`` (as ``add_rms_norm_fp8``
    leaves them, sorted by ``sort_tokens``).  ``offsets`` is int32 ``[E + 1]`` on the device, ascending
    (``TokenOrder.offsets``); without it there is one weight and it takes every row.  The result is
    ``[R, N]`` (``[R, N / 2]`` with swiglu) in ``out_dtype``: fp16, bf16 or fp32; by default ``x``'s type, bf16
    for e4m3 rows.  ``out`` may not overlap ``x``, ``x_scale``, ``offsets`` or the weight's ``data``.

    fp32 sums, one rounding.  fp16 and bf16 rows enter as 8-bit terms: exactly where a number is above 2^-11 (fp16) or
    2^-13 (bf16) of its row's largest, and with an error below 2^-22 (2^-21) of that largest elsewhere, which is also
    below 2^-18 (2^-17) of the largest of its 128 columns.  Rows whose 128-column blocks differ by 5 binades or more, as
    around outliers, take up to 1.35 times as long.  An infinity makes its row's results NaN."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not x.is_cuda:
        raise TypeError("grouped_int4 expects a 2-D CUDA tensor")
    dev = x.device
    if dev != w.device:
        raise RuntimeError(f"device mismatch: x={dev} weight={w.device}")
    R, K = x.shape
    if K != w.k or R > 1 << 28:
        raise RuntimeError(f"x must be [R, {w.k}] with R at most 2^28, got {tuple(x.shape)}")
    if x.dtype == torch.float8_e4m3fn:
        xt = CST_DTYPE_E4M3
        if x_scale is None:
            raise RuntimeError("e4m3 rows need their x_scale")
        if (x_scale.dtype != torch.float32 or tuple(x_scale.shape) != (R, (K + 127) // 128)
                or x_scale.device != dev):
            raise RuntimeError(f"x_scale must be fp32 [{R}, {(K + 127) // 128}] on the device of x")
    elif x.dtype in (torch.float16, torch.bfloat16):
        xt = dtype_code(x.dtype)
        if x_scale is not None:
            raise RuntimeError("x_scale goes with e4m3 rows")
    else:
        raise TypeError(f"x must be float16, bfloat16 or float8_e4m3fn, got {x.dtype}")
    _no_grad("grouped_int4", x, x_scale)
    if offsets is None:
        if w.n_experts != 1:
            raise RuntimeError(f"offsets are needed for {w.n_experts} experts")
    elif offsets.dtype != torch.int32 or offsets.shape != (w.n_experts + 1,) or offsets.device != dev:
        raise RuntimeError(f"offsets must be int32 [{w.n_experts + 1}] on the device of x")
    else:
        offsets = offsets.contiguous()
    if out is None:
        out = _empty(R, w.out_features, out_dtype or (torch.bfloat16 if xt == CST_DTYPE_E4M3 else x.dtype), dev)
    elif (out.shape != (R, w.out_features) or out.device != dev or not out.is_contiguous()
          or out_dtype not in (None, out.dtype)):
        raise RuntimeError(f"out must be contiguous [{R}, {w.out_features}] on the device of x, of the out_dtype given")
    ot = dtype_code(out.dtype)
    x, ldx = _rows(x)
    lds = 0
    if x_scale is not None:
        x_scale, lds = _rows(x_scale)
    room = torch.empty_strided((w._workspace(xt, R),), (1,), dtype=torch.uint8, device=dev)
    with _on(dev):
        check(_lib.lib.cst_grouped_int4(w._ref, w.data.data_ptr(), x.data_ptr(), xt, ldx, _ptr(x_scale), lds,
                                        _ptr(offsets), R, room.data_ptr(), out.data_ptr(), ot, w.out_features,
                                        _stream(dev)))
    return out


class Int4Experts:
    """The routed experts ``[first_expert, first_expert + n_local)`` of a layer, and its shared expert, in 4 bits.

    Takes the place of an ``ExpertContext`` as the compute object of ``MoEStack`` and of
    ``ExpertParallelMoE`` (one rank, or the all-gather exchange): ``route``, ``moe_routed``,
    ``moe_routed_range``, ``moe_layer`` and ``cast_extra``.  Experts are uploaded in the reference's FP8
    format and quantised here (``upload_expert``), or as 4-bit tensors (``load_expert``).  ``x`` is fp16 or
    bf16; the hidden rows between the two products are in ``x``'s type, the experts' outputs and their
    weighted sum in fp32."""

    def __init__(self, device, cfg: MoEConfig, *, max_tokens: int, n_local: int | None = None, first_expert: int = 0,
                 group: int = 128, scale_dtype: torch.dtype = torch.float16, zero_points: bool = False):
        self.cfg = cfg
        self.first_expert = int(first_expert)
        self.n_local = cfg.n_routed_experts - self.first_expert if n_local is None else int(n_local)
        if self.first_expert < 0 or self.n_local < 1 or self.first_expert + self.n_local > cfg.n_routed_experts:
            raise ValueError(f"experts [{self.first_expert}, {self.first_expert + self.n_local}) are not among the "
                             f"{cfg.n_routed_experts} of the router")
        # routing and the final cast run on a context without resident FP8 experts
        self._ctx = ExpertContext(device, cfg, n_slots=0, max_tokens=max_tokens, max_rows=1)
        self.device = self._ctx.device
        self.max_tokens = int(max_tokens)
        H, I = cfg.hidden_size, cfg.moe_intermediate_size
        kw = dict(group=group, scale_dtype=scale_dtype, zero_points=zero_points, device=self.device)
        self.up_gate = Int4Weight.empty(self.n_local, 2 * I, H, swiglu=True, **kw)
        self.down = Int4Weight.empty(self.n_local, H, I, **kw)
        self._shared = None
        self._kw = kw

    def close(self) -> None:
        self._ctx.close()

    # -- residency ---------------------------------------------------------------------
    def load_expert(self, expert_id: int, up_gate, down) -> None:
        """Expert ``expert_id`` (-1: the shared expert) from ``(q, scale, zero)`` of its stacked up and gate
        ``[2 I, H]`` and of its down ``[H, I]`` weight, as ``quantize_int4`` returns them."""
        if expert_id == -1:
            if self._shared is None:
                H, I = self.cfg.hidden_size, self.cfg.moe_intermediate_size
                self._shared = (Int4Weight.empty(1, 2 * I, H, swiglu=True, **self._kw),
                                Int4Weight.empty(1, H, I, **self._kw))
            ug, dn, at = *self._shared, 0
        else:
            ug, dn, at = self.up_gate, self.down, int(expert_id) - self.first_expert
            if not 0 <= at < self.n_local:
                raise ValueError(f"expert {expert_id} is not held here")
        ug.load(at, *up_gate)
        dn.load(at, *down)

    def upload_expert(self, expert_id: int, w_up, w_up_scale, w_gate, w_gate_scale, w_down, w_down_scale) -> None:
        """Quantise one expert of the reference's FP8 format (E4M3 weights, 128 x 128 ``scale_inv``) to 4 bits."""
        def fp32(w, s):
            w = torch.as_tensor(w)
            w = (w.view(torch.uint8) if w.dtype == torch.float8_e4m3fn else w).to(self.device)
            # the reference node reads the bytes 0x7F / 0xFF as +-448 (backend/fp8_lut_v2.cc:59-61)
            w = torch.where((w & 0x7F) == 0x7F, w - 1, w)
            return dequant_fp8_weight_blockwise(w, torch.as_tensor(s).to(self.device), self.cfg.block_size)

        kw = dict(group=self._kw["group"], symmetric=not self._kw["zero_points"],
                  scale_dtype=self._kw["scale_dtype"])
        up_gate = torch.cat([fp32(w_up, w_up_scale), fp32(w_gate, w_gate_scale)])
        self.load_expert(expert_id, quantize_int4(up_gate, **kw), quantize_int4(fp32(w_down, w_down_scale), **kw))

    # -- the layer ---------------------------------------------------------------------
    def route(self, x, gate_weight, bias, *, resident=None, top_k=None, return_aux=False):
        return self._ctx.route(x, gate_weight, bias, resident=resident, top_k=top_k, return_aux=return_aux)

    def cast_extra(self, extra, *, residual=None, out_dtype=torch.bfloat16, out=None):
        return self._ctx.cast_extra(extra, residual=residual, out_dtype=out_dtype, out=out)

    def _check(self, x):
        x = self._ctx._check_x(x)
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"experts in 4 bits take float16 or bfloat16 rows, got {x.dtype}")
        return x

    def _shared_rows(self, x):
        if self._shared is None:
            raise RuntimeError("no shared expert is resident")
        return grouped_int4(grouped_int4(x, self._shared[0]), self._shared[1], out_dtype=torch.float32)

    def _routed(self, x, topk_idx, topk_weight, extra, out_dtype):
        order = sort_routes(topk_idx, self.n_local, first_expert=self.first_expert)
        rows = sort_tokens(x, order)
        h = grouped_int4(rows, self.up_gate, order.offsets)
        y = grouped_int4(h, self.down, order.offsets, out_dtype=torch.float32)
        return unsort_tokens(y, order, topk_weight, residual=extra, out_dtype=out_dtype)

    def moe_routed(self, x, topk_idx, topk_weight, *, add_shared: bool = False, out_dtype=None):
        """Routed experts for given routes (+ the shared expert): ``ExpertContext.moe_routed``."""
        x = self._check(x)
        topk_idx = topk_idx.to(device=self.device)
        topk_weight = topk_weight.to(device=self.device, dtype=torch.float32)
        return self._routed(x, topk_idx, topk_weight, self._shared_rows(x) if add_shared else None,
                            out_dtype or x.dtype)

    def moe_routed_range(self, x, topk_idx, topk_weight, shared_begin: int, shared_end: int, *,
                         out_dtype=torch.float32):
        """Routed rows of every token, the shared expert on tokens ``[shared_begin, shared_end)``."""
        x = self._check(x)
        b, e = int(shared_begin), int(shared_end)
        if not 0 <= b <= e <= x.shape[0]:
            raise RuntimeError(f"invalid shared range [{b}, {e}) of {x.shape[0]} tokens")
        extra = None
        if e > b:
            extra = self._shared_rows(x[b:e])
            if e - b < x.shape[0]:
                whole = torch.zeros((x.shape[0], extra.shape[1]), dtype=torch.float32, device=self.device)
                whole[b:e] = extra
                extra = whole
        return self._routed(x, topk_idx, topk_weight, extra, out_dtype)

    def moe_layer(self, x, gate_weight, bias, *, resident=None, top_k=None, add_shared: bool = True, residual=None,
                  out_dtype=None, return_routes: bool = False):
        """Route, dispatch, experts and combine (+ shared expert, + residual): ``ExpertContext.moe_layer``."""
        x = self._check(x)
        if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
            raise RuntimeError("residual must match hidden in shape and dtype")
        idx, weight = self.route(x, gate_weight, bias, resident=resident, top_k=top_k)
        od = out_dtype or x.dtype
        if add_shared and residual is not None:
            part = self._routed(x, idx, weight, self._shared_rows(x), torch.float32)
            out = self.cast_extra(part, residual=residual.contiguous(), out_dtype=od)
        else:
            out = self._routed(x, idx, weight, self._shared_rows(x) if add_shared else residual, od)
        return (out, idx, weight) if return_routes else out

    def device_error(self) -> None:
        """Synchronise and raise if a kernel's bounded device-side wait gave up."""
        self._ctx.device_error()
        for w in (self.up_gate, self.down, *(self._shared or ())):
            w.device_error()
