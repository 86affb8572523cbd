"""The SwiGLU experts of the MoE layer on 8-bit operands: what `MoE.fp8_experts = True` runs.

forward:   tokens quantised straight into the grouped layout -> 8-bit up projection -> SwiGLU (its inputs and its result
           kept in 8 bits) -> 8-bit down projection -> weighted combine.
backward:  the output gradients are quantised for the two input-gradient products; the weight gradients are 16-bit
           products of the output gradients with the values that the kept 8-bit activations stand for.
What stays alive between the passes is one byte per activation (and the 16-bit expert outputs that the router weights'
gradient needs), where the 16-bit layer keeps two.
"""

from __future__ import annotations

import torch

from .. import _native
from .._native import call, dtype_code, ptr, stream_ptr
from ..ops.swiglu import swiglu_packed
from . import _kernels as K


class _Held:
    """8-bit rows [rows, cols] on the device: one buffer with the values (row pitch: cols rounded up to 16) and, behind
    them, the scales; `values` and `scales` are addresses in it."""

    __slots__ = ("buffer", "rows", "cols", "values", "scales")

    def __init__(self, rows: int, cols: int, device: torch.device, buffer: torch.Tensor | None = None):
        size = rows * ((cols + 15) // 16 * 16)
        if buffer is None:
            scale_bytes = int(_native.lib().fma_b200_fp8_scale_bytes(rows, cols))
            buffer = torch.empty(size + scale_bytes, dtype=torch.uint8, device=device)
        self.buffer, self.rows, self.cols = buffer, rows, cols
        self.values = buffer.data_ptr()
        self.scales = self.values + size


def _quantize_rows(x: torch.Tensor, rows_used: int) -> _Held:
    held = _Held(*x.shape, x.device)
    call("fma_b200_fp8_quantize_rows", ptr(x), x.stride(0), dtype_code(x.dtype), held.rows, held.cols, rows_used, held.values,
         held.scales, stream_ptr(x.device))  # fmt: skip
    return held


def _few_rows(x: torch.Tensor, held, counts: torch.Tensor) -> torch.Tensor:
    E, N, K_ = held.shape
    values, scales = held.addresses
    out = torch.empty(x.size(0), N, dtype=x.dtype, device=x.device)
    call("fma_b200_fp8_few_rows", ptr(x), x.stride(0), dtype_code(x.dtype), x.size(0), values, scales, E, N, K_, ptr(counts),
         counts.element_size(), ptr(out), stream_ptr(x.device))  # fmt: skip
    return out


def _quantize_scatter(x: torch.Tensor, maps: K.RowMaps) -> _Held:
    T, H = x.shape
    held = _Held(maps.rows_cap, H, x.device)
    call("fma_b200_fp8_quantize_scatter", ptr(x), dtype_code(x.dtype), T, H, maps.top_k, ptr(maps.row_of_slot),
         ptr(maps.slot_of_row), ptr(maps.pad_offsets), maps.num_experts, maps.rows_cap, held.values, held.scales,
         stream_ptr(x.device))  # fmt: skip
    return held


def _used(maps: K.RowMaps) -> int:
    """Address of the number of layout rows in use."""
    return maps.pad_offsets.data_ptr() + 4 * maps.num_experts


def _product(a: _Held, w_values: int, w_scales: int, cols: int, dtype, maps: K.RowMaps, dgrad: bool = False) -> torch.Tensor:
    """a . w^T per expert, or with `dgrad` a . w; `cols` of the result.  Its rows behind an expert's are written up to a
    multiple of 64 only, which is as far as anything reads them."""
    dev = a.buffer.device
    out = torch.empty(maps.rows_cap, cols, dtype=dtype, device=dev)
    name, N, K_ = ("fma_b200_fp8_gemm_dgrad", a.cols, cols) if dgrad else ("fma_b200_fp8_gemm", cols, a.cols)
    call(name, a.values, a.scales, maps.rows_cap, w_values, w_scales, maps.num_experts, N, K_,
         ptr(out), dtype_code(dtype), maps.rows_cap, ptr(maps.mtile_expert), None, None, _used(maps),
         ptr(maps.pad_offsets), ptr(maps.expert_count), stream_ptr(dev))  # fmt: skip
    return out


def _weight_gradient(d_rows: torch.Tensor, a: _Held, maps: K.RowMaps) -> torch.Tensor:
    """d_rows^T times the values that `a` stands for, per expert over its token rows."""
    E, N, dtype, dev = maps.num_experts, d_rows.size(1), d_rows.dtype, d_rows.device
    x = torch.empty(a.rows, a.cols, dtype=dtype, device=dev)
    call("fma_b200_fp8_dequantize", a.values, a.scales, 1, a.rows, a.cols, _used(maps), ptr(x), dtype_code(dtype),
         stream_ptr(dev))  # fmt: skip
    d_w = torch.empty(E, N, a.cols, dtype=dtype, device=dev)
    call("fma_b200_linear_wgrad", ptr(d_rows), ptr(x), ptr(d_w), dtype_code(dtype), a.rows, E, N, a.cols,
         ptr(maps.pad_offsets), ptr(maps.expert_count), stream_ptr(dev))  # fmt: skip
    return d_w


class Fp8SwigluExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, w_fc, w_proj, held_fc, held_proj, maps: K.RowMaps, keep: bool):
        """keep: a backward pass may follow (ctx.needs_input_grad says True under torch.no_grad as well)."""
        x, weights = x.contiguous(), weights.contiguous()
        T, H = x.shape
        I, dev, cap = held_proj.shape[-1], x.device, maps.rows_cap
        x8 = _quantize_scatter(x, maps)
        fc, proj = held_fc.addresses, held_proj.addresses
        pre = _product(x8, *fc, 2 * I, x.dtype, maps)
        act8, up8, gate8 = _Held(cap, I, dev), *((_Held(cap, I, dev) if keep else None) for _ in range(2))
        at = (gate8.values, gate8.scales, up8.values, up8.scales) if keep else (None,) * 4
        call("fma_b200_swiglu_fp8_forward", pre.data_ptr() + I * pre.element_size(), 2 * I, ptr(pre), 2 * I, None, I,
             dtype_code(x.dtype), cap, I, _used(maps), *at, act8.values, act8.scales, stream_ptr(dev))  # fmt: skip
        del pre
        out = _product(act8, *proj, H, x.dtype, maps)
        y = K.combine(out, weights, maps, T)
        if keep:
            ctx.save_for_backward(x8.buffer, up8.buffer, gate8.buffer, act8.buffer, out, weights, held_fc.buffer, held_proj.buffer)
            ctx.scales_at = fc[1] - fc[0], proj[1] - proj[0]  # where the weights' scales begin
        ctx.maps, ctx.sizes, ctx.dtype = maps, (T, H, I), x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # what follows leaves no graph: the experts' part of a second derivative would be lost
            raise RuntimeError("fp8_experts: the experts can be differentiated once only (create_graph=False)")
        x8, up8, gate8, act8, out, weights, fc, proj = ctx.saved_tensors
        fc, proj = ((b.data_ptr(), b.data_ptr() + at) for b, at in zip((fc, proj), ctx.scales_at))
        maps, (T, H, I), dtype, dev = ctx.maps, ctx.sizes, ctx.dtype, dy.device
        cap, used = maps.rows_cap, _used(maps)
        x8 = _Held(cap, H, dev, x8)
        up8, gate8, act8 = (_Held(cap, I, dev, b) for b in (up8, gate8, act8))
        need_x, need_w, need_fc, need_proj = ctx.needs_input_grad[:4]
        with torch.cuda.device(dev):
            d_out, d_w = K.combine_backward(dy.contiguous(), out, weights, maps, need_w)
            d_x = d_w_fc = d_w_proj = None
            if need_proj:
                d_w_proj = _weight_gradient(d_out, act8, maps)
            if need_x or need_fc:
                d_act = _product(_quantize_rows(d_out, used), *proj, I, dtype, maps, dgrad=True)
                d_pre = torch.empty(cap, 2 * I, dtype=dtype, device=dev)
                # the same pass quantises d_pre where its blocks of 128 columns do not straddle up and gate
                d_pre8 = _Held(cap, 2 * I, dev) if need_x and I % 128 == 0 else None
                at = (d_pre8.values, d_pre8.scales) if d_pre8 else (None, None)
                call("fma_b200_swiglu_fp8_backward", gate8.values, gate8.scales, up8.values, up8.scales, ptr(d_act), I,
                     d_pre.data_ptr() + I * d_pre.element_size(), 2 * I, ptr(d_pre), 2 * I, dtype_code(dtype), cap, I, used, *at,
                     stream_ptr(dev))  # fmt: skip
                if need_fc:
                    d_w_fc = _weight_gradient(d_pre, x8, maps)
                if need_x:
                    d_xg = _product(d_pre8 or _quantize_rows(d_pre, used), *fc, H, dtype, maps, dgrad=True)
                    d_x = K.scatter_backward(d_xg, maps, T)
        return d_x, d_w, d_w_fc, d_w_proj, None, None, None, None


def few(rows: int, held_proj) -> bool:
    """Whether `few_tokens` is the faster way for this many routed rows."""
    E, H, I = held_proj.shape
    return rows > 0 and _native.binding().few(rows, E, [(2 * I, H), (H, I)])


def few_tokens(x, weights, held_fc, held_proj, maps: K.RowMaps) -> torch.Tensor:
    """The layer without gradients for a few rows per expert; `maps` sorted with row_align = 1."""
    T = x.size(0)
    xg = K.scatter(x.contiguous(), maps)[: T * maps.top_k]
    act = swiglu_packed(_few_rows(xg, held_fc, maps.expert_count))
    out = _few_rows(act, held_proj, maps.expert_count)
    return K.combine(out, weights.contiguous(), maps, T)
