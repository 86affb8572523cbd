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

from .._native import call, dtype_code
from ..ops.fp8 import (
    _FEW_ROWS,
    _FEW_ROWS_MAX_WIDTH,
    Fp8Weight,
    _dequantize,
    _few_rows,
    _pitch,
    _quantize_rows,
    _scale_bytes,
    ptr,
    stream_ptr,
)
from ..ops.swiglu import swiglu_packed
from . import _kernels as K


def _quantize_scatter(x: torch.Tensor, maps: K.RowMaps):
    T, H = x.shape
    values = torch.empty(maps.rows_cap, _pitch(H), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(_scale_bytes(maps.rows_cap, H), dtype=torch.uint8, device=x.device)
    call("fma_b200_fp8_quantize_scatter", ptr(x), dtype_code(x.dtype), T, H, maps.top_k, ptr(maps.row_of_slot),
         ptr(maps.slot_of_row), ptr(maps.pad_offsets), maps.num_experts, maps.rows_cap, ptr(values), ptr(scales),
         stream_ptr(x.device))  # fmt: skip
    return values, scales


def _product(values, scales, w_values, w_scales, N: int, K_: int, dtype, maps: K.RowMaps) -> torch.Tensor:
    out = torch.empty(maps.rows_cap, N, dtype=dtype, device=values.device)
    call("fma_b200_fp8_gemm", ptr(values), ptr(scales), maps.rows_cap, ptr(w_values), ptr(w_scales), maps.num_experts, N,
         K_, ptr(out), dtype_code(dtype), maps.rows_cap, ptr(maps.mtile_expert), None, None,
         ptr(maps.pad_offsets[maps.num_experts :]), stream_ptr(values.device))  # fmt: skip
    return out


def _empty8(rows: int, cols: int, device):
    return (torch.empty(rows, _pitch(cols), dtype=torch.float8_e4m3fn, device=device),
            torch.empty(_scale_bytes(rows, cols), dtype=torch.uint8, device=device))  # fmt: skip


class Fp8SwigluExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, w_fc, w_proj, held_fc: Fp8Weight, held_proj: Fp8Weight, maps: K.RowMaps):
        x, weights = x.contiguous(), weights.contiguous()
        T, H = x.shape
        I, dev, cap = held_proj.shape[-1], x.device, maps.rows_cap
        used = ptr(maps.pad_offsets[maps.num_experts :])
        x8, x_scales = _quantize_scatter(x, maps)
        pre = _product(x8, x_scales, held_fc.values, held_fc.scales, 2 * I, H, x.dtype, maps)
        keep = any(ctx.needs_input_grad)
        up8, up_scales = _empty8(cap, I, dev) if keep else (None, None)
        gate8, gate_scales = _empty8(cap, I, dev) if keep else (None, None)
        act8, act_scales = _empty8(cap, I, dev)
        call("fma_b200_swiglu_fp8_forward", pre.data_ptr() + I * pre.element_size(), 2 * I, ptr(pre), 2 * I, None, I,
             dtype_code(x.dtype), cap, I, used, ptr(gate8), ptr(gate_scales), ptr(up8), ptr(up_scales), ptr(act8),
             ptr(act_scales), stream_ptr(dev))  # fmt: skip
        del pre
        out = _product(act8, act_scales, held_proj.values, held_proj.scales, H, I, x.dtype, maps)
        y = K.combine(out, weights, maps, T)
        ctx.save_for_backward(x8, x_scales, up8, up_scales, gate8, gate_scales, act8, act_scales, out, weights,
                              held_fc.transposed, held_fc.transposed_scales, held_proj.transposed,
                              held_proj.transposed_scales)  # fmt: skip
        ctx.maps, ctx.sizes, ctx.dtype = maps, (T, H, I), x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        (x8, x_scales, up8, up_scales, gate8, gate_scales, act8, act_scales, out, weights, fc_t, fc_t_scales, proj_t,
         proj_t_scales) = ctx.saved_tensors  # fmt: skip
        maps, (T, H, I), dtype, dev = ctx.maps, ctx.sizes, ctx.dtype, dy.device
        E, cap = maps.num_experts, maps.rows_cap
        used = maps.pad_offsets[E:]
        need_x, need_w, need_fc, need_proj = ctx.needs_input_grad[:4]
        d_out, d_w = K.combine_backward(dy.contiguous(), out, weights, maps, need_w)
        d_x = d_w_fc = d_w_proj = None
        if need_proj:
            act = _dequantize(act8, act_scales, 1, cap, (cap, I), dtype, used)
            d_w_proj = K.gemm_wgrad(d_out, act, E, maps.pad_offsets)
            del act
        if need_x or need_fc:
            d8, d_scales = _quantize_rows(d_out, used)
            d_act = _product(d8, d_scales, proj_t, proj_t_scales, I, H, dtype, maps)
            d_pre = torch.empty(cap, 2 * I, dtype=dtype, device=dev)
            call("fma_b200_swiglu_fp8_backward", ptr(gate8), ptr(gate_scales), ptr(up8), ptr(up_scales), ptr(d_act), I,
                 d_pre.data_ptr() + I * d_pre.element_size(), 2 * I, ptr(d_pre), 2 * I, dtype_code(dtype), cap, I, ptr(used),
                 stream_ptr(dev))  # fmt: skip
            if need_fc:
                xg = _dequantize(x8, x_scales, 1, cap, (cap, H), dtype, used)
                d_w_fc = K.gemm_wgrad(d_pre, xg, E, maps.pad_offsets)
                del xg
            if need_x:
                d8, d_scales = _quantize_rows(d_pre, used)
                d_xg = _product(d8, d_scales, fc_t, fc_t_scales, H, 2 * I, dtype, maps)
                d_x = K.scatter_backward(d_xg, maps, T)
        return d_x, d_w, d_w_fc, d_w_proj, None, None, None


def few(rows: int, held_proj: Fp8Weight) -> bool:
    """Whether `few_tokens` is the faster way for this many routed rows."""
    E, H, I = held_proj.shape
    return 0 < rows <= _FEW_ROWS * E and max(H, I) <= _FEW_ROWS_MAX_WIDTH


def few_tokens(x, weights, held_fc: Fp8Weight, held_proj: Fp8Weight, maps: K.RowMaps) -> torch.Tensor:
    """The layer without gradients for a few rows per expert; `maps` sorted with row_align = 1."""
    T, H = x.shape
    I, E, R = held_proj.shape[-1], maps.num_experts, T * maps.top_k
    xg = K.scatter(x.contiguous(), maps)[:R]
    act = swiglu_packed(_few_rows(xg, held_fc, E, 2 * I, H, maps.expert_count))
    out = _few_rows(act, held_proj, E, H, I, maps.expert_count)
    return K.combine(out, weights.contiguous(), maps, T)
