"""Operators on 8-bit values: storing tensors in e4m3 with one power-of-two scale per block of 128, linear maps whose
operands are held that way, and SwiGLU that keeps its inputs in 8 bits for the backward pass.

The format: a block is 128 consecutive columns of one row, or 128 x 128 for weights.  Its scale is 2^e with e the
smallest integer such that the block's largest finite magnitude is at most 448 * 2^e; a value is held as
e4m3(x / 2^e), rounded to nearest even.  Infinities and NaN are held as NaN.

In the linear maps the forward product and the input gradient are products of 8-bit operands (activations, output
gradients and weights are quantised), accumulated in fp32 and rounded once to the 16-bit type.  The weight gradient
sums over tokens, where 1 x 128 blocks do not help: it is the 16-bit product of the output gradient with the values
that the 8-bit activations stand for.  The 8-bit activations are all that the forward pass keeps.
"""

from __future__ import annotations

import contextlib

import torch

from .. import _native
from .._native import call, dtype_code
from .swiglu import _as_rows

_SAME_DEVICE = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes `device` current for the calls inside; nothing to do (and to pay for) if it already is."""
    return _SAME_DEVICE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_ptr(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _pitch(cols: int) -> int:
    return (cols + 15) // 16 * 16


def _scale_bytes(rows: int, cols: int) -> int:
    return (cols + 511) // 512 * ((rows + 127) // 128) * 512


def _rows_2d(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, cols] with unit column stride, rows of a single pitch and 16-byte aligned rows; a copy if it has to be."""
    cols, size = x.size(-1), x.element_size()
    if x.dim() == 2 and x.stride(1) == 1 and x.data_ptr() % 16 == 0:
        pitch = x.stride(0)
        if pitch >= cols and pitch * size % 16 == 0:
            return x
    if x.dim() == 1:
        x = x.unsqueeze(0)
    x = _as_rows(x)
    pitch = x.stride(-2) if x.size(-2) > 1 or x.dim() > 2 else cols
    rows = x.numel() // cols
    if pitch < cols or pitch * size % 16 != 0 or x.data_ptr() % 16 != 0:
        x, pitch = x.clone(memory_format=torch.contiguous_format), cols
    return x.as_strided((rows, cols), (pitch, 1))


def _check_cols(name: str, cols: int) -> None:
    if cols < 8 or cols % 8 != 0:
        raise RuntimeError(f"{name}: the width must be a positive multiple of 8, got {cols}")


class _Held:
    """8-bit rows [rows, cols] on the device: one buffer with the values (row pitch: cols rounded up to 16) and, behind
    them, the scales in the order in which the tensor cores read them."""

    __slots__ = ("buffer", "rows", "cols", "values", "scales")

    def __init__(self, rows: int, cols: int, device: torch.device, buffer: torch.Tensor | None = None):
        size = rows * _pitch(cols)
        if buffer is None:
            buffer = torch.empty(size + _scale_bytes(rows, cols), dtype=torch.uint8, device=device)
        self.buffer, self.rows, self.cols = buffer, rows, cols
        self.values = buffer.data_ptr()
        self.scales = self.values + size


class Fp8Blocks:
    """A tensor held in 8 bits, with the shape and dtype it came from: e4m3 values and a scale per 128 columns of a row."""

    __slots__ = ("_held", "shape", "dtype")

    def __init__(self, held: _Held, shape: torch.Size, dtype: torch.dtype):
        self._held, self.shape, self.dtype = held, shape, dtype

    @property
    def device(self) -> torch.device:
        return self._held.buffer.device

    @property
    def nbytes(self) -> int:
        return self._held.buffer.numel()

    @property
    def values(self) -> torch.Tensor:
        """The e4m3 values without their scales, [rows, cols]."""
        h = self._held
        pitch = _pitch(h.cols)
        return h.buffer[: h.rows * pitch].view(torch.float8_e4m3fn).view(h.rows, pitch)[:, : h.cols]

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values it stands for, rounded to `dtype` (default: the type it was made from)."""
        h = self._held
        return _dequantize(h.values, h.scales, 1, h.rows, self.shape, dtype or self.dtype, h.buffer.device)


class Fp8Weight:
    """A weight [N, K] or [E, N, K] held in 8 bits with a scale per 128 x 128 block: e4m3 `values` (row pitch: K rounded
    up to 16) and `scales` in the order in which the tensor cores read them.  `transposed` is the second copy that input
    gradients read, or None."""

    __slots__ = ("values", "scales", "transposed", "transposed_scales", "shape", "dtype", "device")

    def __init__(self, values, scales, transposed, transposed_scales, shape: torch.Size, dtype: torch.dtype):
        self.values, self.scales = values, scales
        self.transposed, self.transposed_scales = transposed, transposed_scales
        self.shape, self.dtype, self.device = shape, dtype, values.device

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values it stands for, rounded to `dtype` (default: the type it was made from)."""
        experts = self.shape[0] if len(self.shape) == 3 else 1
        return _dequantize(self.values.data_ptr(), self.scales.data_ptr(), experts, self.shape[-2], self.shape,
                           dtype or self.dtype, self.values.device)  # fmt: skip


def _dequantize(values: int, scales: int, batch: int, rows: int, shape, dtype, device, rows_used: int | None = None) -> torch.Tensor:
    code = dtype_code(dtype)
    out = torch.empty(shape, dtype=dtype, device=device)
    if rows:
        with _on(device):
            call("fma_b200_fp8_dequantize", values, scales, batch, rows, shape[-1], rows_used, out.data_ptr(), code,
                 stream_ptr(device))  # fmt: skip
    return out


def _quantize_rows(x: torch.Tensor, rows_used: int | None = None) -> _Held:
    """x [rows, cols] as _rows_2d gives it."""
    rows, cols = x.shape
    held = _Held(rows, cols, x.device)
    call("fma_b200_fp8_quantize_rows", x.data_ptr(), x.stride(0), dtype_code(x.dtype), rows, cols, rows_used, held.values,
         held.scales, stream_ptr(x.device))  # fmt: skip
    return held


def quantize_fp8(x: torch.Tensor) -> Fp8Blocks:
    """Holds x [..., cols] (float32, bfloat16 or float16) in 8 bits with a scale per 128 columns of a row: a quarter or
    half of its bytes.  cols must be a multiple of 8.  `.dequantize()` gives the values back."""
    _native.require_cuda(x)
    dtype_code(x.dtype)
    if x.dim() == 0:
        raise RuntimeError("quantize_fp8: x needs at least one dimension")
    _check_cols("quantize_fp8", x.size(-1))
    with _on(x.device):
        held = _quantize_rows(_rows_2d(x.detach()))
    return Fp8Blocks(held, x.shape, x.dtype)


def quantize_fp8_weight(weight: torch.Tensor, transpose: bool = False) -> Fp8Weight:
    """Holds weight [N, K] or [E, N, K] in 8 bits with a scale per 128 x 128 block.  With `transpose` also the
    transposed copy that the input gradient of a linear map needs.  N and K must be multiples of 8."""
    _native.require_cuda(weight)
    code = dtype_code(weight.dtype)
    if weight.dim() not in (2, 3):
        raise RuntimeError(f"quantize_fp8_weight: weight must be [N, K] or [experts, N, K], got {tuple(weight.shape)}")
    _check_cols("quantize_fp8_weight", weight.size(-1))
    _check_cols("quantize_fp8_weight", weight.size(-2))
    w = weight.detach().contiguous()
    if w.data_ptr() % 16 != 0:
        w = w.clone()
    E, (N, K) = (w.size(0) if w.dim() == 3 else 1), w.shape[-2:]
    dev = w.device
    values = torch.empty(E, N, _pitch(K), dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(_scale_bytes(E * ((N + 127) // 128) * 128, K), dtype=torch.uint8, device=dev)
    turned = turned_scales = None
    if transpose:
        turned = torch.empty(E, K, _pitch(N), dtype=torch.float8_e4m3fn, device=dev)
        turned_scales = torch.empty(_scale_bytes(E * ((K + 127) // 128) * 128, N), dtype=torch.uint8, device=dev)
    with _on(dev):
        call("fma_b200_fp8_quantize_weight", ptr(w), code, E, N, K, ptr(values), ptr(scales), ptr(turned),
             ptr(turned_scales), stream_ptr(dev))  # fmt: skip
    return Fp8Weight(values, scales, turned, turned_scales, weight.shape, weight.dtype)


class GroupMaps:
    """Where rows that are grouped by expert without alignment lie in the 256-aligned layout.  One int32 buffer on the
    device; the attributes are addresses in it."""

    __slots__ = ("buffer", "offsets", "pad_offsets", "used", "used_all", "group_rows", "tile_expert", "tile_row", "tile_rows",
                 "layout_rows", "num_experts")  # fmt: skip

    def __init__(self, expert_frequency: torch.Tensor, rows: int):
        E, dev = expert_frequency.numel(), expert_frequency.device
        self.num_experts = E
        self.layout_rows = (rows + 255) // 256 * 256 + 256 * min(E, rows)
        tiles = self.layout_rows // 128
        self.buffer = torch.empty(3 * E + 3 + 3 * tiles, dtype=torch.int32, device=dev)
        at = self.buffer.data_ptr()
        self.pad_offsets = at
        self.used = at + 4 * E  # rows of the layout that experts use, and with the rows of no expert
        self.used_all = at + 4 * (E + 1)
        self.offsets = at + 4 * (E + 2)
        self.group_rows = at + 4 * (2 * E + 3)
        self.tile_expert = at + 4 * (3 * E + 3)
        self.tile_row = self.tile_expert + 4 * tiles
        self.tile_rows = self.tile_row + 4 * tiles
        call("fma_b200_fp8_group_maps", expert_frequency.data_ptr(), expert_frequency.element_size(), E, rows,
             self.layout_rows, self.offsets, self.pad_offsets, self.group_rows, self.tile_expert, self.tile_row,
             self.tile_rows, stream_ptr(dev))  # fmt: skip


def _quantize_groups(x: torch.Tensor, maps: GroupMaps, copy: torch.Tensor | None = None) -> _Held:
    rows, cols = x.shape
    held = _Held(maps.layout_rows, cols, x.device)
    call("fma_b200_fp8_quantize_groups", x.data_ptr(), x.stride(0), dtype_code(x.dtype), rows, cols, maps.offsets,
         maps.pad_offsets, maps.num_experts, maps.layout_rows, held.values, held.scales, ptr(copy),
         stream_ptr(x.device))  # fmt: skip
    return held


def _product(a: _Held, w_values: torch.Tensor, w_scales: torch.Tensor, E: int, N: int, dtype: torch.dtype, out_rows: int,
             maps: GroupMaps | None) -> torch.Tensor:
    """[out_rows, N] = rows of `a` times the rows of the weight copy, both reduced over a's columns."""
    dev = a.buffer.device
    out = torch.empty(out_rows, N, dtype=dtype, device=dev)
    tables = (None, None, None, None)
    if maps is not None:
        tables = (maps.tile_expert, maps.tile_row, maps.tile_rows, maps.used_all)
    call("fma_b200_fp8_gemm", a.values, a.scales, a.rows, w_values.data_ptr(), w_scales.data_ptr(), E, N, a.cols,
         out.data_ptr(), dtype_code(dtype), out_rows, *tables, stream_ptr(dev))  # fmt: skip
    return out


_FEW_ROWS_MAX_WIDTH = 1 << 16


def _few(rows: int, E: int, K: int) -> bool:
    """Whether the product that reads x itself, in one launch, is the faster way.  Above, x is quantised by a launch of its
    own.  Measured with weights of 4096 x 4096: 5.8 us against 7.4 for one row, 7.6 / 7.9 for 16, 12.0 / 8.7 for 32; of
    14336 x 4096: 13.8 / 16.6, 17.9 / 17.4, 34.2 / 18.4; 128 experts of 1536 x 2048: 81 / 94 for 8 rows each, 101 / 95 for 16."""
    return rows <= (16 if E == 1 else 12 * E) and K <= _FEW_ROWS_MAX_WIDTH


def _few_rows(x: torch.Tensor, held: Fp8Weight, E: int, N: int, K: int, expert_frequency) -> torch.Tensor:
    dev, dtype, rows = x.device, x.dtype, x.size(0)
    out = torch.empty(rows, N, dtype=dtype, device=dev)
    counts, index_bytes = (None, 4) if expert_frequency is None else (expert_frequency.data_ptr(), expert_frequency.element_size())
    call("fma_b200_fp8_few_rows", x.data_ptr(), x.stride(0), dtype_code(dtype), rows, held.values.data_ptr(),
         held.scales.data_ptr(), E, N, K, counts, index_bytes, out.data_ptr(), stream_ptr(dev))  # fmt: skip
    return out


def _forward(x: torch.Tensor, held: Fp8Weight, expert_frequency):
    """The product, the row maps and the 8-bit rows it ran on."""
    N = held.shape[-2]
    if expert_frequency is None:
        maps, rows = None, _quantize_rows(x)
    else:
        maps = GroupMaps(expert_frequency, x.size(0))
        rows = _quantize_groups(x, maps)
    E = 1 if maps is None else maps.num_experts
    return _product(rows, held.values, held.scales, E, N, x.dtype, x.size(0), maps), maps, rows


class _LinearFp8(torch.autograd.Function):
    """weight: the 16-bit parameter (or None: no gradient of it); held: its 8-bit form."""

    @staticmethod
    def forward(ctx, x, weight, held: Fp8Weight, expert_frequency):
        N, K = held.shape[-2:]
        out, maps, rows = _forward(x, held, expert_frequency)
        ctx.maps, ctx.sizes, ctx.dtype = maps, (x.size(0), N, K), x.dtype
        kept = [rows.buffer if ctx.needs_input_grad[1] else None]
        kept += [held.transposed, held.transposed_scales] if ctx.needs_input_grad[0] else [None, None]
        ctx.save_for_backward(*kept)
        return out

    @staticmethod
    def backward(ctx, d_out):
        buffer, turned, turned_scales = ctx.saved_tensors
        rows, N, K = ctx.sizes
        maps, dtype, dev = ctx.maps, ctx.dtype, d_out.device
        want_x, want_w = ctx.needs_input_grad[:2]
        d_x = d_w = None
        with _on(dev):
            d_out = _rows_2d(d_out)
            if maps is None:
                E, layout, used = 1, rows, None
                d_rows = d_out.contiguous()
                d8 = _quantize_rows(d_out) if want_x else None
            else:
                E, layout, used = maps.num_experts, maps.layout_rows, maps.used
                # the same pass lays the rows out for the weight gradient
                d_rows = torch.empty(layout, N, dtype=dtype, device=dev) if want_w else None
                d8 = _quantize_groups(d_out, maps, d_rows)
            if want_x:
                d_x = _product(d8, turned, turned_scales, E, K, dtype, rows, maps)
            if want_w:
                x8 = _Held(layout, K, dev, buffer)
                x_rows = _dequantize(x8.values, x8.scales, 1, layout, (layout, K), dtype, dev, used)
                if maps is None:
                    ends = torch.arange(0, 2 * rows, rows, dtype=torch.int32, device=dev)
                    segments, d_w = (ends.data_ptr(), None), torch.empty(N, K, dtype=dtype, device=dev)
                else:
                    segments, d_w = (maps.pad_offsets, maps.group_rows), torch.empty(E, N, K, dtype=dtype, device=dev)
                call("fma_b200_linear_wgrad", d_rows.data_ptr(), x_rows.data_ptr(), d_w.data_ptr(), dtype_code(dtype), layout,
                     E, N, K, *segments, stream_ptr(dev))  # fmt: skip
        return d_x, d_w, None, None


def _check_linear(name: str, x, weight, expert_frequency, quantized) -> None:
    held = weight if isinstance(weight, Fp8Weight) else quantized
    parameter = None if isinstance(weight, Fp8Weight) else weight
    if held is not None and not isinstance(held, Fp8Weight):
        raise RuntimeError(f"{name}: quantized must be what quantize_fp8_weight returns")
    if held is not None and parameter is not None and held.shape != parameter.shape:
        raise RuntimeError(f"{name}: quantized has shape {tuple(held.shape)}, weight {tuple(parameter.shape)}")
    shape = weight.shape
    _native.require_cuda(x, parameter, expert_frequency)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"{name}: x must be bfloat16 or float16, got {x.dtype}")
    if parameter is not None and parameter.dtype != x.dtype:
        raise RuntimeError(f"{name}: x is {x.dtype}, weight {parameter.dtype}")
    grouped = expert_frequency is not None
    if len(shape) != (3 if grouped else 2):
        raise RuntimeError(f"{name}: unexpected weight shape {tuple(shape)}")
    if x.dim() < 1 or x.size(-1) != shape[-1]:
        raise RuntimeError(f"{name}: x {tuple(x.shape)} does not fit a weight of shape {tuple(shape)}")
    if grouped:
        if x.dim() != 2:
            raise RuntimeError(f"{name}: x must be [rows, {shape[-1]}], got {tuple(x.shape)}")
        if expert_frequency.numel() != shape[0] or expert_frequency.dim() != 1:
            raise RuntimeError(f"{name}: expert_frequency must hold one count for each of the {shape[0]} experts")
        if not 1 <= shape[0] <= 1024:
            raise RuntimeError(f"{name}: 1 to 1024 experts, got {shape[0]}")
        if expert_frequency.dtype not in (torch.int32, torch.uint32, torch.int64):
            raise RuntimeError(f"{name}: expert_frequency must be int32, uint32 or int64, got {expert_frequency.dtype}")
    for t in (weight, held, expert_frequency):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name}: x is on {x.device}, another argument on {t.device}")
    _check_cols(name, shape[-2])
    _check_cols(name, shape[-1])


def _linear(name: str, x, weight, expert_frequency, quantized):
    _check_linear(name, x, weight, expert_frequency, quantized)
    if isinstance(weight, Fp8Weight):
        held, parameter = weight, None
    else:
        held, parameter = quantized, weight
    shape, dims, grouped = weight.shape, x.dim(), expert_frequency is not None
    N, K = shape[-2:]
    rows = x.size(0) if dims == 2 else x.numel() // K
    grad = torch.is_grad_enabled()
    grad_x = grad and x.requires_grad
    grad_w = grad and parameter is not None and parameter.requires_grad
    if grad_x and held is not None and held.transposed is None:
        raise RuntimeError(f"{name}: the gradient of x needs quantize_fp8_weight(weight, transpose=True)")
    if rows == 0:
        out = x.new_empty(*x.shape[:-1], N)
        if grad_x or grad_w:  # keep the graph: every gradient is zero
            out = out + (x.sum() if grad_x else 0) * 0 + (parameter.sum() if grad_w else 0) * 0
        return out
    with _on(x.device):
        if held is None:
            held = quantize_fp8_weight(parameter, transpose=grad_x)
        x2 = _rows_2d(x if dims == 2 else x.reshape(rows, K))
        if grouped and not expert_frequency.is_contiguous():
            expert_frequency = expert_frequency.contiguous()
        if grad_x or grad_w:
            out = _LinearFp8.apply(x2, parameter, held, expert_frequency)
        else:
            E = shape[0] if grouped else 1
            if _few(rows, E, K):
                out = _few_rows(x2, held, E, N, K, expert_frequency)
            else:
                out = _forward(x2, held, expert_frequency)[0]
    return out if dims == 2 else out.view(*x.shape[:-1], N)


def linear_fp8(x: torch.Tensor, weight: torch.Tensor | Fp8Weight, quantized: Fp8Weight | None = None) -> torch.Tensor:
    """x [..., K] times weight [N, K] transposed, both taken in 8 bits; returns [..., N] in x's type (bfloat16 or
    float16).  `weight` is a parameter, quantised in the call, or an Fp8Weight (serving: no gradient of the weight).
    `quantized` is the 8-bit form of `weight` where the caller has it already, for example once per step for several
    micro-batches.  Differentiable in x and in a `weight` that is a tensor; rounding to 8 bits passes gradients
    through unchanged.  The forward pass keeps x in 8 bits only.  N and K must be multiples of 8."""
    return _linear("linear_fp8", x, weight, None, quantized)


def grouped_linear_fp8(
    x: torch.Tensor,
    weight: torch.Tensor | Fp8Weight,
    expert_frequency: torch.Tensor,
    quantized: Fp8Weight | None = None,
) -> torch.Tensor:
    """linear_fp8 with a weight per expert [E, N, K]: x [rows, K] holds expert_frequency[e] consecutive rows for expert e,
    in expert order and without alignment, as in `Experts.cuda_forward`.  The counts stay on the device.  Rows behind
    the last expert's (the counts sum to less than `rows`) give zeros; counts that overshoot are cut off."""
    return _linear("grouped_linear_fp8", x, weight, expert_frequency, quantized)


def _swiglu_fp8(gate: torch.Tensor, up: torch.Tensor, keep: bool):
    """out, and with `keep` gate and up in 8 bits: one buffer of twice their rows."""
    shape, cols = gate.shape, gate.size(-1)
    gate, up = _rows_2d(gate), _rows_2d(up)
    rows, dev = gate.size(0), gate.device
    out = torch.empty(shape, dtype=gate.dtype, device=dev)
    kept, at = None, (None, None, None, None)
    if keep:
        size, scale_bytes = rows * _pitch(cols), _scale_bytes(rows, cols)
        kept = torch.empty(2 * (size + scale_bytes), dtype=torch.uint8, device=dev)
        first = kept.data_ptr()
        at = (first, first + 2 * size, first + size, first + 2 * size + scale_bytes)
    call("fma_b200_swiglu_fp8_forward", gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), out.data_ptr(), cols,
         dtype_code(gate.dtype), rows, cols, None, *at, None, None, stream_ptr(dev))  # fmt: skip
    return out, kept


class _SwigluFp8Checkpoint(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        out, kept = _swiglu_fp8(gate, up, True)
        ctx.save_for_backward(kept)
        ctx.shape = gate.shape
        return out

    @staticmethod
    def backward(ctx, d_out):
        (kept,) = ctx.saved_tensors
        cols, dev = ctx.shape[-1], d_out.device
        gate_grad = torch.empty(ctx.shape, dtype=d_out.dtype, device=dev)
        up_grad = torch.empty(ctx.shape, dtype=d_out.dtype, device=dev)
        with _on(dev):
            d_out = _rows_2d(d_out)
            rows = d_out.size(0)
            size, scale_bytes, first = rows * _pitch(cols), _scale_bytes(rows, cols), kept.data_ptr()
            call("fma_b200_swiglu_fp8_backward", first, first + 2 * size, first + size, first + 2 * size + scale_bytes,
                 d_out.data_ptr(), d_out.stride(0), gate_grad.data_ptr(), cols, up_grad.data_ptr(), cols,
                 dtype_code(d_out.dtype), rows, cols, None, stream_ptr(dev))  # fmt: skip
        return gate_grad, up_grad


def swiglu_fp8_checkpoint(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """`swiglu(gate, up)` that keeps gate and up in 8 bits between the passes: half the memory of a 16-bit SwiGLU, a
    quarter of an fp32 one.  The result is that of `swiglu`; the gradients are those at the values the 8-bit form
    stands for.  The last dimension must be a multiple of 8."""
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise RuntimeError("swiglu_fp8_checkpoint: gate and up must have the same shape, dtype and device")
    _native.require_cuda(gate, up)
    dtype_code(gate.dtype)
    if gate.dim() == 0:
        raise RuntimeError("swiglu_fp8_checkpoint: gate needs at least one dimension")
    _check_cols("swiglu_fp8_checkpoint", gate.size(-1))
    with _on(gate.device):
        if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
            return _SwigluFp8Checkpoint.apply(gate, up)
        return _swiglu_fp8(gate, up, False)[0]
