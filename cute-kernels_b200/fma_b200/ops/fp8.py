"""Operators on 8-bit values: storing tensors in e4m3 with one power-of-two scale per block of 128, linear maps whose
operands are held that way, and SwiGLU that keeps its inputs in 8 bits for the backward pass.

The format: a block is 128 consecutive columns of one row, or 128 x 128 for weights.  Its scale is 2^e with e the
smallest integer such that the block's largest finite magnitude is at most 448 * 2^e; a value is held as
e4m3(x / 2^e), rounded to nearest even.  Infinities and NaN are held as NaN.

In the linear maps the forward product and the input gradient are products of 8-bit operands (activations, output
gradients and weights are quantised), accumulated in fp32 and rounded once to the 16-bit type.  The weight gradient
sums over tokens, where 1 x 128 blocks do not help: it is the 16-bit product of the output gradient with the values
that the 8-bit activations stand for.  The 8-bit activations are all that the forward pass keeps.

The checks, the memory and the autograd nodes are in csrc/torch_fp8.cpp; the kernels are launched on the current stream of
the arguments' device, and none of the calls waits for the device.  The gradients can be taken once (no create_graph); there are
no forward-mode derivatives.  What is held in 8 bits by `quantize_fp8` or `quantize_fp8_weight` is a constant to autograd.
"""

from __future__ import annotations

import torch

from .. import _native


def __getattr__(name: str):
    if name in ("Fp8Blocks", "Fp8Weight"):  # classes of the binding, which is loaded at the first use
        return getattr(_native.binding(), name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def quantize_fp8(x: torch.Tensor) -> Fp8Blocks:
    """Holds x [..., cols] (float32, bfloat16 or float16) in 8 bits with a scale per 128 columns of a row: a quarter or
    half of its bytes.  cols must be a multiple of 8.  `.dequantize()` gives the values back."""
    return _native.binding().quantize_fp8(x)


def quantize_fp8_weight(weight: torch.Tensor) -> Fp8Weight:
    """Holds weight [N, K] or [E, N, K] in 8 bits with a scale per 128 x 128 block, for a linear map and for its
    input gradient.  N and K must be multiples of 8."""
    return _native.binding().quantize_fp8_weight(weight)


def linear_fp8(x: torch.Tensor, weight: torch.Tensor | Fp8Weight, quantized: Fp8Weight | None = None) -> torch.Tensor:
    """x [..., K] times weight [N, K] transposed, both taken in 8 bits; returns [..., N] in x's type (bfloat16 or
    float16).  `weight` is a parameter, quantised in the call, or an Fp8Weight (serving: no gradient of the weight).
    `quantized` is the 8-bit form of `weight` where the caller has it already, for example once per step for several
    micro-batches.  Differentiable in x and in a `weight` that is a tensor; rounding to 8 bits passes gradients
    through unchanged.  The forward pass keeps x in 8 bits only.  N and K must be multiples of 8."""
    return _native.binding().linear_fp8(x, weight, quantized)


def grouped_linear_fp8(
    x: torch.Tensor,
    weight: torch.Tensor | Fp8Weight,
    expert_frequency: torch.Tensor,
    quantized: Fp8Weight | None = None,
) -> torch.Tensor:
    """linear_fp8 with a weight per expert [E, N, K]: x [rows, K] holds expert_frequency[e] consecutive rows for expert e,
    in expert order and without alignment, as in `Experts.cuda_forward`.  The counts stay on the device.  Rows behind
    the last expert's (the counts sum to less than `rows`) give zeros; counts that overshoot are cut off."""
    return _native.binding().grouped_linear_fp8(x, weight, expert_frequency, quantized)


def swiglu_fp8_checkpoint(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """`swiglu(gate, up)` that keeps gate and up in 8 bits between the passes: half the memory of a 16-bit SwiGLU, a
    quarter of an fp32 one.  The result is that of `swiglu`; the gradients are those at the values the 8-bit form
    stands for.  The last dimension must be a multiple of 8."""
    return _native.binding().swiglu_fp8_checkpoint(gate, up)
