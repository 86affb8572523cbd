"""Counts of the grouped 8-bit linear map at the ends of their types."""

import pytest
import torch

import _fp8_ref as R
from _util import DEV, check_device_status, randn

pytestmark = pytest.mark.gpu

MOST = {torch.int32: 2**31 - 1, torch.uint32: 2**32 - 1, torch.int64: 2**63 - 1}


@pytest.mark.parametrize("rows", [30, 700])
@pytest.mark.parametrize("dtype", list(MOST))
@pytest.mark.parametrize("place", [0, 1, 39])
def test_the_largest_counts_are_cut_off(dtype, rows, place):
    import fma_b200 as fma

    E = 40
    x, w = randn((rows, 128), torch.bfloat16, 1).to(DEV), randn((E, 64, 128), torch.bfloat16, 2).to(DEV)
    counts = [0] * E
    counts[0], counts[place], counts[39] = rows - 9, MOST[dtype], MOST[dtype]
    cut = [0] * E
    cut[0] = rows if place == 0 else rows - 9
    cut[place] += rows - cut[0] if place else 0
    values, sizes = R.grouped(x, w, cut, torch.zeros(rows, 64, device=DEV))
    count = torch.tensor(counts, dtype=dtype).to(DEV)
    R.check_product(fma.grouped_linear_fp8(x, fma.quantize_fp8_weight(w), count), values[0], sizes[0], 128)
    a = x.clone().requires_grad_()
    R.check_product(fma.grouped_linear_fp8(a, w, count).detach(), values[0], sizes[0], 128)
    check_device_status()


@pytest.mark.parametrize("rows", [30, 700])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_negative_counts_are_none(dtype, rows):
    import fma_b200 as fma

    x, w = randn((rows, 128), torch.bfloat16, 3).to(DEV), randn((3, 64, 128), torch.bfloat16, 4).to(DEV)
    values, sizes = R.grouped(x, w, [0, rows - 4, 0], torch.zeros(rows, 64, device=DEV))
    count = torch.tensor([-5, rows - 4, -MOST[dtype]], dtype=dtype).to(DEV)
    R.check_product(fma.grouped_linear_fp8(x, fma.quantize_fp8_weight(w), count), values[0], sizes[0], 128)
    a = x.clone().requires_grad_()
    R.check_product(fma.grouped_linear_fp8(a, w, count).detach(), values[0], sizes[0], 128)
    check_device_status()
