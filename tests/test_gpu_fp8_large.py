"""The 8-bit operators on tensors of more than 2^31 elements: 264 copies of 1024 rows give 264 times the same results."""

import pytest
import torch

import _fp8_ref as R
from _util import DEV, check_device_status, randn

pytestmark = pytest.mark.gpu

ROWS, COPIES, WIDE = 1024, 264, 8192
assert ROWS * COPIES * WIDE > 2**31


@pytest.fixture(autouse=True)
def _memory():
    if torch.cuda.get_device_properties(0).total_memory < 80e9:
        pytest.skip("needs 80 GB")
    yield
    torch.cuda.empty_cache()


def _same_copies(big, small):
    for part in big.view(-1, *small.shape):
        assert torch.equal(part, small)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store(dtype):
    import fma_b200 as fma

    small = randn((ROWS, WIDE), dtype, 1).to(DEV)
    held = fma.quantize_fp8(small).dequantize()
    assert torch.equal(held[:8].double(), R.hold(small[:8]))
    _same_copies(fma.quantize_fp8(small.repeat(COPIES, 1)).dequantize(), held)


def test_linear():
    import fma_b200 as fma

    K = 136
    x, w = randn((ROWS, K), torch.bfloat16, 2).to(DEV), randn((WIDE, K), torch.bfloat16, 3, scale=0.05).to(DEV)
    d_out = randn((ROWS, WIDE), torch.bfloat16, 4, scale=0.1).to(DEV)
    values, sizes = R.linear(x, w, d_out)
    a = x.clone().requires_grad_()
    out = fma.linear_fp8(a, w)
    (d_x,) = torch.autograd.grad(out, a, d_out)
    R.check_product(out.detach(), values[0], sizes[0], K)
    R.check_product(d_x, values[1], sizes[1], WIDE)
    b, c = x.repeat(COPIES, 1).requires_grad_(), w.clone().requires_grad_()
    big = fma.linear_fp8(b, c)
    _same_copies(big.detach(), out.detach())
    big.backward(d_out.repeat(COPIES, 1))
    _same_copies(b.grad, d_x)
    R.check_product(c.grad, COPIES * values[2], COPIES * sizes[2], COPIES * ROWS)
    check_device_status()


def test_grouped():
    """Three experts of the same weights, so that every copy has the same result, whichever expert it falls to."""
    import fma_b200 as fma

    K = 136
    x, w = randn((ROWS, K), torch.bfloat16, 5).to(DEV), randn((1, WIDE, K), torch.bfloat16, 6, scale=0.05).to(DEV)
    d_out = randn((ROWS, WIDE), torch.bfloat16, 7, scale=0.1).to(DEV)
    a = x.clone().requires_grad_()
    out = fma.grouped_linear_fp8(a, w, torch.tensor([ROWS], device=DEV))
    (d_x,) = torch.autograd.grad(out, a, d_out)
    rows = COPIES * ROWS
    b = x.repeat(COPIES, 1).requires_grad_()
    big = fma.grouped_linear_fp8(b, w.repeat(3, 1, 1), torch.tensor([rows // 3 + 77, 0, rows], device=DEV))
    _same_copies(big.detach(), out.detach())
    big.backward(d_out.repeat(COPIES, 1))
    _same_copies(b.grad, d_x)
    check_device_status()


def test_swiglu():
    import fma_b200 as fma

    gate, up, d_out = (randn((ROWS, WIDE), torch.bfloat16, s).to(DEV) for s in (8, 9, 10))
    g, u = gate.clone().requires_grad_(), up.clone().requires_grad_()
    out = fma.swiglu_fp8_checkpoint(g, u)
    out.backward(d_out)
    a, b = gate.repeat(COPIES, 1).requires_grad_(), up.repeat(COPIES, 1).requires_grad_()
    big = fma.swiglu_fp8_checkpoint(a, b)
    _same_copies(big.detach(), out.detach())
    big.backward(d_out.repeat(COPIES, 1))
    _same_copies(a.grad, g.grad)
    _same_copies(b.grad, u.grad)


def test_weights():
    import fma_b200 as fma

    E, N, K = 66, 8192, 4096
    one = randn((N, K), torch.bfloat16, 11, scale=0.02).to(DEV)
    held = fma.quantize_fp8_weight(one)
    many = fma.quantize_fp8_weight(one.repeat(E, 1, 1))
    _same_copies(many.values.view(torch.uint8), held.values[0].view(torch.uint8))
    _same_copies(many.dequantize(), held.dequantize())
    x = randn((300, K), torch.bfloat16, 12).to(DEV)
    want = fma.linear_fp8(x, held)
    got = fma.grouped_linear_fp8(x, many, torch.tensor([0] * (E - 2) + [150, 150], device=DEV))
    assert torch.equal(got, want)  # pair tiles of the last experts
    few = fma.grouped_linear_fp8(x[:9], many, torch.tensor([0] * (E - 2) + [4, 5], device=DEV))
    R.check_product(few, *(t[:9] for t in (R.hold(x[:9]) @ R.hold(one, 128).T, R.hold(x[:9]).abs() @ R.hold(one, 128).abs().T)), K)
    check_device_status()
