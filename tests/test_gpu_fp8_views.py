"""Inputs of the 8-bit operators that are no plain matrices: what is a view of rows is taken as it lies, in both directions."""

import pytest
import torch

import _fp8_ref as R
from _util import DEV, randn

pytestmark = pytest.mark.gpu

K, N = 264, 136
NAMES = ["contiguous", "columns", "one of a size-1 dimension", "vector", "some rows", "turned", "repeated", "misaligned"]


def _nodes(fn):
    seen, todo = [], [fn]
    while todo:
        f = todo.pop()
        if f is not None:
            seen.append(f.name())
            todo += [n for n, _ in f.next_functions]
    return seen


def _views():
    wide = randn((4, 30, 2 * K), torch.bfloat16, 1).to(DEV)
    flat = randn((120 * K + 1,), torch.bfloat16, 2).to(DEV)
    return {
        "contiguous": (lambda t: t[:, :, :K].contiguous(), wide, True),
        "columns": (lambda t: t[:, :, K:], wide, True),
        "one of a size-1 dimension": (lambda t: t[:, :, :K].unsqueeze(2), wide, True),
        "vector": (lambda t: t[1, 2, :K], wide, True),
        "some rows": (lambda t: t[:, 3:17, :K], wide, False),
        "turned": (lambda t: t[:, :, :K].transpose(0, 1), wide, False),
        "repeated": (lambda t: t[:, :1, :K].expand(4, 7, K), wide, False),
        "misaligned": (lambda t: t[1:].view(2, 60, K), flat, False),
    }


@pytest.mark.parametrize("name", NAMES)
def test_linear_on_views(name):
    import fma_b200 as fma

    view, leaf, as_it_lies = _views()[name]
    w = randn((N, K), torch.bfloat16, 3, scale=0.05).to(DEV)
    leaf = leaf.clone().requires_grad_()
    x = view(leaf)
    out = fma.linear_fp8(x, w)
    names = _nodes(out.grad_fn)
    assert not any("AsStrided" in n for n in names), names
    copies = [n for n in names if "Clone" in n]
    if as_it_lies:
        assert len(copies) == (1 if name == "contiguous" else 0), names  # the test's own
    else:
        assert len(copies) <= 1, names
    assert out.shape == (*x.shape[:-1], N)
    rows = x.detach().reshape(-1, K)
    d_out = randn(out.shape, torch.bfloat16, 4).to(DEV)
    (y, dx, _), (sy, sx, _) = R.linear(rows, w, d_out.reshape(-1, N))
    R.check_product(out.detach().reshape(-1, N), y, sy, K)
    (got,) = torch.autograd.grad(out, x, d_out, retain_graph=True)
    R.check_product(got.reshape(-1, K), dx, sx, N)
    out.backward(d_out)  # through the view to the leaf: torch's own sums
    want = torch.autograd.grad(view(leaf), leaf, got)[0]
    assert torch.equal(leaf.grad, want)


def test_backward_of_a_batch_needs_no_extra_memory():
    """The gradient of x [batch, tokens, K] is what the product wrote."""
    import fma_b200 as fma

    x = randn((4, 2048, 1024), torch.bfloat16, 5).to(DEV).requires_grad_()
    w = fma.quantize_fp8_weight(randn((64, 1024), torch.bfloat16, 6, scale=0.05).to(DEV))
    d_out = randn((4, 2048, 64), torch.bfloat16, 7).to(DEV)
    out = fma.linear_fp8(x, w)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(out, x, d_out)
    assert torch.cuda.max_memory_allocated() - before <= 1.25 * 2 * x.numel()


def test_swiglu_and_store_on_views():
    import fma_b200 as fma

    for name, (view, leaf, _) in _views().items():
        x = view(leaf)
        held = fma.quantize_fp8(x).dequantize()
        assert held.shape == x.shape
        assert torch.equal(held.double().reshape(-1, K), R.hold(x.reshape(-1, K))), name
        gate, up = x.detach().requires_grad_(), (x.detach() * 0.5).requires_grad_()
        plain, rest = x.detach().contiguous().requires_grad_(), up.detach().contiguous().requires_grad_()
        a, b = fma.swiglu_fp8_checkpoint(gate, up), fma.swiglu_fp8_checkpoint(plain, rest)
        assert torch.equal(a, b)
        d = randn(a.shape, torch.bfloat16, 8).to(DEV)
        for g, h in zip(torch.autograd.grad(a, (gate, up), d), torch.autograd.grad(b, (plain, rest), d)):
            assert torch.equal(g, h), name
