"""The 8-bit products and the weight gradient where one pair of SMs walks many tiles: accumulators that share columns of
tensor memory change hands, a third tile takes the first one's accumulator again, scale buffers and ring stages go round.  An
SM limit makes small problems do that; the sums of an element are in the same order however the tiles are dealt, so the results
also equal those without a limit bit by bit."""

import contextlib

import pytest
import torch

import _fp8_ref as R
from _util import DEV, check_device_status, randn

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


@contextlib.contextmanager
def sm_limit(n):
    from fma_b200 import _native

    _native.lib().fma_b200_set_sm_limit(n)
    try:
        yield
    finally:
        _native.lib().fma_b200_set_sm_limit(0)


def _step(call, x, w, d_out):
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = call(a, b)
    out.backward(d_out)
    return out.detach(), a.grad, b.grad


# full tiles of 256 rows and a lower last one; sums of 1, 2, 5 and 9 blocks of 128 in both directions
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("sms", [2, 3, 6])
@pytest.mark.parametrize("rows,K,N", [(1793, 128, 520), (1100, 264, 776), (900, 1032, 136), (1030, 520, 1160), (256, 392, 1800)])
def test_linear_on_few_pairs(dtype, sms, rows, K, N):
    import fma_b200 as fma

    x, w = randn((rows, K), dtype, 1).to(DEV), randn((N, K), dtype, 2, scale=0.05).to(DEV)
    d_out = randn((rows, N), dtype, 3, scale=0.1).to(DEV)
    free = _step(fma.linear_fp8, x, w, d_out)
    with sm_limit(sms):
        got = _step(fma.linear_fp8, x, w, d_out)
        torch.cuda.synchronize()
    values, sizes = R.linear(x, w, d_out)
    for g, f, want, size, terms in zip(got, free, values, sizes, (K, N, rows)):
        R.check_product(g, want, size, terms)
        assert torch.equal(g, f)
    check_device_status()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("sms", [2, 4])
@pytest.mark.parametrize("K,N", [(136, 776), (1032, 264), (648, 520)])
def test_grouped_on_few_pairs(dtype, sms, K, N):
    """Tiles of 256 rows behind low ones and the other way round, an odd number of tiles, experts without rows."""
    import fma_b200 as fma

    counts = [513, 0, 256, 1, 255, 700, 31, 225, 0, 288]
    rows = sum(counts) + 5
    x, w = randn((rows, K), dtype, 4).to(DEV), randn((len(counts), N, K), dtype, 5, scale=0.05).to(DEV)
    d_out, count = randn((rows, N), dtype, 6, scale=0.1).to(DEV), torch.tensor(counts, dtype=torch.int32, device=DEV)
    call = lambda a, b: fma.grouped_linear_fp8(a, b, count)  # noqa: E731
    free = _step(call, x, w, d_out)
    with sm_limit(sms):
        got = _step(call, x, w, d_out)
        torch.cuda.synchronize()
    values, sizes = R.grouped(x, w, counts, d_out)
    for g, f, want, size, terms in zip(got, free, values, sizes, (K, N, max(counts))):
        R.check_product(g, want, size, terms)
        assert torch.equal(g, f)
    check_device_status()


def test_all_pairs_walk_several_full_tiles():
    """Without a limit: five rounds of 256-row tiles on every pair, in both directions and in the weight gradient."""
    import fma_b200 as fma

    rows, K, N = 32 * 256 + 40, 264, 2568
    x, w = randn((rows, K), torch.bfloat16, 7).to(DEV), randn((N, K), torch.bfloat16, 8, scale=0.05).to(DEV)
    d_out = randn((rows, N), torch.bfloat16, 9, scale=0.1).to(DEV)
    got = _step(fma.linear_fp8, x, w, d_out)
    values, sizes = R.linear(x, w, d_out)
    for g, want, size, terms in zip(got, values, sizes, (K, N, rows)):
        R.check_product(g, want, size, terms)
    # the input gradient with many columns
    x, w = randn((rows, N), torch.bfloat16, 10).to(DEV), randn((K, N), torch.bfloat16, 11, scale=0.05).to(DEV)
    d_out = randn((rows, K), torch.bfloat16, 12, scale=0.1).to(DEV)
    got = _step(fma.linear_fp8, x, w, d_out)
    values, sizes = R.linear(x, w, d_out)
    for g, want, size, terms in zip(got, values, sizes, (N, K, rows)):
        R.check_product(g, want, size, terms)
    check_device_status()


@pytest.mark.parametrize("sms", [2, 6])
def test_layer_on_few_pairs(sms):
    import fma_b200 as fma

    moe = fma.MoE(5, 3, 392, 264, fma.swiglu_packed, True, False, 0.05)
    with torch.no_grad():
        for i, p in enumerate((moe.gate.weight, moe.c_fc.weight, moe.c_proj.weight)):
            p.copy_(randn(p.shape, torch.float32, 20 + i, scale=0.1))
    moe = moe.to(DEV).bfloat16()
    moe.fp8_experts = True
    x, dy = randn((1500, 392), torch.bfloat16, 23).to(DEV), randn((1500, 392), torch.bfloat16, 24).to(DEV)

    def step():
        a = x.clone().requires_grad_()
        moe.zero_grad(set_to_none=True)
        y, _ = moe(a)
        y.backward(dy)
        return y.detach(), a.grad, moe.c_fc.weight.grad, moe.c_proj.weight.grad

    free = step()
    with sm_limit(sms):
        got = step()
        torch.cuda.synchronize()
    for g, f in zip(got, free):
        assert bool(torch.isfinite(g).all()) and torch.equal(g, f)
    check_device_status()


# reductions of 1 to 128 groups of 512 columns, shared by one to eight CTAs, the last group short; tiles of 128 weight rows
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K,N", [(520, 40), (1032, 4104), (2056, 264), (4104, 1800), (4104, 8200), (8200, 136), (14336, 264), (20488, 136), (65536, 24)])
@pytest.mark.parametrize("rows", [1, 16, 49, 100])
def test_few_rows_share_the_reduction(dtype, K, N, rows):
    import fma_b200 as fma

    x, w = randn((rows, K), dtype, 30).to(DEV), randn((N, K), dtype, 31, scale=0.02).to(DEV)
    want, size = R.hold(x) @ R.hold_weight(w).T, R.hold(x).abs() @ R.hold_weight(w).abs().T
    held = fma.quantize_fp8_weight(w)
    got = fma.linear_fp8(x, held)
    R.check_product(got, want, size, K)
    assert torch.equal(got, fma.linear_fp8(x, held))
    check_device_status()


@pytest.mark.parametrize("K,N,E,rows", [(4104, 1032, 8, 8), (4104, 264, 8, 100), (8200, 264, 5, 30), (20488, 72, 3, 6), (2056, 776, 40, 64), (14344, 136, 2, 200), (1032, 264, 100, 700)])
def test_few_rows_of_experts_share_the_reduction(K, N, E, rows):
    import fma_b200 as fma

    g = torch.Generator().manual_seed(K + rows)
    counts = torch.bincount(torch.randint(0, E, (rows - 1,), generator=g), minlength=E).tolist()
    x, w = randn((rows, K), torch.bfloat16, 32).to(DEV), randn((E, N, K), torch.bfloat16, 33, scale=0.02).to(DEV)
    values, sizes = R.grouped(x, w, counts, torch.zeros(rows, N, device=DEV))
    held, count = fma.quantize_fp8_weight(w), torch.tensor(counts, device=DEV)
    got = fma.grouped_linear_fp8(x, held, count)
    R.check_product(got, values[0], sizes[0], K)
    assert torch.equal(got, fma.grouped_linear_fp8(x, held, count))
    check_device_status()
