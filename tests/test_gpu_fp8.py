"""The 8-bit operators on the GPU against their definition in 64 bits (tests/_fp8_ref.py)."""

import pytest
import torch

import _fp8_ref as R
from _util import DEV, check_device_status, randn

pytestmark = pytest.mark.gpu

ALL = [torch.bfloat16, torch.float16, torch.float32]
HALF = [torch.bfloat16, torch.float16]


def _same(got, want):
    """Exact: what is held in 8 bits has at most 4 significant bits."""
    assert torch.equal(torch.nan_to_num(got.double(), nan=12345.0), torch.nan_to_num(want.to(got.dtype).double(), nan=12345.0))


# ---- storing and restoring -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", [(1, 8), (3, 136), (130, 520), (257, 1000), (5, 4096), (2, 3, 264)])
def test_store(dtype, shape):
    import fma_b200 as fma

    x = randn(shape, dtype, 1, scale=3.0).to(DEV)
    held = fma.quantize_fp8(x)
    got = held.dequantize()
    assert got.shape == x.shape and got.dtype == dtype
    _same(got.reshape(-1, shape[-1]), R.hold(x.reshape(-1, shape[-1])))
    assert held.dequantize(torch.float32).dtype == torch.float32
    assert held.nbytes <= x.numel() * 1.25 + 16 * x.numel() // shape[-1] + 512 * (shape[-1] // 512 + 1) * (x.numel() // shape[-1] // 128 + 1)


@pytest.mark.parametrize("dtype", ALL)
def test_store_special_values(dtype):
    import fma_b200 as fma

    info = torch.finfo(dtype)
    x = randn((16, 256), dtype, 2)
    x[0] = 0
    x[1, :128] = 0
    x[2, 5], x[2, 200] = float("inf"), float("nan")  # neighbours keep their scale
    x[3] = float("nan")
    x[4] = -0.0
    x[5] = info.tiny  # the smallest normal number
    x[6, 0] = info.max
    x[7, 0] = -info.max
    x[8, :] = 448 * 2.0**-10  # a block maximum exactly on the border
    x[9, :] = torch.tensor(448 * 2.0**-10, dtype=torch.float32).to(dtype) * (1 + info.eps)  # and one step above
    x[10, :128] = 2.0**-14
    x[10, 0] = 1.0
    x[11] = torch.linspace(-464, 464, 256).to(dtype)
    x[12] = info.smallest_normal * info.eps  # the smallest subnormal number
    x = x.to(DEV)
    got = fma.quantize_fp8(x).dequantize()
    want = R.hold(x)
    want = torch.where(want.abs() > info.max, torch.copysign(torch.tensor(info.max, dtype=torch.float64, device=DEV), want), want)
    _same(got, want)


@pytest.mark.parametrize("dtype", ALL)
def test_store_strides(dtype):
    import fma_b200 as fma

    wide = randn((70, 528), dtype, 3).to(DEV)
    for x in (wide[:, 264:], wide[::2, :264], wide[:, 8:272], wide[1:].t()[:64, :64], wide[:, :264].unsqueeze(1), wide[:1].expand(9, 528),
              wide.flatten()[1 : 1 + 40 * 24].view(40, 24)):  # fmt: skip
        _same(fma.quantize_fp8(x).dequantize().reshape(-1, x.size(-1)), R.hold(x.reshape(-1, x.size(-1))))


def test_store_nothing():
    import fma_b200 as fma

    x = torch.empty(0, 16, device=DEV, dtype=torch.bfloat16)
    assert fma.quantize_fp8(x).dequantize().shape == (0, 16)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", [(8, 8), (136, 264), (3, 264, 136), (2, 128, 1024)])
def test_weight(dtype, shape):
    import fma_b200 as fma

    w = randn(shape, dtype, 4, scale=0.02).to(DEV)
    held = fma.quantize_fp8_weight(w)
    _same(held.dequantize(), R.hold_weight(w))
    N, K = shape[-2:]
    assert held.values.shape[-2] == N and bool((held.values.float()[..., K:] == 0).all())


def test_what_is_held_can_be_copied_and_saved(tmp_path):
    import copy

    import fma_b200 as fma

    x, w = randn((9, 264), torch.bfloat16, 24).to(DEV), randn((2, 136, 264), torch.bfloat16, 25).to(DEV)
    for held in (fma.quantize_fp8(x), fma.quantize_fp8_weight(w)):
        torch.save(held, tmp_path / "held.pt")
        for other in (copy.deepcopy(held), torch.load(tmp_path / "held.pt", weights_only=False)):
            assert type(other) is type(held) and other.shape == held.shape and other.dtype == held.dtype
            assert other.device == held.device and torch.equal(other.dequantize(), held.dequantize())
    assert isinstance(held, fma.Fp8Weight) and isinstance(fma.quantize_fp8(x), fma.Fp8Blocks)
    assert held.scales.data_ptr() != other.scales.data_ptr() and torch.equal(held.scales, other.scales)


def test_second_derivatives_are_refused():
    import fma_b200 as fma

    x, w = randn((40, 16), torch.bfloat16, 26).to(DEV).requires_grad_(), randn((8, 16), torch.bfloat16, 27).to(DEV)
    for y in (fma.linear_fp8(x, w), fma.swiglu_fp8_checkpoint(x, x)):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


# ---- the linear map --------------------------------------------------------------------------------
LINEAR = [(1, 8, 8), (1, 128, 16), (5, 1000, 1544), (16, 520, 136), (17, 392, 264), (127, 128, 128), (129, 264, 520), (300, 2056, 1032),
          (1025, 136, 392), (9, 4104, 264), (40, 2056, 392), (64, 1024, 2048), (90, 4104, 136), (120, 8200, 72), (33, 520, 8), (200, 136, 8),
          (130, 8, 40), (260, 40, 72)]  # fmt: skip


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,K,N", LINEAR)
def test_linear(dtype, rows, K, N):
    import fma_b200 as fma

    x, w = randn((rows, K), dtype, 5).to(DEV), randn((N, K), dtype, 6, scale=0.05).to(DEV)
    d_out = randn((rows, N), dtype, 7, scale=0.1).to(DEV)
    (y, dx, dw), (sy, sx, sw) = R.linear(x, w, d_out)
    R.check_product(fma.linear_fp8(x, fma.quantize_fp8_weight(w)), y, sy, K)  # serving
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fma.linear_fp8(a, b)
    out.backward(d_out)
    R.check_product(out.detach(), y, sy, K)
    R.check_product(a.grad, dx, sx, N)
    R.check_product(b.grad, dw, sw, rows)
    check_device_status()


@pytest.mark.parametrize("rows", [4, 40])
def test_linear_gradients_one_at_a_time_and_kept_weights(rows):
    import fma_b200 as fma

    x, w = randn((2, rows // 2, 264), torch.bfloat16, 8).to(DEV), randn((136, 264), torch.bfloat16, 9, scale=0.05).to(DEV)
    d = randn((2, rows // 2, 136), torch.bfloat16, 10).to(DEV)
    (y, dx, dw), (sy, sx, sw) = R.linear(x.reshape(rows, 264), w, d.reshape(rows, 136))
    held = fma.quantize_fp8_weight(w)
    a = x.clone().requires_grad_()
    out = fma.linear_fp8(a, held)
    out.backward(d)
    assert out.shape == (2, rows // 2, 136)
    R.check_product(out.detach().view(rows, 136), y, sy, 264)
    R.check_product(a.grad.view(rows, 264), dx, sx, 136)
    b = w.clone().requires_grad_()
    fma.linear_fp8(x, b, held).backward(d)
    R.check_product(b.grad, dw, sw, rows)
    # an upstream gradient with a zero stride, and rows of x with a pitch
    c = torch.zeros(rows, 528, dtype=torch.bfloat16, device=DEV)
    c[:, 264:] = x.reshape(rows, 264)
    e = c[:, 264:].detach().requires_grad_()
    fma.linear_fp8(e, w).sum().backward()
    ones = torch.ones(rows, 136, dtype=torch.bfloat16, device=DEV)
    R.check_product(e.grad, *(t[1] for t in R.linear(x.reshape(rows, 264), w, ones)), 136)


def test_linear_gradient_is_that_of_differences():
    """Straight-through: at points that the 8-bit form holds exactly, with exact weights, the map is linear."""
    import fma_b200 as fma

    x = torch.randint(-8, 9, (24, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    w = torch.randint(-8, 9, (128, 128), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    x[:, 0], w[0, 0] = 8, 8
    a = x.clone().requires_grad_()
    out = fma.linear_fp8(a, w)
    pick = torch.zeros_like(out)
    pick[3, 7] = 1
    out.backward(pick)
    step = torch.zeros_like(x)
    step[3, 5] = 1 if x[3, 5] < 8 else -1
    moved = fma.linear_fp8(x + step, w)[3, 7].double() - out[3, 7].double()
    assert float(moved.detach()) == float(a.grad[3, 5]) * float(step[3, 5])


@pytest.mark.parametrize("rows", [9, 60, 150])
def test_linear_far_scales(rows):
    """Every row and every weight block with a scale of its own, far apart, rows and blocks of zeros among them."""
    import fma_b200 as fma

    K, N = 1544, 264
    x, w = randn((rows, K), torch.bfloat16, 31).to(DEV), randn((N, K), torch.bfloat16, 32).to(DEV)
    block = torch.arange(K, device=DEV) // 128
    power = (torch.arange(rows, device=DEV)[:, None] * 7 + block * 5) % 81 - 40
    x = (x.double() * torch.exp2(power.double())).to(torch.bfloat16)
    power = ((torch.arange(N, device=DEV)[:, None] // 128) * 11 + block * 3) % 61 - 30
    w = (w.double() * torch.exp2(power.double())).to(torch.bfloat16)
    x[2], x[4, :256], w[:128, 384:512] = 0, 0, 0
    d_out = randn((rows, N), torch.bfloat16, 33).to(DEV)
    (y, dx, dw), (sy, sx, sw) = R.linear(x, w, d_out)
    R.check_product(fma.linear_fp8(x, fma.quantize_fp8_weight(w)), y, sy, K)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fma.linear_fp8(a, b)
    out.backward(d_out)
    R.check_product(out.detach(), y, sy, K)
    R.check_product(a.grad, dx, sx, N)
    R.check_product(b.grad, dw, sw, rows)


@pytest.mark.parametrize("rows", [3, 200])
def test_linear_keeps_a_bad_row_to_itself(rows):
    import fma_b200 as fma

    x, w = randn((rows, 264), torch.bfloat16, 11).to(DEV), randn((136, 264), torch.bfloat16, 12).to(DEV)
    held = fma.quantize_fp8_weight(w)
    clean = fma.linear_fp8(x, held)
    x[1, 130] = float("inf")
    got = fma.linear_fp8(x, held)
    assert bool(torch.isnan(got[1]).all())
    keep = torch.arange(rows, device=DEV) != 1
    assert torch.equal(got[keep], clean[keep])


def test_linear_without_rows():
    import fma_b200 as fma

    x = torch.empty(0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = randn((8, 16), torch.bfloat16, 13).to(DEV).requires_grad_()
    y = fma.linear_fp8(x, w)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 16) and bool((w.grad == 0).all())


# ---- the grouped linear map ------------------------------------------------------------------------
GROUPED = [
    (264, 136, [5, 0, 8]),  # few rows
    (264, 136, [0, 300, 1, 0, 129]),  # an expert over several tiles, empty ones around
    (520, 264, [256, 0, 512]),  # full tiles
    (136, 392, [0, 0, 0, 40]),
    (128, 8, [37]),
    (392, 264, [17] * 40),
    (2056, 136, [1, 70, 0, 16]),  # reductions that several CTAs share
    (2056, 136, [20, 0, 0, 0]),
    (1032, 264, [128, 0, 127, 129, 1, 64, 65, 33]),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K,N,counts", GROUPED)
@pytest.mark.parametrize("rest", [0, 3])
def test_grouped(dtype, K, N, counts, rest):
    import fma_b200 as fma

    rows, E = sum(counts) + rest, len(counts)
    x, w = randn((rows, K), dtype, 14).to(DEV), randn((E, N, K), dtype, 15, scale=0.05).to(DEV)
    d_out = randn((rows, N), dtype, 16, scale=0.1).to(DEV)
    (y, dx, dw), (sy, sx, sw) = R.grouped(x, w, counts, d_out)
    count = torch.tensor(counts, dtype=torch.int32, device=DEV)
    held = fma.quantize_fp8_weight(w)
    R.check_product(fma.grouped_linear_fp8(x, held, count), y, sy, K)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fma.grouped_linear_fp8(a, b, count)
    out.backward(d_out)
    R.check_product(out.detach(), y, sy, K)
    R.check_product(a.grad, dx, sx, N)
    R.check_product(b.grad, dw, sw, max(counts))
    if rest:
        assert bool((out[-rest:] == 0).all()) and bool((a.grad[-rest:] == 0).all())
    check_device_status()


@pytest.mark.parametrize("dtype", [torch.int32, torch.uint32, torch.int64])
@pytest.mark.parametrize("rows", [30, 700])
def test_grouped_counts_that_do_not_fit(dtype, rows):
    """Counts that overshoot (or are negative) are cut off, never followed."""
    import fma_b200 as fma

    x, w = randn((rows, 128), torch.bfloat16, 17).to(DEV), randn((4, 64, 128), torch.bfloat16, 18).to(DEV)
    held = fma.quantize_fp8_weight(w)
    wild = [rows - 9, 20, 2**31 - 1, 5] if dtype != torch.uint32 else [rows - 9, 20, 2**30, 5]
    want = R.grouped(x, w, [rows - 9, 9, 0, 0], torch.zeros(rows, 64, device=DEV))
    got = fma.grouped_linear_fp8(x, held, torch.tensor(wild, dtype=dtype).to(DEV))
    R.check_product(got, want[0][0], want[1][0], 128)
    a = x.clone().requires_grad_()
    out = fma.grouped_linear_fp8(a, held, torch.tensor(wild, dtype=dtype).to(DEV))
    R.check_product(out.detach(), want[0][0], want[1][0], 128)
    out.sum().backward()
    assert bool(torch.isfinite(a.grad).all())
    none = torch.zeros(4, dtype=dtype).to(DEV)
    assert bool((fma.grouped_linear_fp8(x, held, none) == 0).all())


# ---- SwiGLU ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape,halves", [((1, 8), False), ((3, 5, 136), False), ((77, 264), True), ((130, 1032), True)])
def test_swiglu(dtype, shape, halves):
    import fma_b200 as fma

    if halves:
        up, gate = randn((*shape[:-1], 2 * shape[-1]), dtype, 19, scale=2.0).to(DEV).chunk(2, dim=-1)
    else:
        up, gate = randn(shape, dtype, 19, scale=2.0).to(DEV), randn(shape, dtype, 20, scale=2.0).to(DEV)
    d_out = randn(shape, dtype, 21).to(DEV)
    a, b = gate.detach().requires_grad_(), up.detach().requires_grad_()
    out = fma.swiglu_fp8_checkpoint(a, b)
    out.backward(d_out)
    with torch.no_grad():
        assert torch.equal(fma.swiglu_fp8_checkpoint(gate, up), out)
    # One rounding; fp32 arithmetic of about 10 operations, with the approximate exponential and reciprocal (2 ulp each)
    # for the 16-bit types.  The factor s + g s (1 - s) of d_gate cancels for negative gates: its error counts against
    # s + |g| s (1 - s).
    half, fp32 = torch.finfo(dtype).eps / 2, 16 * 2.0**-23
    tiny = 2 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    want = R.swiglu(gate, up, d_out)
    g = R.hold(gate.reshape(-1, shape[-1])).reshape(shape)
    u = R.hold(up.reshape(-1, shape[-1])).reshape(shape)
    s = torch.sigmoid(g)
    # |g| 2^-23 relative error of exp(-g) from its argument's rounding
    grow = 1 + torch.maximum(g.abs(), gate.double().abs())
    sizes = (want[0].abs(), (d_out.double() * u).abs() * (s + g.abs() * s * (1 - s)), want[2].abs())
    for got, ref, size in zip((out.detach(), a.grad, b.grad), want, sizes):
        off = (got.double() - ref).abs()
        assert bool((off <= half * ref.abs() + (1 + half) * fp32 * grow * size + tiny).all())
    check_device_status()


@pytest.mark.parametrize("rows", [40, 700])
def test_grouped_rows_that_nothing_writes_are_not_read(rows):
    import fma_b200 as fma

    x, w = randn((rows, 264), torch.bfloat16, 34).to(DEV), randn((3, 136, 264), torch.bfloat16, 35).to(DEV)
    d_out, count = randn((rows, 136), torch.bfloat16, 36).to(DEV), torch.tensor([rows // 2, 3, rows // 4], device=DEV)
    results = []
    for byte in (0, 0xFF):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        blocks = [torch.full((n,), byte, dtype=torch.uint8, device=DEV) for n in [1 << 26] * 2 + [1 << 20] * 32 + [1 << 13] * 128]
        torch.cuda.synchronize()
        del blocks
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = fma.grouped_linear_fp8(a, b, count)
        out.backward(d_out)
        results.append((out.detach(), a.grad, b.grad))
    for one, other in zip(*results):
        assert bool(torch.isfinite(one).all()) and torch.equal(one, other)


@pytest.mark.parametrize("N,K", [(8, 8), (200, 136), (136, 520), (392, 128)])
def test_an_expert_without_a_number_stays_alone(N, K):
    """Tiles and k-blocks that reach into the next expert's weights, and rows behind an expert's, spoil nothing."""
    import fma_b200 as fma

    counts = [70, 0, 33, 300]
    x, w = randn((sum(counts), K), torch.bfloat16, 31).to(DEV), randn((4, N, K), torch.bfloat16, 32).to(DEV)
    d_out = randn((sum(counts), N), torch.bfloat16, 33).to(DEV)
    w[1], w[3] = float("nan"), float("inf")
    x[70 + 33 + 5] = float("nan")
    (y, dx, dw), (sy, sx, sw) = R.grouped(x, w, counts, d_out)
    count = torch.tensor(counts, device=DEV)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fma.grouped_linear_fp8(a, b, count)
    out.backward(d_out)
    R.check_product(out.detach()[:103], y[:103], sy[:103], K)
    R.check_product(a.grad[:103], dx[:103], sx[:103], N)
    R.check_product(b.grad[:3], dw[:3], sw[:3], 70)
    assert bool(torch.isnan(out[103:]).all()) and bool(torch.isnan(a.grad[103:]).all())


def test_many_experts():
    import fma_b200 as fma

    E = 1024
    counts = [0] * E
    counts[0], counts[511], counts[512], counts[1022], counts[1023] = 3, 1, 20, 2, 130
    rows = sum(counts) + 2
    x, w = randn((rows, 16), torch.bfloat16, 28).to(DEV), randn((E, 8, 16), torch.bfloat16, 29).to(DEV)
    d_out = randn((rows, 8), torch.bfloat16, 30).to(DEV)
    (y, dx, dw), (sy, sx, sw) = R.grouped(x, w, counts, d_out)
    count = torch.tensor(counts, device=DEV)
    R.check_product(fma.grouped_linear_fp8(x, fma.quantize_fp8_weight(w), count), y, sy, 16)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = fma.grouped_linear_fp8(a, b, count)
    out.backward(d_out)
    R.check_product(out.detach(), y, sy, 16)
    R.check_product(a.grad, dx, sx, 8)
    R.check_product(b.grad, dw, sw, 130)


def test_swiglu_keeps_half_the_memory():
    import fma_b200 as fma

    gate, up = (randn((1024, 2048), torch.bfloat16, s).to(DEV).requires_grad_() for s in (22, 23))
    fma.swiglu_fp8_checkpoint(gate, up)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = fma.swiglu_fp8_checkpoint(gate, up)
    kept = torch.cuda.memory_allocated() - before - out.numel() * out.element_size()
    assert kept <= 1.02 * 2 * gate.numel()


# ---- streams, graphs, several calls at once --------------------------------------------------------
def _step(fma, x, w, count, d):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = fma.grouped_linear_fp8(a, b, count)
    z = fma.swiglu_fp8_checkpoint(y, y * 0.5)
    return (z.detach(), *torch.autograd.grad(z, (a, b), d))


def _problem(seed, rows=390):
    x, w = randn((rows, 264), torch.bfloat16, seed).to(DEV), randn((3, 136, 264), torch.bfloat16, seed + 1, scale=0.05).to(DEV)
    count = torch.tensor([rows - 150, 0, 150], dtype=torch.int32, device=DEV)
    return x, w, count, randn((rows, 136), torch.bfloat16, seed + 2).to(DEV)


def test_training_step_in_a_graph():
    """Captured, then replayed on other inputs while an eager step of the same leaves lives; two graphs in turn."""
    import fma_b200 as fma

    problems = [_problem(s) for s in (30, 40, 50)]
    want = [_step(fma, *p) for p in problems]
    eager = _step(fma, *problems[0])
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        static = [t.clone() for t in problems[0]]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(fma, *static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(fma, *static)
        graphs.append((graph, static, out))
    for i in (1, 2, 0):
        for graph, static, out in graphs:
            for s, t in zip(static, problems[i]):
                s.copy_(t)
            graph.replay()
        for _, _, out in graphs:
            for got, ref in zip(out, want[i]):
                assert torch.equal(got, ref)
    for got, ref in zip(eager, want[0]):
        assert torch.equal(got, ref)
    check_device_status()


def test_serving_in_a_graph_and_on_other_streams():
    import fma_b200 as fma

    w = randn((5, 264, 392), torch.float16, 60, scale=0.05).to(DEV)
    held = fma.quantize_fp8_weight(w)
    cases = []
    for rows, count in ((7, [1, 2, 0, 3, 1]), (333, [100, 0, 233, 0, 0])):
        x, c = randn((rows, 392), torch.float16, rows).to(DEV), torch.tensor(count, device=DEV)
        want = R.grouped(x, w, count, torch.zeros(rows, 264, device=DEV))
        cases.append((x, c, want[0][0], want[1][0]))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):  # at once
        with torch.cuda.stream(s):
            got.append([fma.grouped_linear_fp8(cases[(i + j) % 2][0], held, cases[(i + j) % 2][1]) for j in range(8)])
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for j, out in enumerate(outs):
            R.check_product(out, *cases[(i + j) % 2][2:], 392)
    x, c = cases[0][0].clone(), cases[0][1].clone()
    fma.grouped_linear_fp8(x, held, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fma.grouped_linear_fp8(x, held, c)
    x.copy_(cases[0][0].flip(0))
    c.copy_(torch.tensor([0, 0, 0, 0, 7]))
    graph.replay()
    want = R.grouped(x, w, [0, 0, 0, 0, 7], torch.zeros(7, 264, device=DEV))
    R.check_product(out, want[0][0], want[1][0], 392)
    check_device_status()


def test_results_do_not_change_between_runs():
    import fma_b200 as fma

    p = _problem(70)
    first = _step(fma, *p)
    for _ in range(5):
        for a, b in zip(first, _step(fma, *p)):
            assert torch.equal(a, b)


# ---- refusals --------------------------------------------------------------------------------------
def test_refusals():
    import fma_b200 as fma

    x, w = torch.zeros(4, 16, device=DEV, dtype=torch.bfloat16), torch.zeros(8, 16, device=DEV, dtype=torch.bfloat16)
    count = torch.tensor([2, 2], device=DEV)
    w3 = torch.zeros(2, 8, 16, device=DEV, dtype=torch.bfloat16)

    def refused(match, f, *args):
        with pytest.raises(RuntimeError, match=match):
            f(*args)

    refused("multiple of 8", fma.quantize_fp8, x[:, :12])
    refused("dtype", fma.quantize_fp8, x.int())
    refused("dimension", fma.quantize_fp8, x[0, 0])
    refused("multiple of 8", fma.quantize_fp8_weight, w[:4])
    refused("must be", fma.quantize_fp8_weight, w[0])
    refused("float16", fma.linear_fp8, x.float(), w.float())
    refused("weight torch.float16", fma.linear_fp8, x, w.half())
    refused("does not fit", fma.linear_fp8, x[:, :8], w)
    refused("weight shape", fma.linear_fp8, x, w3)
    refused("weight shape", fma.grouped_linear_fp8, x, w, count)
    refused("one count", fma.grouped_linear_fp8, x, w3, count[:1])
    refused("int32", fma.grouped_linear_fp8, x, w3, count.float())
    refused("must be", fma.grouped_linear_fp8, x[None], w3, count)
    refused("CUDA", fma.linear_fp8, x, w.cpu())
    refused("CUDA", fma.grouped_linear_fp8, x, w3, count.cpu())
    refused("quantize_fp8_weight", fma.linear_fp8, x, w, w)
    refused("shape", fma.linear_fp8, x, w, fma.quantize_fp8_weight(w3))
    refused("same shape", fma.swiglu_fp8_checkpoint, x, x[:2])
    refused("multiple of 8", fma.swiglu_fp8_checkpoint, x[:, :4], x[:, :4])
    refused("same shape, dtype", fma.swiglu_fp8_checkpoint, x, x.half())
