"""The MoE layer with its experts on 8-bit operands, against the same chain of operators in 64 bits with the same
roundings (tests/_fp8_ref.py)."""

import copy

import pytest
import torch

import _fp8_ref as R
from _util import DEV, check_device_status, randn, rel_l2, to_np

pytestmark = pytest.mark.gpu

# Both sides round at the same places; they part where an fp32 sum and the exact one fall on different sides of a 16-bit
# rounding (a share of about 2^-10 of the elements in bfloat16, 2^-7 in half), which moves the element by a step, and its
# 8-bit form by a step of 2^-3 for 2^-4 (2^-7) of those: rel-L2 about sqrt(2^-14) * 2^-3 = 1e-3 per product, three of
# them in a row for the gradients, next to at most half a step (2^-8, 2^-11) for the last rounding.
TOL = {torch.bfloat16: 2.0**-8 + 4e-3, torch.float16: 2.0**-11 + 4e-3}


def _layer(E, k, H, I, dtype, seed=0, **kw):
    import fma_b200 as fma

    moe = fma.MoE(E, k, H, I, fma.swiglu_packed, True, False, 0.05)
    with torch.no_grad():
        for i, p in enumerate((moe.gate.weight, moe.c_fc.weight, moe.c_proj.weight)):
            p.copy_(randn(p.shape, torch.float32, seed + i, scale=0.1))
    moe = moe.to(DEV).to(dtype)
    moe.fp8_experts = True
    return moe


def _chain(x, weights, selected, w_fc, w_proj, dy):
    """(y, dx, d_weights, d_w_fc, d_w_proj) in 64 bits, rounded to the type where the layer rounds."""
    dtype, (T, k), (E, H, I) = x.dtype, selected.shape, w_proj.shape
    rnd = lambda t: t.to(dtype).double()  # noqa: E731
    hx, hdy = x.double(), dy.double()
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    dx, d_weights = torch.zeros_like(y), torch.zeros(T, k, dtype=torch.float64, device=x.device)
    d_fc, d_proj = torch.zeros(E, 2 * I, H, dtype=torch.float64, device=x.device), torch.zeros(E, H, I, dtype=torch.float64, device=x.device)
    for e in range(E):
        t, j = torch.nonzero(selected == e, as_tuple=True)
        if not len(t):
            continue
        fc, proj = R.hold(w_fc[e], 128), R.hold(w_proj[e], 128)
        xe = R.hold(x[t])
        pre = rnd(xe @ fc.T)
        up, gate = pre[:, :I], pre[:, I:]
        act = R.hold(rnd(up * gate * torch.sigmoid(gate)))
        out = rnd(act @ proj.T)
        w = weights.double()[t, j][:, None]
        y.index_add_(0, t, w * out)
        d_out = rnd(w * hdy[t])
        d_weights[t, j] = (out * hdy[t]).sum(1)
        d_proj[e] = d_out.T @ act
        d_act = rnd(R.hold(d_out) @ proj)
        u, g = R.hold(up), R.hold(gate)
        s = torch.sigmoid(g)
        d_pre = rnd(torch.cat([d_act * g * s, d_act * u * (s + g * s * (1 - s))], 1))
        d_fc[e] = d_pre.T @ xe
        dx.index_add_(0, t, rnd(R.hold(d_pre) @ fc))
    return y, dx, d_weights, d_fc, d_proj


def _fill_free_memory(byte):
    """The allocator's free blocks, small ones and large ones, hold this byte."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    blocks = [torch.full((n,), byte, dtype=torch.uint8, device=DEV) for n in [1 << 28] * 2 + [1 << 20] * 64 + [1 << 13] * 256]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("T,E,k,H,I", [(300, 4, 2, 264, 136), (2000, 5, 3, 256, 128)])
def test_rows_that_nothing_writes_are_not_read(T, E, k, H, I):
    """Padding rows of the grouped layout that stay as the allocator left them do not reach a result."""
    moe = _layer(E, k, H, I, torch.bfloat16)
    x, dy = randn((T, H), torch.bfloat16, 10).to(DEV), randn((T, H), torch.bfloat16, 11).to(DEV)
    results = []
    for byte in (0, 0xFF):  # zeros, and NaN in every type and scale
        a = x.clone().requires_grad_()
        moe.zero_grad(set_to_none=True)
        _fill_free_memory(byte)
        y, _ = moe(a)
        y.backward(dy)
        results.append([t.detach().clone() for t in (y, a.grad, moe.c_fc.weight.grad, moe.c_proj.weight.grad, moe.gate.weight.grad)])
    for one, other in zip(*results):
        assert bool(torch.isfinite(one).all()) and torch.equal(one, other)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", [(300, 4, 2, 264, 136), (37, 8, 3, 128, 256), (1, 4, 2, 136, 8), (700, 3, 1, 520, 392)])
def test_layer(dtype, T, E, k, H, I):
    from fma_b200.modules import _kernels as K

    moe = _layer(E, k, H, I, dtype)
    x, dy = randn((T, H), dtype, 10).to(DEV), randn((T, H), dtype, 11).to(DEV)
    weights, selected = K.router_topk_softmax(moe.gate(x).detach(), k)
    if E == 8:
        selected = torch.where(selected == 3, 4, selected)  # an expert without tokens, and a token with one expert twice
    want = _chain(x, weights, selected, moe.c_fc.weight.detach(), moe.c_proj.weight.detach(), dy)
    a, b = x.clone().requires_grad_(), weights.clone().requires_grad_()
    y = moe._compute_experts(a, b, selected)
    y.backward(dy)
    got = (y.detach(), a.grad, b.grad, moe.c_fc.weight.grad, moe.c_proj.weight.grad)
    errors = [rel_l2(to_np(g), to_np(w)) for g, w in zip(got, want)]
    assert all(e <= TOL[dtype] for e in errors), errors
    # serving: the same values without a graph, with weights quantised for the call and once for all
    with torch.no_grad():
        served = moe._compute_experts(x, weights, selected)
        moe.quantize_experts()
        assert torch.equal(moe._compute_experts(x, weights, selected), served)
    assert rel_l2(to_np(served), to_np(want[0])) <= TOL[dtype]
    check_device_status()


def test_layer_through_its_forward_and_a_step_of_training():
    moe = _layer(8, 2, 256, 128, torch.bfloat16)
    x = randn((4, 96, 256), torch.bfloat16, 12).to(DEV).requires_grad_()
    y, logits = moe(x)
    assert y.shape == x.shape and logits.shape == (384, 8)
    y.backward(randn((4, 96, 256), torch.bfloat16, 13).to(DEV))
    plain = copy.deepcopy(moe)
    plain.fp8_experts = False
    ref, _ = plain(x.detach())
    # A rounding to e4m3 is uniform in a step of 2^-3 of its binade: at most 2^-3 / sqrt(12) = 0.036 of the value in the
    # 2-norm.  up and gate are products of two such factors: sqrt(2) * 0.036 = 0.051.  act has up and silu(gate) as factors,
    # whose relative errors are 0.051 and about 1.05 * 0.051 (E[silu'^2] s^2 / E[silu^2] = 1.1 at s = 1.6): 0.074.  The down
    # projection adds the roundings of act and of its weight: sqrt(0.074^2 + 2 * 0.036^2) = 0.090.
    assert rel_l2(to_np(y), to_np(ref)) <= 0.09
    for p in (x, moe.gate.weight, moe.c_fc.weight, moe.c_proj.weight):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all())
    for tokens in (1, 3, 384):  # few and many rows per expert agree with the training forward
        with torch.no_grad():
            z, _ = moe(x.detach().reshape(-1, 256)[:tokens])
        assert rel_l2(to_np(z), to_np(y.reshape(-1, 256)[:tokens])) <= 2.0**-7
    check_device_status()


def test_layer_without_tokens():
    moe = _layer(4, 2, 64, 32, torch.bfloat16)
    y, _ = moe(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    assert y.shape == (0, 64)
    with torch.no_grad():
        assert moe(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))[0].shape == (0, 64)


def test_layer_keeps_fewer_bytes():
    def kept(fp8):
        moe = _layer(4, 2, 512, 512, torch.bfloat16)
        moe.fp8_experts = fp8
        x = randn((4096, 512), torch.bfloat16, 14).to(DEV)
        moe(x)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y, logits = moe(x)
        return torch.cuda.memory_allocated() - before, (y, logits)

    # 8192 routed rows: x, up, gate, act and out of 512 columns: 2 bytes each, against 1, 1, 1, 1 and 2
    rows = 8192 * 512
    assert kept(False)[0] - kept(True)[0] >= 0.9 * 4 * rows - 4 * 4 * 1536 * 512


def test_refusals():
    import fma_b200 as fma

    x = randn((5, 64), torch.bfloat16, 15).to(DEV)
    moe = _layer(4, 2, 64, 32, torch.bfloat16)
    with torch.no_grad():
        moe.quantize_experts()
        moe(x)
        moe.c_proj.weight.mul_(2)
        with pytest.raises(RuntimeError, match="have changed"):
            moe(x)
        moe.quantize_experts()
        moe(x)
        moe.half()
        with pytest.raises(RuntimeError, match="have changed"):
            moe(x.half())
    moe(x.half())  # with gradients the weights are always those of the call
    wide = fma.MoE(4, 2, 64, 32, fma.swiglu_packed, True, False, 0.05).to(DEV)
    wide.fp8_experts = True
    with pytest.raises(RuntimeError, match="bfloat16"):
        wide(x.float())
    biased = fma.MoE(4, 2, 64, 32, fma.swiglu_packed, True, True, 0.05).to(DEV).bfloat16()
    biased.fp8_experts = True
    with pytest.raises(RuntimeError, match="without bias"):
        biased(x)


def test_second_derivatives_are_refused():
    x = randn((300, 64), torch.bfloat16, 16).to(DEV).requires_grad_()
    moe = _layer(4, 2, 64, 32, torch.bfloat16)
    y, _ = moe(x)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    y, _ = moe(x)
    (d_x,) = torch.autograd.grad(y.sum(), x)
    assert bool(torch.isfinite(d_x).all()) and not d_x.requires_grad


def _refuses_until_quantized_again(moe, x):
    with torch.no_grad():
        for _ in range(2):
            with pytest.raises(RuntimeError, match="have changed"):
                moe(x)
        moe.quantize_experts()
        held, _ = moe(x)
        moe._held_experts = None
        assert torch.equal(held, moe(x)[0])
        moe.quantize_experts()


def test_experts_quantized_once_follow_the_weights_or_refuse():
    x = randn((5, 64), torch.bfloat16, 15).to(DEV)
    moe, other = _layer(4, 2, 64, 32, torch.bfloat16), _layer(4, 2, 64, 32, torch.bfloat16, seed=7)
    moe.quantize_experts()
    with torch.no_grad():
        first, _ = moe(x)
    # writes that the parameters count
    moe.load_state_dict(other.state_dict())
    _refuses_until_quantized_again(moe, x)
    optimizer = torch.optim.SGD(moe.parameters(), lr=0.1)
    moe(x)[0].sum().backward()
    optimizer.step()
    _refuses_until_quantized_again(moe, x)
    # other parameters: of three sets one after the other the third may get the memory of the first
    shape = moe.c_fc.weight.shape
    first_set = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    moe.c_fc.weight = torch.nn.Parameter(first_set)
    moe.quantize_experts()
    del first_set
    for fill in (1.0, 2.0):
        moe.c_fc.weight = torch.nn.Parameter(torch.full(shape, fill, dtype=torch.bfloat16, device=DEV))
    _refuses_until_quantized_again(moe, x)
    # moved away and back
    moe.cpu()
    moe.cuda()
    _refuses_until_quantized_again(moe, x)
    # a copy has the same weights, whatever it holds, and follows its own
    twin = copy.deepcopy(moe)
    with torch.no_grad():
        twin.c_proj.weight.mul_(2)
        moe(x)
    _refuses_until_quantized_again(twin, x)
    assert first.shape == x.shape


def test_writes_through_data_are_seen_after_the_next_call():
    """What the documentation of quantize_experts says of writes that torch does not count."""
    x = randn((5, 64), torch.bfloat16, 15).to(DEV)
    moe = _layer(4, 2, 64, 32, torch.bfloat16)
    moe.quantize_experts()
    with torch.no_grad():
        before, _ = moe(x)
        moe.c_proj.weight.data.mul_(2)
        assert torch.equal(moe(x)[0], before)
        moe.quantize_experts()
        assert torch.equal(moe(x)[0], 2 * before)  # a power of two: every rounding is the same


def test_parameters_made_in_inference_mode():
    x = randn((5, 64), torch.bfloat16, 15).to(DEV)
    with torch.inference_mode():
        moe = _layer(4, 2, 64, 32, torch.bfloat16)
        assert moe.c_fc.weight.is_inference()
        want, _ = moe(x)
        moe.quantize_experts()
        assert torch.equal(moe(x)[0], want)


def test_old_weights_are_let_go_when_the_layer_moves():
    moe = _layer(4, 2, 512, 512, torch.bfloat16)
    moe.quantize_experts()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    moe.cpu()
    gone = before - torch.cuda.memory_allocated()
    assert gone >= 3 * 4 * 512 * 512 * (2 + 1)  # in 16 bits and in 8


def test_serving_keeps_nothing_for_a_backward_pass(monkeypatch):
    from fma_b200.modules import _fp8_experts

    calls = []

    def record(name, *args):
        if name == "fma_b200_swiglu_fp8_forward":
            calls.append([a is not None for a in args[10:14]])  # gate and up in 8 bits, and their scales
        return call(name, *args)

    call = _fp8_experts.call
    monkeypatch.setattr(_fp8_experts, "call", record)
    x = randn((300, 64), torch.bfloat16, 17).to(DEV)
    moe = _layer(4, 2, 64, 32, torch.bfloat16)
    with torch.no_grad():
        served, _ = moe(x)
    trained, _ = moe(x)
    moe.requires_grad_(False)
    frozen, _ = moe(x)
    assert calls == [[False] * 4, [True] * 4, [False] * 4]
    assert torch.equal(served, trained) and torch.equal(served, frozen)
