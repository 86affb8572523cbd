"""The 8-bit operators without a GPU: refusals of the C entry points (checked before any CUDA call), sizes, and the
definition that the GPU tests compare with against torch's own e4m3 conversion."""

import ctypes

import pytest
import torch

import _fp8_ref as R


def test_entry_points_refuse_bad_arguments():
    from fma_b200 import _native

    lib = _native.lib()
    null, at = ctypes.c_void_p(None), ctypes.c_void_p(16)
    odd = ctypes.c_void_p(24)
    OK, BAD, UNSUPPORTED = 0, 1, 2
    assert lib.fma_b200_fp8_scale_bytes(1, 8) == 512
    assert lib.fma_b200_fp8_scale_bytes(129, 513) == 4 * 512
    assert lib.fma_b200_fp8_scale_bytes(0, 4096) == 0
    assert lib.fma_b200_fp8_scale_bytes(-1, 8) == 0
    q = lib.fma_b200_fp8_quantize_rows
    assert q(at, 16, 7, 4, 16, null, at, at, null) == UNSUPPORTED
    assert q(at, 16, 1, 4, 12, null, at, at, null) == BAD  # width
    assert q(at, 8, 1, 4, 16, null, at, at, null) == BAD  # pitch below the width
    assert q(at, 20, 1, 4, 16, null, at, at, null) == BAD  # pitch not whole 16 bytes
    assert q(null, 16, 1, 4, 16, null, at, at, null) == BAD
    assert q(odd, 16, 1, 4, 16, null, at, at, null) == BAD
    assert q(at, 16, 1, -1, 16, null, at, at, null) == BAD
    assert q(null, 16, 1, 0, 16, null, null, null, null) == OK
    g = lib.fma_b200_fp8_quantize_groups
    assert g(at, 16, 1, 4, 16, at, at, 0, 256, at, at, null, null) == BAD
    assert g(at, 16, 1, 4, 16, null, at, 2, 256, at, at, null, null) == BAD
    assert g(at, 16, 1, 4, 16, at, at, 2, 256, at, at, odd, null) == BAD
    s = lib.fma_b200_fp8_quantize_scatter
    assert s(at, 1, 4, 16, 0, at, at, at, 2, 256, at, at, null) == BAD  # k
    assert s(at, 1, 4, 16, 2, at, null, at, 2, 256, at, at, null) == BAD
    w = lib.fma_b200_fp8_quantize_weight
    assert w(at, 1, 1, 12, 16, at, at, null) == BAD  # N
    assert w(at, 1, 2000, 16, 16, at, at, null) == BAD  # E
    assert w(at, 1, 1, 16, 16, at, null, null) == BAD
    assert w(at, 1, 1024, 1 << 22, 16, at, at, null) == BAD  # E * N
    d = lib.fma_b200_fp8_dequantize
    assert d(at, at, 0, 4, 16, null, at, 1, null) == BAD
    assert d(at, at, 1, 4, 16, null, at, 5, null) == UNSUPPORTED
    assert d(at, null, 1, 4, 16, null, at, 1, null) == BAD
    m = lib.fma_b200_fp8_group_maps
    assert m(at, 2, 4, 100, 2048, at, at, at, at, at, at, null) == UNSUPPORTED
    assert m(at, 4, 4, 100, 1024, at, at, at, at, at, at, null) == BAD  # layout too small: 256 + 4 * 256
    assert m(at, 4, 1025, 100, 1 << 20, at, at, at, at, at, at, null) == BAD
    assert m(null, 4, 4, 100, 2048, at, at, at, at, at, at, null) == BAD
    p = lib.fma_b200_fp8_gemm
    assert p(at, at, 256, at, at, 1, 16, 16, at, 0, 256, null, null, null, null, null, null, null) == UNSUPPORTED  # fp32 result
    assert p(at, at, 256, at, at, 2, 16, 16, at, 1, 256, null, null, null, null, null, null, null) == BAD  # experts without a table
    assert p(at, at, 256, at, at, 1, 12, 16, at, 1, 256, null, null, null, null, null, null, null) == BAD
    assert p(at, at, 256, at, at, 1, 16, 20, at, 1, 256, null, null, null, null, null, null, null) == BAD
    assert p(at, null, 256, at, at, 1, 16, 16, at, 1, 256, null, null, null, null, null, null, null) == BAD
    assert p(null, null, 0, null, null, 1, 16, 16, null, 1, 0, null, null, null, null, null, null, null) == OK
    g = lib.fma_b200_fp8_gemm_dgrad
    assert g(at, at, 256, at, at, 1, 16, 16, at, 0, 256, null, null, null, null, null, null, null) == UNSUPPORTED  # fp32 result
    assert g(at, at, 256, at, at, 2, 16, 16, at, 1, 256, null, null, null, null, null, null, null) == BAD  # experts without a table
    assert g(at, at, 256, at, odd, 1, 16, 16, at, 1, 256, null, null, null, null, null, null, null) == BAD
    assert g(at, at, 256, at, at, 1024, 1 << 22, 16, at, 1, 256, at, null, null, null, null, null, null) == BAD  # E * N
    assert g(null, null, 0, null, null, 1, 16, 16, null, 1, 0, null, null, null, null, null, null, null) == OK
    for call in (p, g):
        assert call(at, at, 256, at, at, 2, 16, 16, at, 1, 256, at, null, null, null, at, null, null) == BAD  # offsets without counts
        assert call(at, at, 256, at, at, 2, 16, 16, at, 1, 256, at, at, at, null, at, at, null) == BAD  # both kinds
        assert call(at, at, 256, at, at, 1, 16, 16, at, 1, 256, null, null, null, null, at, at, null) == BAD
    f = lib.fma_b200_fp8_few_rows
    assert f(at, 16, 0, 4, at, at, 1, 16, 16, null, 4, at, null) == UNSUPPORTED
    assert f(at, 8, 1, 4, at, at, 1, 16, 16, null, 4, at, null) == BAD
    assert f(at, 16, 1, 4, at, at, 3, 16, 16, null, 4, at, null) == BAD  # experts without counts
    assert f(at, 16, 1, 4, at, at, 3, 16, 16, at, 2, at, null) == UNSUPPORTED
    assert f(at, 16, 1, 4, null, at, 1, 16, 16, null, 4, at, null) == BAD
    assert f(null, 16, 1, 0, null, null, 1, 16, 16, null, 4, null, null) == OK
    v = lib.fma_b200_linear_wgrad
    assert v(at, at, at, 0, 4, 1, 16, 16, at, null, null) == UNSUPPORTED
    assert v(at, at, at, 1, 0, 1, 16, 16, at, null, null) == BAD
    assert v(at, at, at, 1, 4, 2, 16, 16, null, null, null) == BAD  # several experts without offsets
    assert v(at, null, at, 1, 4, 1, 16, 16, null, null, null) == BAD
    fw, bw = lib.fma_b200_swiglu_fp8_forward, lib.fma_b200_swiglu_fp8_backward
    assert fw(at, 16, at, 16, at, 16, 1, 4, 12, null, at, at, at, at, null, null, null) == BAD
    assert fw(at, 16, at, 16, at, 16, 1, 4, 16, null, at, null, at, at, null, null, null) == BAD  # values without scales
    assert fw(at, 16, null, 16, at, 16, 1, 4, 16, null, at, at, at, at, null, null, null) == BAD
    assert bw(at, at, at, null, at, 16, at, 16, at, 16, 1, 4, 16, null, null, null, null) == BAD
    assert bw(at, at, at, at, at, 12, at, 16, at, 16, 1, 4, 16, null, null, null, null) == BAD
    assert bw(at, at, at, at, at, 16, at, 16, at, 16, 1, 4, 16, null, at, at, null) == BAD  # grad8: width
    assert bw(at, at, at, at, at, 128, at, 128, at, 128, 1, 4, 128, null, at, null, null) == BAD


def test_operators_need_cuda_tensors():
    import fma_b200 as fma

    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    for call in (lambda: fma.quantize_fp8(x), lambda: fma.quantize_fp8_weight(w), lambda: fma.linear_fp8(x, w),
                 lambda: fma.grouped_linear_fp8(x, w[None], torch.tensor([4])),
                 lambda: fma.swiglu_fp8_checkpoint(x, x)):  # fmt: skip
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_layer_switch_is_off_and_leaves_the_state_dict_alone():
    import fma_b200 as fma

    moe = fma.MoE(4, 2, 32, 16, fma.swiglu_packed, True, False, 0.02)
    assert moe.fp8_experts is False
    keys = list(moe.state_dict())
    moe.fp8_experts = True
    assert list(moe.state_dict()) == keys


@pytest.mark.parametrize("tall", [1, 128])
def test_definition_against_torchs_conversion(tall):
    x = torch.randn(200, 300, generator=torch.Generator().manual_seed(3)) * torch.exp2(torch.arange(200.0) / 8 - 12)[:, None]
    x[7] = 0
    held = R.hold(x, tall)
    for r in range(0, 200, tall):
        for c in range(0, 300, 128):
            part = x[r : r + tall, c : c + 128]
            amax = float(part.abs().max())
            e = 0
            if amax > 0:
                e = -60
                while amax > 448 * 2.0**e:
                    e += 1
            want = (part * 2.0**-e).to(torch.float8_e4m3fn).double() * 2.0**e
            assert torch.equal(held[r : r + tall, c : c + 128], want)


def test_tangents_are_refused():
    """A dual tensor need not require a gradient; its tangent must not get lost on the way without an autograd node."""
    import torch.autograd.forward_ad as fwd

    import fma_b200 as fma

    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    moe = fma.MoE(2, 1, 16, 8, fma.swiglu_packed, True, False, 0.02).bfloat16()
    moe.fp8_experts = True
    with fwd.dual_level():
        dx, dw = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for call in (lambda: fma.linear_fp8(dx, w), lambda: fma.linear_fp8(x, dw),
                     lambda: fma.grouped_linear_fp8(dx, w[None], torch.tensor([4])),
                     lambda: fma.grouped_linear_fp8(x, dw[None], torch.tensor([4])),
                     lambda: fma.swiglu_fp8_checkpoint(dx, x), lambda: fma.swiglu_fp8_checkpoint(x, dx),
                     lambda: moe._compute_experts(dx, torch.ones(4, 1).bfloat16(), torch.zeros(4, 1, dtype=torch.int64))):  # fmt: skip
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        for call in (lambda: fma.linear_fp8(x, w), lambda: fma.swiglu_fp8_checkpoint(x, x)):
            with pytest.raises(RuntimeError, match="CUDA"):  # without a tangent the call goes on
                call()


def test_second_derivatives_of_the_experts_are_refused():
    from fma_b200.modules._fp8_experts import Fp8SwigluExperts

    with torch.enable_grad(), pytest.raises(RuntimeError, match="once"):  # how the engine calls it under create_graph=True
        Fp8SwigluExperts.backward(None, torch.zeros(1))


def test_kinds_of_counts():
    from fma_b200 import _native

    lib = _native.lib()
    null, at, odd = ctypes.c_void_p(None), ctypes.c_void_p(16), ctypes.c_void_p(24)
    for index_bytes in (0, 2, -2, -8):
        assert lib.fma_b200_fp8_group_maps(at, index_bytes, 4, 100, 2048, at, at, at, at, at, at, null) == 2
        assert lib.fma_b200_fp8_few_rows(at, 16, 1, 4, at, at, 3, 16, 16, at, index_bytes, at, null) == 2
    for index_bytes in (4, 8, -4):  # accepted: what is refused is the next argument
        assert lib.fma_b200_fp8_group_maps(at, index_bytes, 4, 100, 1024, at, at, at, at, at, at, null) == 1
        assert lib.fma_b200_fp8_few_rows(odd, 16, 1, 4, at, at, 3, 16, 16, at, index_bytes, at, null) == 1


# (experts, N, K, rows, us of the product in one launch, us with a launch that quantises): what the rule's comment quotes
FEW = [(1, 14336, 4096, 1, 14.6, 19.0), (1, 14336, 4096, 16, 18.6, 19.3), (1, 14336, 4096, 24, 27.3, 19.4), (1, 28672, 4096, 8, 30.3, 31.1),
       (1, 28672, 4096, 16, 35.1, 31.3), (1, 32768, 8192, 1, 53.4, 54.8), (1, 32768, 8192, 8, 58.2, 55.2), (1, 8192, 28672, 1, 73, 47),
       (2, 14336, 4096, 4, 28.6, 38.3), (2, 14336, 4096, 24, 34.6, 37.7), (2, 14336, 4096, 48, 50.3, 37.4), (8, 14336, 4096, 8, 59.5, 63.4),
       (8, 14336, 4096, 128, 130, 98), (8, 4096, 4096, 64, 33.8, 39.0), (32, 8192, 4096, 64, 183, 169), (32, 8192, 4096, 384, 246, 186),
       (32, 1536, 2048, 384, 28.2, 33.4), (128, 1536, 2048, 8, 11.5, 18.9), (128, 1536, 2048, 512, 73, 89), (128, 2048, 768, 64, 24.7, 30.2),
       (128, 2048, 768, 512, 58.9, 52.1), (128, 4096, 4096, 8, 32, 40), (128, 4096, 4096, 64, 173, 152)]  # fmt: skip


@pytest.mark.parametrize("E,N,K,rows,one,two", FEW)
def test_the_faster_product_is_taken(E, N, K, rows, one, two):
    from fma_b200 import _native

    # 2 to 3 % are what two runs differ by: no matter
    assert _native.binding().few(rows, E, [(N, K)]) == (one < two) or abs(one - two) <= 0.03 * min(one, two)


def test_both_products_of_the_layer_go_one_way():
    from fma_b200 import _native

    few = _native.binding().few
    fine, wide = [(1536, 2048), (2048, 768)], [(28672, 4096), (4096, 14336)]
    assert [few(8 * tokens, 128, fine) for tokens in (1, 64, 96, 192)] == [True, True, True, False]
    assert [few(2 * tokens, 8, wide) for tokens in (1, 4, 16, 64)] == [True, True, False, False]
    assert not few(17 * 4, 4, [(8, 8)]) and not few(1, 1, [(8, (1 << 16) + 8)])


def test_what_was_loaded_to_the_cpu_stays_there():
    import fma_b200 as fma

    held = fma.Fp8Blocks.__new__(fma.Fp8Blocks)  # as unpickling makes it
    held.__setstate__((torch.zeros(16 * 16 + 512, dtype=torch.uint8), 16, 16, [16, 16], 15))
    assert held.device.type == "cpu" and held.shape == (16, 16) and held.dtype == torch.bfloat16 and held.nbytes == 768
    weight = fma.Fp8Weight.__new__(fma.Fp8Weight)
    weight.__setstate__((torch.zeros(16 * 16 + 512, dtype=torch.uint8), [16, 16], 15, 1, 16, 16))
    for other in (held, weight):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            other.dequantize()
