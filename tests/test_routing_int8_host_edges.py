"""Routing and 8-bit products without a GPU: refusals beyond those of test_routing_int8_host."""
import ctypes

import pytest
import torch

from moe_quant_amd import _lib, moe_layer, ops, quant_utils

F32, BF16, F16, I32 = torch.float32, torch.bfloat16, torch.float16, torch.int32


def test_combine_types():
    s, w = torch.zeros(3, 2, dtype=I32), torch.zeros(3, 2)
    for y, to in ((BF16, F32), (BF16, F16), (F16, BF16), (F16, F32), (F32, torch.float64), (F32, torch.int8)):
        with pytest.raises(ValueError):
            ops.combine_experts(torch.zeros(4, 8, dtype=y), s, w, to)
    for y, to in ((BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (F32, F16), (BF16, None)):
        with pytest.raises(_lib.MoeQuantHipError):  # fine but for the device
            ops.combine_experts(torch.zeros(4, 8, dtype=y), s, w, to)
    lib = _lib.load()
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    f32, bf16, f16 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_F16
    for y, to in ((bf16, f32), (bf16, f16), (f16, bf16), (f16, f32), (f32, 3), (f32, -1), (3, 3)):
        assert lib.mq_combine_experts_to(p, y, 8, 2, 8, p, p, 2, 2, p, to, 8, None) == _lib.MQ_ERR_ARG
    for y, to in ((bf16, bf16), (f32, bf16), (f32, f16), (f32, f32)):
        assert lib.mq_combine_experts_to(p, y, 8, 2, 8, p, p, 0, 2, p, to, 8, None) == _lib.MQ_OK
        assert lib.mq_combine_experts_to(p, y, 8, 2, 8, p, p, 2, 2, p, to, 7, None) == _lib.MQ_ERR_ARG


def test_grouped_tiles_beyond_32_bits_are_refused():
    """Offsets come from the device and may say that every expert has all rows: where the kernel could not count such tiles in 32
    bits, the call is refused before a device is looked for."""
    lib = _lib.load()
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)

    def grouped(S, E, N, swiglu=0, K=32):
        return lib.mq_matmul_int8_grouped(p, K, p, 4, p, S, p, K, N * K * (1 + swiglu), p, E, p, p, N, 1, N, K, swiglu, None)

    assert grouped(1 << 30, 1024, 8) == _lib.MQ_ERR_TOO_LARGE
    assert grouped(1 << 24, 1024, 16384) == _lib.MQ_ERR_TOO_LARGE
    assert grouped(1 << 24, 1024, 7168, 1) == _lib.MQ_ERR_TOO_LARGE


def test_linear_without_columns_is_refused_in_any_shape():
    for x in (torch.zeros(0), torch.zeros(2, 0), torch.zeros(2, 3, 0), torch.zeros(0, 3, 0)):
        with pytest.raises(ValueError):
            quant_utils.linear_int8(x, torch.zeros(6, 0, dtype=torch.int8), torch.zeros(6))
    with pytest.raises(_lib.MoeQuantHipError):  # no tokens, but columns: fine but for the device
        quant_utils.linear_int8(torch.zeros(0, 3, 32), torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6))


def test_experts_whose_halves_differ_are_refused():
    """Gate and up rows are stacked: with six and two of them the products would pair the wrong ones."""
    mk = lambda r, c: (torch.full((r, c), 8, dtype=torch.uint8), torch.ones(r, 1), torch.full((r, 1), 8.0))
    from_quantized = moe_layer.Int8Experts.from_quantized
    assert from_quantized([(mk(4, 8), mk(4, 8), mk(8, 4))]).gate_up.shape == (1, 8, 8)
    for bad in ((mk(6, 8), mk(2, 8), mk(8, 4)), (mk(4, 8), mk(4, 6), mk(8, 4)), (mk(4, 8), mk(4, 8), mk(8, 6)), (mk(4, 8), mk(4, 8), mk(6, 4))):
        with pytest.raises(ValueError):
            from_quantized([bad])
