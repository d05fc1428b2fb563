"""Refusals of the row-scaled and grouped products, on the CPU: the C entries'
status codes before any device access, and the Python surface's checks."""
import pytest
import torch

OK, SHAPE, ALIGN, ARG, WORKSPACE = 0, 1, 2, 5, 7


def L():
    from tensorcoreptx_b200 import _native
    return _native.lib()


def test_empty_results_succeed_without_a_device():
    assert L().tcg_quantize_rows_s8(None, 0, None, None, 0, 16, None) == OK
    assert L().tcg_gemm_s8_scaled(None, None, None, 1, 0, 8, 16, 1, None, None, None, None) == OK
    assert L().tcg_gemm_s8_grouped(None, None, None, 1, None, 1, 8, 0, 16, None, None, None, 1, None) == OK
    assert L().tcg_gemm_16_grouped(None, None, 1, None, 1, None, 1, 0, 8, 8, 1, 0, None) == OK
    assert L().tcg_gemm_16_grouped_wgrad(None, None, 1, None, 1, None, 0, 4, 8, 8, None) == OK
    assert L().tcg_dequantize_rows_s8(None, None, None, 1, 4, 0, None) == OK
    assert L().tcg_linear_s8(None, 1, None, None, 1, 0, 8, 16, None, None, None, 0, None) == OK


def test_quantize_rows_refusals():
    f = L().tcg_quantize_rows_s8
    assert f(16, 3, 16, 16, 4, 8, None) == ARG
    assert f(16, 0, 16, 16, -1, 8, None) == SHAPE
    assert f(16, 0, 16, 16, 4, -8, None) == SHAPE
    assert f(16, 0, 16, None, 4, 8, None) == ARG
    assert f(None, 0, 16, 16, 4, 8, None) == ARG
    assert f(16, 0, None, 16, 4, 8, None) == ARG
    assert f(18, 0, 16, 16, 4, 8, None) == ALIGN
    assert f(17, 1, 16, 16, 4, 8, None) == ALIGN
    assert f(16, 0, 16, 18, 4, 8, None) == ALIGN


def test_dequantize_rows_refusals():
    f = L().tcg_dequantize_rows_s8  # codes scale dst type rows k stream
    ok = [16, 16, 16, 1, 4, 8, None]
    for i, v, st in ((3, 3, ARG), (4, -1, SHAPE), (5, -1, SHAPE), (0, None, ARG), (1, None, ARG), (2, None, ARG),
                     (1, 18, ALIGN), (2, 17, ALIGN)):
        args = list(ok)
        args[i] = v
        assert f(*args) == st, (i, v)


def test_int8_product_refusals():
    f = L().tcg_gemm_s8_scaled  # A B C type M N K batches scale_a scale_b bias stream
    assert f(16, 16, 16, 3, 4, 4, 16, 1, 16, 16, None, None) == ARG
    assert f(16, 16, 16, 1, -4, 4, 16, 1, 16, 16, None, None) == SHAPE
    assert f(16, 16, 16, 1, 4, 4, 16, -1, 16, 16, None, None) == SHAPE
    assert f(16, 16, 16, 1, 4, 4, 24, 1, 16, 16, None, None) == SHAPE
    assert f(16, 16, 16, 1, 4, 4, 0, 1, 16, 16, None, None) == SHAPE
    assert f(16, 16, 16, 1, 4, 4, 16, 65536, 16, 16, None, None) == SHAPE
    assert f(16, 16, 16, 1, 1 << 30, 4, 16, 4, 16, 16, None, None) == SHAPE  # 2^32 rows
    assert f(16, 16, 16, 1, 4, 4, 131072, 1, 16, 16, None, None) == SHAPE  # a sum could pass 2^31
    for i in (0, 1, 2, 8, 9):
        args = [16, 16, 16, 1, 4, 4, 16, 1, 16, 16, None, None]
        args[i] = None
        assert f(*args) == ARG, i
    for i, at in ((0, 24), (1, 24), (2, 17), (8, 18), (9, 18), (10, 18)):
        args = [16, 16, 16, 1, 4, 4, 16, 1, 16, 16, None, None]
        args[i] = at
        assert f(*args) == ALIGN, i
    g = L().tcg_gemm_s8_grouped  # A B C type offsets groups M N K scale_a scale_b bias rest stream
    assert g(16, 16, 16, 1, 16, 0, 4, 4, 16, 16, 16, None, 1, None) == SHAPE
    assert g(16, 16, 16, 1, 16, 1025, 4, 4, 16, 16, 16, None, 1, None) == SHAPE
    assert g(16, 16, 16, 1, None, 3, 4, 4, 16, 16, 16, None, 1, None) == SHAPE
    assert g(16, 16, 16, 1, 18, 3, 4, 4, 16, 16, 16, None, 1, None) == ALIGN


def test_linear_int8_refusals():
    f = L().tcg_linear_s8  # x type B C type M N K scale_b bias workspace bytes stream
    need = L().tcg_linear_s8_workspace_size(5, 16)
    assert need == 512 and L().tcg_linear_s8_workspace_size(0, 16) == 0
    assert L().tcg_linear_s8_workspace_size(1 << 20, 1 << 14) == (1 << 34) + (1 << 22)
    ok = [16, 1, 16, 16, 1, 5, 4, 16, 16, None, 256, need, None]  # more rows than a product quantises itself
    for i, v, st in ((1, 3, ARG), (4, -1, ARG), (0, None, ARG), (2, None, ARG), (3, None, ARG), (8, None, ARG),
                     (10, None, WORKSPACE), (11, need - 1, WORKSPACE), (10, 128, ALIGN), (0, 17, ALIGN), (2, 24, ALIGN),
                     (7, 8, SHAPE), (7, 131072, SHAPE), (5, -1, SHAPE)):
        args = list(ok)
        args[i] = v
        assert f(*args) == st, (i, v)


def test_16_bit_refusals():
    f = L().tcg_gemm_16_grouped  # A B type C type offsets groups M N K layout rest stream
    ok = [16, 16, 1, 16, 1, 16, 2, 4, 8, 8, 1, 1, None]
    for i, v, st in ((2, 0, ARG), (2, 3, ARG), (4, 3, ARG), (10, 2, ARG), (0, None, ARG), (1, None, ARG), (3, None, ARG),
                     (6, 0, SHAPE), (6, 1025, SHAPE), (9, 12, SHAPE), (9, 0, SHAPE), (7, -1, SHAPE), (0, 24, ALIGN),
                     (1, 24, ALIGN), (3, 17, ALIGN), (5, 17, ALIGN)):
        args = list(ok)
        args[i] = v
        assert f(*args) == st, (i, v)
    kn = list(ok)
    kn[10], kn[8] = 0, 12
    assert f(*kn) == SHAPE  # N of a K x N operand
    w = L().tcg_gemm_16_grouped_wgrad  # dC A type dB type offsets groups M N K stream
    ok = [16, 16, 1, 16, 1, 16, 2, 4, 8, 16, None]
    for i, v, st in ((2, 0, ARG), (4, 3, ARG), (0, None, ARG), (1, None, ARG), (3, None, ARG), (6, 1025, SHAPE),
                     (8, 4, SHAPE), (9, 12, SHAPE), (7, -1, SHAPE), (0, 24, ALIGN), (1, 24, ALIGN), (3, 17, ALIGN)):
        args = list(ok)
        args[i] = v
        assert w(*args) == st, (i, v)


def test_python_surface_refuses_cpu_tensors_and_wrong_types():
    import tensorcoreptx_b200 as T
    i8, f16, f32 = torch.int8, torch.float16, torch.float32
    o = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="contiguous CUDA"):
        T.quantize_rows_int8(torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.gemm_int8_scaled(torch.zeros(4, 16, dtype=i8), torch.zeros(4, 16, dtype=i8), torch.zeros(4), torch.zeros(4))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.linear_int8(torch.zeros(4, 16), torch.zeros(4, 16, dtype=i8), torch.zeros(4))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.linear_int8_grouped(torch.zeros(4, 16), torch.zeros(2, 4, 16, dtype=i8), o, torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.gemm_int8_grouped(torch.zeros(4, 16, dtype=i8), torch.zeros(2, 4, 16, dtype=i8), o, torch.zeros(4),
                            torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.gemm_grouped(torch.zeros(4, 16, dtype=f16), torch.zeros(2, 4, 16, dtype=f16), o)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.gemm_grouped_wgrad(torch.zeros(4, 16, dtype=f16), torch.zeros(4, 16, dtype=f16), o)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        T.linear(torch.zeros(4, 16, dtype=f16), torch.zeros(8, 16, dtype=f16))
    with pytest.raises(RuntimeError, match="W 3-D"):
        T.linear_grouped(torch.zeros(4, 16, dtype=f32), torch.zeros(8, 16, dtype=f32), o)
