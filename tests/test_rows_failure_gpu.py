"""The abort path of the row-scaled and grouped products: with a wait limit far
below what a product takes its waits run out; the kernel records the failure,
waits (bounded) for its own copies, MMAs and launch-control answer, frees its
tensor memory and returns.  The failure is reported once, and with the default
limit the same product is right again."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
LIMIT_NS = 1000


def T():
    import tensorcoreptx_b200 as t
    return t


def randn(*shape):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    return torch.randn(*shape, generator=g, device=DEV).to(BF16)


def bounds(*edges):
    return torch.tensor(edges, dtype=torch.int32, device=DEV)


def grouped(rows, edges, n, k, out):
    A, W, o = randn(rows, k), randn(len(edges) - 1, n, k), bounds(*edges)
    return lambda: T().gemm_grouped(A, W, o, out_dtype=out)


def layer(rows, n, k):
    x, W = randn(rows, k), randn(n, k)
    return lambda: T().linear(x, W)


def int8_layer(rows, n, k):
    x = randn(rows, k)
    B, sb = T().quantize_rows_int8(randn(n, k))
    return lambda: T().linear_int8(x, B, sb)


def gradient(rows, n, k):
    dy, x, o = randn(rows, n), randn(rows, k), bounds(0, rows)
    return lambda: T().gemm_grouped_wgrad(dy, x, o)


# each way a product is laid out on the GPU: tile, CTAs that share a sum, the call
FORMS = {
    "one CTA a tile": (64, 1, lambda: layer(40, 2304, 16384)),
    "split sum": (64, 4, lambda: layer(40, 2304, 32768)),
    "split int8 sum, early start": (16, 2, lambda: int8_layer(40, 2304, 32768)),
    "fp32 in chunks, 16 rows": (16, 1, lambda: grouped(40, [1, 9, 9, 39], 2304, 8192, F32)),
    "fp32 in chunks, 128 rows": (128, 1, lambda: grouped(2400, [3, 1000, 1000, 2390], 2304, 8192, F32)),
    "split gradient": (128, 2, lambda: gradient(16384, 1024, 512)),
    "256 rows, every so manieth tile": (256, 1, lambda: grouped(9000, [3, 4000, 4000, 8990], 2304, 2048, BF16)),
    "256 rows, taken over": (256, 1, lambda: layer(16384, 2304, 2048)),
    "256 rows int8, taken over, early start": (256, 1, lambda: int8_layer(9600, 2304, 8192)),
    "256 rows gradient, taken over": (256, 1, lambda: gradient(16384, 4096, 4096)),
}


@pytest.mark.parametrize("name", list(FORMS))
def test_wait_expiry_aborts_cleanly(name):
    from tensorcoreptx_b200 import _native as nat
    L = nat.lib()
    tile, split, make = FORMS[name]
    call = make()
    stream = torch.cuda.current_stream().cuda_stream
    T().set_rows_tile(tile, split)
    try:
        want = call()
        assert L.tcg_check_device_error(stream, None) == 0
        word = C.c_uint64(0)
        L.tcg_set_wait_timeout_ns(LIMIT_NS)
        try:
            for _ in range(3):  # one behind the other
                call()
            st = L.tcg_check_device_error(stream, C.byref(word))
        finally:
            L.tcg_set_wait_timeout_ns(0)  # the default limit
        # (a sum in chunks waits for one chunk at a time, and the hardware's own
        # wait may outlast that)
        assert st == nat.TCG_ERR_TIMEOUT or (st == 0 and "chunks" in name)
        assert st == 0 or (word.value >> 32) == 1
        torch.cuda.synchronize()  # no CUDA error: the kernels returned
        assert L.tcg_check_device_error(stream, None) == 0  # reported once
        assert torch.equal(call(), want)
        assert L.tcg_check_device_error(stream, None) == 0
    finally:
        T().set_rows_tile(0, 0)


def test_failures_of_both_kinds_of_kernel_are_reported_by_one_check():
    """The dense kernels and these have a failure word each; a check reports the
    dense one first and leaves neither behind."""
    from tensorcoreptx_b200 import _native as nat
    L = nat.lib()
    call = layer(16384, 2304, 2048)
    call()
    stream = torch.cuda.current_stream().cuda_stream
    assert L.tcg_check_device_error(stream, None) == 0
    L.tcg_set_wait_timeout_ns(LIMIT_NS)
    try:
        call()
    finally:
        L.tcg_set_wait_timeout_ns(0)
    assert L.tcg_selftest_wait_timeout(1_000_000, stream) == 0  # 1 ms, in the dense kernels' file
    word = C.c_uint64(0)
    assert L.tcg_check_device_error(stream, C.byref(word)) == nat.TCG_ERR_TIMEOUT
    assert (word.value >> 32) == 1 and (word.value & 0xFF) in (0xFF, 0xFE)  # the self test's code
    assert L.tcg_check_device_error(stream, C.byref(word)) == 0 and word.value == 0
