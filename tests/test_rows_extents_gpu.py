"""Extents that the other tests leave out: rows and results beyond 2^31 elements,
and groups of equal size without offsets (the C ABI's NULL) in 16 bits.

The large tests use small whole numbers, whose sums fp32 holds exactly, so that
results have to be equal; 4099 different rows in turn, so that an index that wraps
does not meet the same row again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PERIOD, LONG, WIDE = 4099, 1_050_011, 2064  # LONG * WIDE = 2.17e9


def T():
    import tensorcoreptx_b200 as t
    return t


@pytest.fixture(autouse=True)
def _clean():
    torch.cuda.empty_cache()
    yield
    T().set_rows_tile(0, 0)
    assert T().check_device_error() == 0
    torch.cuda.empty_cache()


def whole(g, *shape, most=1):
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).to(BF16)


def in_turn(base, rows):
    """Rows of base over and over: base[i % PERIOD]."""
    return base.repeat((rows + PERIOD - 1) // PERIOD, 1)[:rows].contiguous()


def equal_in_turn(got, base):
    """got[i] == base[i % PERIOD], block by block."""
    return all(torch.equal(got[i:i + PERIOD], base[:got.size(0) - i]) for i in range(0, got.size(0), PERIOD))


@pytest.mark.parametrize("tile", [0, 16, 256])
def test_a_long_result(tile):
    g = torch.Generator(device=DEV).manual_seed(1)
    base, W = whole(g, PERIOD, 16), whole(g, 2, WIDE, 16)
    at = PERIOD * 200 + 7
    o = torch.tensor([0, at, LONG - 3], dtype=torch.int32, device=DEV)
    T().set_rows_tile(tile, 0)
    C = T().gemm_grouped(in_turn(base, LONG), W, o)
    want = [(base.float() @ W[e].float().t()).to(BF16) for e in range(2)]
    assert equal_in_turn(C[:at], want[0])
    assert equal_in_turn(C[at:LONG - 3], want[1].roll(-7, 0))
    assert (C[LONG - 3:] == 0).all()


def test_long_rows_in_a_product_and_its_weight_gradient():
    g = torch.Generator(device=DEV).manual_seed(2)
    base, W = whole(g, PERIOD, WIDE), whole(g, 1, 24, WIDE)
    x = in_turn(base, LONG)
    o = torch.tensor([0, LONG], dtype=torch.int32, device=DEV)
    C = T().gemm_grouped(x, W, o, out_dtype=F32)
    assert equal_in_turn(C, base.float() @ W[0].float().t())
    del C
    dbase = whole(g, PERIOD, 16)
    times = torch.full((PERIOD, 1), LONG // PERIOD, device=DEV)  # how often each row occurs
    times[:LONG % PERIOD] += 1
    want = dbase.double().t() @ (base.double() * times)  # below 2^24: exact in fp32
    assert want.abs().max() < 2 ** 24
    assert torch.equal(T().gemm_grouped_wgrad(in_turn(dbase, LONG), x, o, out_dtype=F32)[0].double(), want)


def test_long_rows_in_int8():
    g = torch.Generator(device=DEV).manual_seed(3)
    base = whole(g, PERIOD, WIDE, most=120)
    base[:, 5] = 127.0  # every row's scale is 1
    x = in_turn(base, LONG)
    q, s = T().quantize_rows_int8(x)
    assert (s == 1).all() and equal_in_turn(q, base.to(torch.int8))
    assert torch.equal(T().dequantize_rows_int8(q, s, BF16), x)
    del q
    B = torch.randint(-1, 2, (40, WIDE), generator=g, device=DEV, dtype=torch.int8)
    y = T().linear_int8(x.float()[:, :WIDE], B, torch.ones(40, device=DEV))
    assert equal_in_turn(y, base.float() @ B.float().t())


def reference(a, b):
    return a.double() @ b.double(), a.double().abs() @ b.double().abs()


def within(got, ref, bound, dtype):
    f = torch.finfo(dtype)
    bound = bound + f.eps / 2 * (ref.abs() + bound) + f.tiny * f.eps / 2
    return bool(((got.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("tile", [0, 16, 64, 128, 256])
@pytest.mark.parametrize("groups,per,N,K,dtype", [(3, 37, 136, 200, F16), (5, 300, 72, 1032, BF16), (1500, 3, 24, 16, BF16)])
def test_equal_groups_without_offsets(groups, per, N, K, dtype, tile):
    """Forward ("nk" and "kn") and weight gradient; a group of NaN touches no other."""
    from tensorcoreptx_b200 import _native as nat
    L = nat.lib()
    g = torch.Generator(device=DEV).manual_seed(groups)
    kind = nat.TCG_F16 if dtype == F16 else nat.TCG_BF16
    A = torch.randn(groups, per, K, generator=g, device=DEV).to(dtype)
    W = torch.randn(groups, N, K, generator=g, device=DEV).to(dtype)
    D = torch.randn(groups, per, N, generator=g, device=DEV).to(dtype)
    A[1], D[1] = float("nan"), float("nan")
    clean = [e for e in range(groups) if e != 1]
    M = groups * per
    st = torch.cuda.current_stream().cuda_stream
    T().set_rows_tile(tile, 0)
    for layout, B in ((nat.TCG_B_NK, W), (nat.TCG_B_KN, W.transpose(1, 2).contiguous())):
        C = torch.full((groups, per, N), 7.0, device=DEV, dtype=F32)
        assert L.tcg_gemm_16_grouped(A.data_ptr(), B.data_ptr(), kind, C.data_ptr(), nat.TCG_F32, None, groups, M, N, K,
                                     layout, 0, st) == 0
        ref, size = reference(A[clean], W[clean].transpose(1, 2))
        assert within(C[clean], ref, 2 * U * K * size, F32) and torch.isnan(C[1]).all()
    dW = torch.full((groups, N, K), 7.0, device=DEV, dtype=dtype)
    assert L.tcg_gemm_16_grouped_wgrad(D.data_ptr(), A.data_ptr(), kind, dW.data_ptr(), kind, None, groups, M, N, K, st) == 0
    ref, size = reference(D[clean].transpose(1, 2), A[clean])
    assert within(dW[clean], ref, 2 * U * per * size, dtype) and torch.isnan(dW[1]).all()
