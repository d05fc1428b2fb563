"""Row-scaled int8 products, products grouped by expert and layers with 8-bit
checkpoints against plain 64-bit forms.

Tolerances are sums of the roundings that the kernels make (u = 2^-24, half a
step of fp32; h = half a step of the output type):
* int8: the int32 sum is exact; to fp32 (u), times scale_a (u), and one fused
  multiply-add by scale_b and bias (u of the result), then h of the result;
* 16 bits: products of 16-bit values are exact in fp32; each of the K additions
  is off by at most a whole step (2u) of a partial sum that sum|a b| bounds, and
  the CTAs' parts are added within that count; then h of the result;
* 8-bit checkpoints: scale x code in fp32 (u) and to 16 bits (h) per term.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def T():
    import tensorcoreptx_b200 as t
    return t


@pytest.fixture(autouse=True)
def _automatic_tiles():
    yield
    T().set_rows_tile(0, 0)
    assert T().check_device_error() == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def codes(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def half_step(dtype):
    """(relative, absolute below the normal range) half a step of a type."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.tiny * f.eps / 2


def rounded(ref, bound, dtype):
    rel, tiny = half_step(dtype)
    return bound + rel * (ref.abs() + bound) + tiny


def check(got, ref, bound):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), float((err / bound.clamp_min(1e-300)).max()), bad.nonzero()[:4].tolist())


def edges_of(sizes):
    e = [0]
    for s in sizes:
        e.append(e[-1] + s)
    return e


def offsets_of(edges):
    return torch.tensor(edges, dtype=torch.int32, device=DEV)


def per_group(edges, rows, f):
    """Rows of each group through f(e, a, b); rows outside the groups zero."""
    parts = [(a, b, f(e, a, b)) for e, (a, b) in enumerate(zip(edges, edges[1:]))]
    out = torch.zeros(rows, parts[0][2].size(1), dtype=torch.float64, device=DEV)
    for a, b, y in parts:
        out[a:b] = y
    return out


# ------------------------------------------------------------- quantisation --

def quantize_host(x):
    """The definition in IEEE single precision, on the host."""
    x = x.float().cpu().numpy()
    scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        q = np.clip((x * inv[..., None]).astype(np.float32), np.float32(-127), np.float32(127))
    q[np.isnan(q)] = 0  # 0 x inf: the scale is too small to have an inverse
    return np.where(q >= 0, np.floor(q + np.float32(0.5)), np.ceil(q - np.float32(0.5))).astype(np.int8), scale


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (3, 33), (1, 4096), (700, 520), (5, 20000), (2, 70001), (601, 8),
                                    (1300, 2048)])
def test_quantize_rows_bit_exact(rows, k, dtype):
    x = randn(gen(rows * k), rows, k, dtype=dtype) * 3
    x[rows // 2] = 0
    q, s = T().quantize_rows_int8(x)
    qh, sh = quantize_host(x)
    assert np.array_equal(q.cpu().numpy(), qh)
    assert np.array_equal(s.cpu().numpy().view(np.uint32), sh.view(np.uint32))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_rows_every_code_and_size(dtype):
    """All codes, halves between them, signed zeros, and rows from the smallest to the largest magnitudes."""
    base = torch.cat([torch.arange(-254, 255), torch.tensor([0.0, -0.0, 253.5])]).to(F32) / 2
    tiny = torch.finfo(dtype).smallest_normal
    sizes = [1.0, 2.0, 0.75, 1e-3, 100.0, float(tiny), float(tiny) * 2 ** -7, float(torch.finfo(dtype).max) / 128]
    x = torch.stack([(base.double() * s).to(dtype) for s in sizes]).to(DEV)
    for k in (512, 504, 511):
        y = x[:, :k].contiguous() if k < 512 else x
        q, s = T().quantize_rows_int8(y)
        qh, sh = quantize_host(y)
        assert np.array_equal(s.cpu().numpy().view(np.uint32), sh.view(np.uint32))
        assert np.array_equal(q.cpu().numpy(), qh), k


def test_quantize_rows_leading_axes_and_ties():
    x = torch.tensor([[[254.0, 1.0, 3.0, -1.0, -5.0, 0.0]], [[0.0] * 6]], device=DEV)  # scale 2: halves tie away
    q, s = T().quantize_rows_int8(x)
    assert q.tolist() == [[[127, 1, 2, -1, -3, 0]], [[0] * 6]] and s.tolist() == [[2.0], [0.0]]
    q, s = T().quantize_rows_int8(torch.zeros(3, 0, device=DEV))
    assert q.shape == (3, 0) and s.tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (2, 5, 64), (700, 528), (5, 20000), (1300, 2048)])
def test_dequantize_rows_rounds_once(shape, dtype):
    g = gen(sum(shape))
    q, s = codes(g, *shape), torch.rand(shape[:-1], generator=g, device=DEV) * 0.1
    got = T().dequantize_rows_int8(q, s, dtype)
    assert torch.equal(got, (q.float() * s[..., None]).to(dtype))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("k", [48, 41])
def test_quantize_rows_not_finite_stays_visible(value, k):
    x = torch.ones(3, k, device=DEV)
    x[1, 7] = value
    q, s = T().quantize_rows_int8(x)
    assert not torch.isfinite(s[1]) and torch.isfinite(s[[0, 2]]).all()
    assert torch.isnan(q[1].float() * s[1]).all()


# ------------------------------------------------------------ int8 products --

def int8_reference(A, B, sa, sb, bias, dtype):
    prod = (A.double() @ B.double().t()) * sa.double()[:, None] * sb.double()
    ref = prod if bias is None else prod + bias.double()
    return ref, rounded(ref, 2.1 * U * prod.abs() + U * ref.abs(), dtype)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 4096, 4096), (7, 129, 48), (17, 1000, 272), (33, 260, 2064),
                                   (65, 128, 128), (130, 77, 4112), (300, 515, 256), (1100, 2309, 144),
                                   (4100, 4099, 80)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_int8_scaled(M, N, K, dtype):
    g = gen(M + N + K)
    A, B = codes(g, M, K), codes(g, N, K)
    sa, sb = torch.rand(M, generator=g, device=DEV) * 0.01, torch.rand(N, generator=g, device=DEV) * 0.001
    bias = randn(g, N) if (M + N) % 2 else None
    check(T().gemm_int8_scaled(A, B, sa, sb, bias, out_dtype=dtype), *int8_reference(A, B, sa, sb, bias, dtype))


@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
def test_int8_scaled_every_tile_and_split(tile, split):
    g = gen(tile + split)
    M, N, K = 150, 300, 1040
    A, B = codes(g, M, K), codes(g, N, K)
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    bias = randn(g, N)
    T().set_rows_tile(tile, split)
    check(T().gemm_int8_scaled(A, B, sa, sb, bias, out_dtype=F32), *int8_reference(A, B, sa, sb, bias, F32))


@pytest.mark.parametrize("K", [4096, 4112])
def test_more_tiles_than_sms_taken_over(K):
    """Long sums in more 256-row tiles than there are SMs, last tiles partial in both directions."""
    g = gen(K)
    M, N = 3400, 3336
    A, B = codes(g, M, K), codes(g, N, K)
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    T().set_rows_tile(256, 0)
    check(T().gemm_int8_scaled(A, B, sa, sb, out_dtype=BF16), *int8_reference(A, B, sa, sb, None, BF16))
    x, W, dy = randn(g, 2200, 3400, dtype=BF16), randn(g, 3336, 3400, dtype=BF16), randn(g, 2200, 3336, dtype=BF16)
    check(T().linear(x, W), *product_reference(x, W.t(), BF16, 3400))
    got = T().gemm_grouped_wgrad(dy, x, offsets_of([0, 2200]))
    check(got, *wgrad_reference(dy, x, [0, 2200], BF16))


def test_int8_scaled_batches():
    g = gen(5)
    b, M, N, K = 3, 37, 65, 96
    A, B = codes(g, b, M, K), codes(g, b, N, K)
    sa, sb, bias = torch.rand(b, M, generator=g, device=DEV), torch.rand(b, N, generator=g, device=DEV), randn(g, b, N)
    C = T().gemm_int8_scaled(A, B, sa, sb, bias, out_dtype=BF16)
    for i in range(b):
        check(C[i], *int8_reference(A[i], B[i], sa[i], sb[i], bias[i], BF16))


def test_int8_scaled_more_batches_than_groups():
    g = gen(6)
    b, M, N, K = 1500, 3, 17, 32
    A, B = codes(g, b, M, K), codes(g, b, N, K)
    sa, sb = torch.rand(b, M, generator=g, device=DEV), torch.rand(b, N, generator=g, device=DEV)
    C = T().gemm_int8_scaled(A, B, sa, sb, out_dtype=F32)
    prod = torch.bmm(A.double(), B.double().transpose(1, 2)) * sa.double()[..., None] * sb.double()[:, None]
    check(C, prod, rounded(prod, 3.1 * U * prod.abs(), F32))


def test_int8_largest_sums_are_exact():
    K = 8192  # 127 * 127 * 8192 needs 27 bits: rounded to fp32 once
    A = torch.full((2, K), 127, dtype=torch.int8, device=DEV)
    B = torch.full((130, K), -127, dtype=torch.int8, device=DEV)
    one = torch.ones(130, device=DEV)
    C = T().gemm_int8_scaled(A, B, one[:2], one, out_dtype=F32)
    assert (C == -127 * 127 * K).all()


@pytest.mark.parametrize("shape", [(1, 4096), (2, 5, 512), (48, 1024), (4096,), (900, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_int8_is_quantise_then_product(shape, dtype):
    g = gen(len(shape))
    x, B = randn(g, *shape, dtype=dtype), codes(g, 530, shape[-1])
    sb, bias = torch.rand(530, generator=g, device=DEV) * 0.01, randn(g, 530)
    y = T().linear_int8(x, B, sb, bias)
    q, s = T().quantize_rows_int8(x)
    two = T().gemm_int8_scaled(q.view(-1, shape[-1]), B, s.view(-1), sb, bias, out_dtype=dtype)
    assert y.dtype == dtype and y.shape == shape[:-1] + (530,) and torch.equal(y.view(two.shape), two)
    qh, sh = quantize_host(x.view(-1, shape[-1]))
    ref, bound = int8_reference(torch.from_numpy(qh).to(DEV), B, torch.from_numpy(sh).to(DEV), sb, bias, dtype)
    check(y.view(ref.shape), ref, bound)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (2, 130, 48), (3, 300, 1040), (4, 1000, 4112), (1, 4099, 16384),
                                   (1, 20000, 512), (2, 2049, 4096), (4, 6143, 4096), (3, 2500, 8192), (3, 70, 8208),
                                   (4, 257, 6144), (1, 33, 24576), (1, 33, 24592), (3, 16384, 4096)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_int8_of_few_rows(M, N, K, dtype):
    """Products that quantise their rows themselves, on either side of their limits: the two-step
    result, bit for bit."""
    g = gen(M + K)
    x, B = randn(g, M, K, dtype=dtype), codes(g, N, K)
    x[M - 1] *= 0 if M == 3 else 1
    sb, bias = torch.rand(N, generator=g, device=DEV) * 0.01, randn(g, N)
    y = T().linear_int8(x, B, sb, bias)
    q, s = T().quantize_rows_int8(x)
    assert torch.equal(y, T().gemm_int8_scaled(q, B, s, sb, bias, out_dtype=dtype))
    # at an address that is not a multiple of 16 bytes, too
    z = torch.empty(M * K + 1, dtype=dtype, device=DEV)[1:].view(M, K)
    z.copy_(x)
    assert torch.equal(T().linear_int8(z, B, sb, bias), y)


def test_linear_int8_of_few_rows_not_finite():
    x = torch.ones(3, 64, device=DEV)
    x[1, 5] = float("nan")
    y = T().linear_int8(x, torch.ones(40, 64, dtype=torch.int8, device=DEV), torch.ones(40, device=DEV))
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


GROUPS = [
    ([5], 0, 5),
    ([0, 0, 0], 0, 4),                      # no rows in any group
    ([3, 0, 1, 0, 0, 17, 1, 2], 0, 24),     # few rows, empty groups at either end of a run
    ([0, 130, 0, 257, 64, 1], 0, 500),      # rows behind the last group
    ([40, 300, 7], 9, 360),                 # rows before the first one too
    ([1] * 100, 0, 100),
    ([700, 20, 1100], 0, 1820),
]


@pytest.mark.parametrize("sizes,lead,rows", GROUPS)
@pytest.mark.parametrize("bias", [False, True])
def test_int8_grouped(sizes, lead, rows, bias):
    g = gen(rows)
    E, N, K = len(sizes), 264, 208
    edges = [lead + e for e in edges_of(sizes)]
    x, B = randn(g, rows, K, dtype=BF16), codes(g, E, N, K)
    sb = torch.rand(E, N, generator=g, device=DEV) * 0.01
    b = randn(g, E, N) if bias else None
    q, s = T().quantize_rows_int8(x)
    got = T().gemm_int8_grouped(q, B, offsets_of(edges), s, sb, b, out_dtype=BF16)
    bound = torch.zeros(rows, N, dtype=torch.float64, device=DEV)

    def one(e, a, z):
        ref, bnd = int8_reference(q[a:z], B[e], s[a:z], sb[e], None if b is None else b[e], BF16)
        bound[a:z] = bnd
        return ref

    check(got, per_group(edges, rows, one), bound)
    assert torch.equal(T().linear_int8_grouped(x, B, offsets_of(edges), sb, b), got)


# ---------------------------------------------------------- 16-bit products --

def product_reference(A, Bt, dtype, K, widen=0.0):
    """A [m,K] times Bt [K,n] and the bound of its fp32 sums and last rounding."""
    ref = A.double() @ Bt.double()
    total = A.double().abs() @ Bt.double().abs()
    return ref, rounded(ref, (2 * U * K + widen) * total, dtype)


@pytest.mark.parametrize("sizes,lead,rows", GROUPS)
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("dtype,out", [(BF16, None), (F16, None), (F16, F32)])
def test_grouped(sizes, lead, rows, layout, dtype, out):
    g = gen(rows)
    E, N, K = len(sizes), 328, 200
    edges = [lead + e for e in edges_of(sizes)]
    A = randn(g, rows, K, dtype=dtype)
    B = randn(g, *((E, N, K) if layout == "nk" else (E, K, N)), dtype=dtype)
    got = T().gemm_grouped(A, B, offsets_of(edges), b_layout=layout, out_dtype=out)
    assert got.dtype == (out or dtype)
    bound = torch.zeros(rows, N, dtype=torch.float64, device=DEV)

    def one(e, a, z):
        ref, bnd = product_reference(A[a:z], B[e].t() if layout == "nk" else B[e], got.dtype, K)
        bound[a:z] = bnd
        return ref

    check(got, per_group(edges, rows, one), bound)


@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("N,out", [(1, None), (77, None), (331, F32), (515, None)])
def test_grouped_into_rows_of_odd_length(tile, N, out):
    g = gen(N)
    sizes, rows, K = [33, 0, 200, 7], 244, 136
    edges = edges_of(sizes)
    A, B = randn(g, rows, K, dtype=F16), randn(g, 4, N, K, dtype=F16)
    T().set_rows_tile(tile, 0)
    got = T().gemm_grouped(A, B, offsets_of(edges), out_dtype=out)
    bound = torch.zeros(rows, N, dtype=torch.float64, device=DEV)

    def one(e, a, z):
        ref, bnd = product_reference(A[a:z], B[e].t(), got.dtype, K)
        bound[a:z] = bnd
        return ref

    check(got, per_group(edges, rows, one), bound)


@pytest.mark.parametrize("K", [520, 2048, 4104])
@pytest.mark.parametrize("rows", [20, 700])
def test_fp32_results_of_long_sums(K, rows):
    """Chunks of 512: the error of a chain is counted over 512 terms, and one rounding per chunk."""
    g = gen(K)
    A, B = randn(g, rows, K, dtype=F16), randn(g, 1, 256, K, dtype=F16)
    got = T().gemm_grouped(A, B, offsets_of([0, rows]), out_dtype=F32)
    ref = A.double() @ B[0].double().t()
    total = A.double().abs() @ B[0].double().abs().t()
    check(got, ref, rounded(ref, (2 * U * 512 + U * (K // 512 + 1)) * total, F32))
    assert (got.double() - ref).norm() / ref.norm() < 1e-6


@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_grouped_every_tile_and_split(tile, split, layout):
    g = gen(tile)
    sizes, rows, N, K = [70, 0, 300, 13], 390, 392, 1096
    E, edges = len(sizes), edges_of(sizes)
    A = randn(g, rows, K, dtype=BF16)
    B = randn(g, *((E, N, K) if layout == "nk" else (E, K, N)), dtype=BF16)
    T().set_rows_tile(tile, split)
    got = T().gemm_grouped(A, B, offsets_of(edges), b_layout=layout, out_dtype=F32)
    bound = torch.zeros(rows, N, dtype=torch.float64, device=DEV)

    def one(e, a, z):
        ref, bnd = product_reference(A[a:z], B[e].t() if layout == "nk" else B[e], F32, K)
        bound[a:z] = bnd
        return ref

    check(got, per_group(edges, rows, one), bound)


def wgrad_reference(dC, X, edges, dtype, widen=0.0):
    ref, bound = [], []
    for a, z in zip(edges, edges[1:]):
        r, b = product_reference(dC[a:z].t(), X[a:z], dtype, z - a, widen)
        ref.append(r)
        bound.append(b)
    return torch.stack(ref), torch.stack(bound)


@pytest.mark.parametrize("sizes,lead,rows", GROUPS)
@pytest.mark.parametrize("dtype,out", [(BF16, None), (F16, F32)])
def test_wgrad(sizes, lead, rows, dtype, out):
    g = gen(rows)
    edges = [lead + e for e in edges_of(sizes)]
    dC, A = randn(g, rows, 136, dtype=dtype), randn(g, rows, 200, dtype=dtype)
    got = T().gemm_grouped_wgrad(dC, A, offsets_of(edges), out_dtype=out)
    check(got, *wgrad_reference(dC, A, edges, got.dtype))


@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("eight", [False, True])
def test_wgrad_every_tile_and_split(tile, split, eight):
    g = gen(tile + split)
    sizes, rows = [70, 0, 1001, 16, 64, 1], 1160
    edges = edges_of(sizes)
    dC, A = randn(g, rows, 264, dtype=BF16), randn(g, rows, 400, dtype=BF16)
    T().set_rows_tile(tile, split)
    if eight:
        q, s = T().quantize_rows_int8(A)
        got = T().gemm_grouped_wgrad(dC, q, offsets_of(edges), scale_a=s, out_dtype=F32)
        A = q.double() * s.double()[:, None]
        check(got, *wgrad_reference(dC, A, edges, F32, widen=1.01 * half_step(BF16)[0]))
    else:
        got = T().gemm_grouped_wgrad(dC, A, offsets_of(edges), out_dtype=F32)
        check(got, *wgrad_reference(dC, A, edges, F32))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,N,K", [(1, 8, 16), (64, 8, 16), (65, 520, 144), (3000, 1032, 272), (515, 2048, 4096)])
def test_wgrad_from_codes(rows, N, K, dtype):
    g = gen(rows)
    dC, A = randn(g, rows, N, dtype=dtype), randn(g, rows, K, dtype=dtype) * 0.1
    q, s = T().quantize_rows_int8(A)
    got = T().gemm_grouped_wgrad(dC, q, offsets_of([0, rows]), scale_a=s)
    rel, tiny = half_step(dtype)
    ref, bound = wgrad_reference(dC, q.double() * s.double()[:, None], [0, rows], dtype, widen=1.01 * rel)
    # widened values below the 16-bit normal range are off by an absolute half step
    check(got, ref, bound + tiny * dC.double().abs().sum(0)[:, None])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tile", [16, 128, 256])
def test_other_groups_rows_do_not_leak(bad, tile):
    """Rows of a group full of NaN (or outside every group) touch nothing else."""
    g = gen(3)
    edges, rows = [2, 23, 60, 200], 230
    clean = torch.zeros(rows, dtype=torch.bool, device=DEV)
    clean[2:23] = True
    clean[60:200] = True
    A, dC = randn(g, rows, 256, dtype=BF16), randn(g, rows, 128, dtype=BF16)
    W = randn(g, 3, 128, 256, dtype=BF16)
    A2, dC2 = A.clone(), dC.clone()
    A2[~clean] = bad
    dC2[~clean] = bad
    T().set_rows_tile(tile, 0)
    o = offsets_of(edges)
    y = T().gemm_grouped(A2, W, o)
    assert torch.equal(y[clean], T().gemm_grouped(A, W, o)[clean])
    assert (y[:2] == 0).all() and (y[200:] == 0).all() and not torch.isfinite(y[23:60]).any()
    dB, want = T().gemm_grouped_wgrad(dC2, A2, o), T().gemm_grouped_wgrad(dC, A, o)
    assert torch.equal(dB[[0, 2]], want[[0, 2]]) and not torch.isfinite(dB[1]).any()
    q, s = T().quantize_rows_int8(A2)
    dB = T().gemm_grouped_wgrad(dC2, q, o, scale_a=s)
    assert torch.isfinite(dB[[0, 2]]).all()


@pytest.mark.parametrize("tile", [16, 64, 256])
def test_rows_outside_a_given_result_stay(tile):
    g = gen(4)
    A, W = randn(g, 90, 64, dtype=F16), randn(g, 2, 72, 64, dtype=F16)
    o = offsets_of([5, 30, 61])
    out = torch.full((90, 72), 7.0, dtype=F16, device=DEV)
    T().set_rows_tile(tile, 0)
    assert T().gemm_grouped(A, W, o, out=out) is out
    new = T().gemm_grouped(A, W, o)
    assert (out[:5] == 7).all() and (out[61:] == 7).all() and torch.equal(out[5:61], new[5:61])
    assert (new[:5] == 0).all() and (new[61:] == 0).all()
    q, s = T().quantize_rows_int8(A)
    B, sb = codes(g, 2, 72, 64), torch.rand(2, 72, generator=g, device=DEV)
    out.fill_(7.0)
    T().gemm_int8_grouped(q, B, o, s, sb, out=out)
    assert (out[:5] == 7).all() and (out[61:] == 7).all()
    assert torch.equal(out[5:61], T().gemm_int8_grouped(q, B, o, s, sb)[5:61])


@pytest.mark.parametrize("values", [[0, 50, 20, 90], [0, 10, 40, 1000], [-5, 10, 10, 60], [70, 60, 50, 40]])
def test_offsets_that_descend_or_exceed_are_clamped(values):
    g = gen(6)
    rows = 60
    A, W = randn(g, rows, 64, dtype=BF16), randn(g, 3, 72, 64, dtype=BF16)
    edges, top = [], 0
    for v in values:
        top = max(top, min(max(v, 0), rows))
        edges.append(top)
    got = T().gemm_grouped(A, W, offsets_of(values))
    assert torch.equal(got, T().gemm_grouped(A, W, offsets_of(edges)))
    dC = randn(g, rows, 72, dtype=BF16)
    assert torch.equal(T().gemm_grouped_wgrad(dC, A, offsets_of(values)),
                       T().gemm_grouped_wgrad(dC, A, offsets_of(edges)))


def test_many_groups():
    g = gen(8)
    E, K, N = 1024, 32, 40
    sizes = [(i * 7) % 5 for i in range(E)]
    edges = edges_of(sizes)
    rows = edges[-1] + 3
    A, W = randn(g, rows, K, dtype=BF16), randn(g, E, N, K, dtype=BF16)
    group = torch.repeat_interleave(torch.arange(E, device=DEV), torch.tensor(sizes, device=DEV))
    ref = torch.einsum("mk,mnk->mn", A[:edges[-1]].double(), W.double()[group])
    total = torch.einsum("mk,mnk->mn", A[:edges[-1]].double().abs(), W.double().abs()[group])
    got = T().gemm_grouped(A, W, offsets_of(edges), out_dtype=F32)
    check(got[:edges[-1]], ref, rounded(ref, 2 * U * K * total, F32))
    assert (got[edges[-1]:] == 0).all()


# ------------------------------------------------------------------- layers --

@pytest.mark.parametrize("save", ["input", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,N", [((1, 64), 72), ((515, 768), 1024), ((3, 40, 256), 264), ((64,), 16)])
def test_linear_gradients(shape, N, dtype, save):
    g = gen(N)
    K = shape[-1]
    x = randn(g, *shape, dtype=dtype).requires_grad_(True)
    W = (randn(g, N, K) * K ** -0.5).to(dtype).requires_grad_(True)
    dy = randn(g, *shape[:-1], N, dtype=dtype)
    y = T().linear(x, W, save=save)
    y.backward(dy)
    X, D = x.detach().view(-1, K), dy.view(-1, N)
    with torch.no_grad():
        check(y.view(-1, N), *product_reference(X, W.t(), dtype, K))
        check(x.grad.view(-1, K), *product_reference(D, W, dtype, N))
        if save == "int8":
            q, s = T().quantize_rows_int8(X)
            kept = q.double() * s.double()[:, None]
            rel, tiny = half_step(dtype)
            ref, bound = product_reference(D.t(), kept, dtype, X.size(0), widen=1.01 * rel)
            check(W.grad, ref, bound + tiny * D.double().abs().sum(0)[:, None])
            # and the codes' own error against x: half a code step per value
            plain = D.double().t() @ X.double()
            step = D.double().abs().t() @ (s.double()[:, None] * 0.5 * (1 + 2 * U) + 254 * U * s.double()[:, None])
            assert ((ref - plain).abs() <= step).all()
        else:
            check(W.grad, *product_reference(D.t(), X, dtype, X.size(0)))


@pytest.mark.parametrize("save", ["input", "int8"])
def test_linear_grouped_gradients(save):
    g = gen(11)
    sizes, rows, N, K = [130, 0, 33, 257, 1], 440, 200, 144
    E, edges = len(sizes), edges_of(sizes)
    o = offsets_of(edges)
    x = randn(g, rows, K, dtype=BF16).requires_grad_(True)
    W = randn(g, E, N, K, dtype=BF16).requires_grad_(True)
    dy = randn(g, rows, N, dtype=BF16)
    y = T().linear_grouped(x, W, o, save=save)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    with torch.no_grad():
        assert torch.equal(y, T().gemm_grouped(x, W, o)) and torch.equal(dx, T().gemm_grouped(dy, W, o, b_layout="kn"))
        if save == "int8":
            q, s = T().quantize_rows_int8(x)
            kept, widen = q.double() * s.double()[:, None], 1.01 * half_step(BF16)[0]
        else:
            kept, widen = x, 0.0
        check(dW, *wgrad_reference(dy, kept, edges, BF16, widen))
        assert (dx[edges[-1]:] == 0).all() and (dW[1] == 0).all()


def test_linear_gradients_against_differences():
    """d/dt sum(f * (x + t v) (W + t u)^T) of the quadratic form by central differences, in 64 bits."""
    g = gen(12)
    x, W = randn(g, 40, 64, dtype=F16), randn(g, 24, 64, dtype=F16)
    f, v, u = randn(g, 40, 24, dtype=F16), randn(g, 40, 64).double(), randn(g, 24, 64).double()
    x.requires_grad_(True)
    W.requires_grad_(True)
    (T().linear(x, W) * f).sum().backward()

    def at(t):
        return (f.double() * ((x.detach().double() + t * v) @ (W.detach().double() + t * u).t())).sum()

    slope = (at(0.5) - at(-0.5))  # exact for a quadratic
    got = (x.grad.double() * v).sum() + (W.grad.double() * u).sum()
    rel = half_step(F16)[0]
    size = (x.grad.double() * v).abs().sum() + (W.grad.double() * u).abs().sum()
    sums = (f.double().abs() @ W.detach().double().abs() * v.abs()).sum() + \
        (f.double().abs().t() @ x.detach().double().abs() * u.abs()).sum()
    assert (got - slope).abs() <= 1.01 * rel * size + 2 * U * 64 * sums


def test_linear_gradient_of_an_expanded_output_and_partial_needs():
    g = gen(13)
    x, W = randn(g, 70, 64, dtype=BF16).requires_grad_(True), randn(g, 40, 64, dtype=BF16).requires_grad_(True)
    T().linear(x, W, save="int8").sum().backward()  # the output's gradient is a broadcast one
    want = T().gemm_grouped(torch.ones(70, 40, dtype=BF16, device=DEV), W.detach()[None], offsets_of([0, 70]), "kn")
    assert torch.equal(x.grad, want)
    y = T().linear(x.detach(), W)  # only W
    assert torch.autograd.grad(y.sum(), W)[0].shape == W.shape
    y = T().linear(x, W.detach(), save="int8")  # only x: nothing of x is kept
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)
    assert not T().linear(x.detach(), W.detach()).requires_grad


@pytest.mark.parametrize("save", ["input", "int8"])
def test_linear_gradient_that_starts_off_a_16_byte_boundary(save):
    """The output's gradient as a slice of a concatenation's, at an odd element."""
    g = gen(26)
    x, W = randn(g, 33, 64, dtype=F16).requires_grad_(True), randn(g, 24, 64, dtype=F16).requires_grad_(True)
    dy = randn(g, 33, 24, dtype=F16)
    want = torch.autograd.grad(T().linear(x, W, save=save), (x, W), dy)
    y = T().linear(x, W, save=save)
    all_of = torch.cat([torch.zeros(3, dtype=F16, device=DEV), y.flatten()])
    got = torch.autograd.grad(all_of, (x, W), torch.cat([torch.ones(3, dtype=F16, device=DEV), dy.flatten()]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_linear_computes_only_the_gradients_that_a_pass_asks_for():
    g = gen(27)
    x, W = randn(g, 64, 64, dtype=BF16).requires_grad_(True), randn(g, 2048, 64, dtype=BF16).requires_grad_(True)
    dy = randn(g, 64, 2048, dtype=BF16)
    y = T().linear(x, W)
    both = torch.autograd.grad(y, (x, W), dy, retain_graph=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    only_x, = torch.autograd.grad(y, x, dy, retain_graph=True)
    assert torch.cuda.max_memory_allocated() - before < W.numel() * 2  # no gradient of W was made
    only_W, = torch.autograd.grad(y, W, dy)
    assert torch.equal(only_x, both[0]) and torch.equal(only_W, both[1])


def test_linear_refuses_a_second_differentiation():
    x, W = torch.randn(8, 64, device=DEV).to(BF16).requires_grad_(True), torch.randn(16, 64, device=DEV).to(BF16)
    W.requires_grad_(True)
    y = T().linear(x, W)
    first = torch.autograd.grad(y.float().square().sum(), (x, W), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        first[0].float().sum().backward()
    y = T().linear(x, W)
    with torch.no_grad():
        W.add_(1.0)  # what the backward pass needs has changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y.sum(), x)


def test_linear_keeps_half_the_bytes():
    x = torch.randn(4096, 2048, device=DEV).to(BF16).requires_grad_(True)
    W = torch.randn(64, 2048, device=DEV).to(BF16).requires_grad_(True)

    def kept(save):
        h = torch.nn.functional.relu(x)  # an input that only the layer keeps
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
            y = T().linear(h, W, save=save)
        return sum(t.numel() * t.element_size() for t in seen if t.numel() and t.size(-1) != 64 and t.shape != W.shape), y

    full, eight = kept("input")[0], kept("int8")[0]
    assert full == 4096 * 2048 * 2 and eight == 4096 * 2048 + 4096 * 4


# ------------------------------------------------- streams, graphs, together --

def test_empty_inputs():
    t = T()
    o = offsets_of([0, 0, 0])
    W = torch.ones(2, 16, 32, dtype=BF16, device=DEV)
    x = torch.ones(0, 32, dtype=BF16, device=DEV)
    assert t.gemm_grouped(x, W, o).shape == (0, 16)
    dB = t.gemm_grouped_wgrad(torch.ones(0, 16, dtype=BF16, device=DEV), x, o)
    assert dB.shape == (2, 16, 32) and (dB == 0).all()
    sb = torch.ones(16, device=DEV)
    assert t.linear_int8(x, torch.ones(16, 32, dtype=torch.int8, device=DEV), sb).shape == (0, 16)
    assert t.quantize_rows_int8(x)[1].shape == (0,)
    x.requires_grad_(True)
    W2 = W[0].clone().requires_grad_(True)
    t.linear(x, W2, save="int8").sum().backward()
    assert (W2.grad == 0).all() and x.grad.shape == (0, 32)


def _expert_layer(t, x, W1, W2, o):
    """Two grouped layers with a nonlinearity, the second keeping 8 bits."""
    h = torch.nn.functional.silu(t.linear_grouped(x, W1, o, save="int8"))
    return t.linear_grouped(h, W2, o, save="int8")


def test_expert_layers_train_step_captured_and_replayed():
    """A training step of grouped layers, captured into a graph and replayed
    with other rows and other group bounds, equals the eager step."""
    t = T()
    g = gen(20)
    E, M, K, N = 5, 700, 128, 256
    W1, W2 = randn(g, E, N, K, dtype=BF16) * 0.1, randn(g, E, K, N, dtype=BF16) * 0.1
    W1.requires_grad_(True)
    W2.requires_grad_(True)
    xs = [randn(g, M, K, dtype=BF16) for _ in range(2)]
    os_ = [offsets_of([0, 100, 100, 350, 351, 690]), offsets_of([0, 0, 300, 333, 600, 700])]
    dy = randn(g, M, K, dtype=BF16)

    def step(x, o):
        return torch.autograd.grad(_expert_layer(t, x, W1, W2, o), (W1, W2), dy)

    want = [step(x, o) for x, o in zip(xs, os_)]
    x, o = xs[0].clone(), os_[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, o)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, o)
    for i in (1, 0, 1):
        x.copy_(xs[i])
        o.copy_(os_[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_serving_step_captured_and_replayed():
    t = T()
    g = gen(21)
    B1, B2 = codes(g, 1024, 512), codes(g, 512, 1024)
    s1, s2 = torch.rand(1024, generator=g, device=DEV) * 1e-3, torch.rand(512, generator=g, device=DEV) * 1e-3
    xs = [randn(g, 3, 512, dtype=BF16) for _ in range(2)]

    def step(x):
        return t.linear_int8(torch.relu(t.linear_int8(x, B1, s1)), B2, s2)

    want = [step(x) for x in xs]
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x)
    for i in (1, 0):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


def test_layers_on_another_stream_and_from_another_thread():
    """A step whose forward runs on a side stream, its backward from another host thread."""
    import threading
    t = T()
    g = gen(25)
    x, W = randn(g, 200, 128, dtype=BF16).requires_grad_(True), randn(g, 136, 128, dtype=BF16).requires_grad_(True)
    dy = randn(g, 200, 136, dtype=BF16)
    want = torch.autograd.grad(t.linear(x, W, save="int8"), (x, W), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.cuda.stream(side):
        y = t.linear(x, W, save="int8")

    def backward():
        with torch.cuda.stream(side):
            got.extend(torch.autograd.grad(y, (x, W), dy))

    th = threading.Thread(target=backward)
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_two_streams_do_not_share_anything():
    t = T()
    g = gen(22)
    x = [randn(g, m, 1024, dtype=BF16) for m in (1, 40)]
    B, sb = codes(g, 2048, 1024), torch.rand(2048, generator=g, device=DEV)
    want = [t.linear_int8(v, B, sb) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(t.linear_int8(x[i], B, sb))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_results_repeat_bit_for_bit():
    t = T()
    g = gen(23)
    A, W = randn(g, 40, 4096, dtype=BF16), randn(g, 2, 256, 4096, dtype=BF16)
    o = offsets_of([0, 11, 40])
    dC = randn(g, 40, 256, dtype=BF16)
    first = (t.gemm_grouped(A, W, o), t.gemm_grouped_wgrad(dC, A, o))
    for _ in range(10):
        assert torch.equal(t.gemm_grouped(A, W, o), first[0])
        assert torch.equal(t.gemm_grouped_wgrad(dC, A, o), first[1])


def test_serving_and_training_products_together():
    """The set as a mixture-of-experts block uses it: rows sorted by expert,
    grouped 16-bit training layers, then the same weights quantised and served
    in int8 on the same rows; int8 serving is near the 16-bit layer."""
    t = T()
    g = gen(24)
    E, M, K, N = 6, 333, 256, 384
    W = (randn(g, E, N, K) * K ** -0.5).to(BF16)
    expert = torch.randint(0, E, (M,), generator=g, device=DEV)
    order = torch.argsort(expert, stable=True)
    o = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    o[1:] = torch.cumsum(torch.bincount(expert, minlength=E), 0)
    x = randn(g, M, K, dtype=BF16)[order]
    y16 = t.linear_grouped(x, W, o)
    BT, sb = t.quantize_rows_int8(W)
    y8 = t.linear_int8_grouped(x, BT, o, sb)
    # each factor is within half a code step of its row's largest value; plus
    # both results' last roundings and the fp32 sums
    sx = x.float().abs().amax(1).double() / 254 * 1.001
    sw = W.float().abs().amax(2).double() / 254 * 1.001
    e = expert[order]
    ax, aw = x.double().abs(), W.double().abs()
    bound = sx[:, None] * aw.sum(2)[e] + ax.sum(1)[:, None] * sw[e] + K * sx[:, None] * sw[e]
    rel = half_step(BF16)[0]
    assert ((y8.double() - y16.double()).abs() <= bound * (1 + 4 * rel) + 2.1 * rel * y16.double().abs() + 1e-4).all()


@pytest.mark.parametrize("op", ["quantize_rows", "dequantize_rows", "gemm_int8_scaled", "linear_int8"])
def test_opbench_runs(op, capsys):
    from tensorcoreptx_b200 import opbench
    opbench.main([op, "--m", "96", "--n", "128", "--k", "256", "--iters", "2", "--warmup", "1"])
    assert "per call" in capsys.readouterr().out


@pytest.mark.parametrize("op", ["gemm_grouped", "gemm_grouped_wgrad", "linear_int8_grouped", "linear_train", "linear_train_int8"])
def test_opbench_runs_by_groups(op, capsys):
    from tensorcoreptx_b200 import opbench
    opbench.main([op, "--m", "96", "--n", "128", "--k", "256", "--groups", "3", "--iters", "2", "--warmup", "1"])
    assert "per call" in capsys.readouterr().out
