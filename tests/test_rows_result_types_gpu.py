"""16-bit products with results of the other 16-bit type: fp32 sums, one rounding
to the result's type.  Tolerance: 2 u K sum|a b| of the sums (u = 2^-24, a whole
step an addition), then half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, F16 = torch.bfloat16, torch.float16


def rounded(ref, bound, dtype):
    f = torch.finfo(dtype)
    return bound + f.eps / 2 * (ref.abs() + bound) + f.tiny * f.eps / 2


@pytest.mark.parametrize("dtype,out", [(F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("rows,N,K", [(5, 40, 64), (130, 257, 520), (2000, 1032, 264)])
def test_results_of_the_other_16_bit_type(rows, N, K, dtype, out):
    import tensorcoreptx_b200 as t
    g = torch.Generator(device=DEV).manual_seed(rows)
    edges = [0, rows // 3, rows]
    o = torch.tensor(edges, dtype=torch.int32, device=DEV)
    A, W = (torch.randn(rows, K, generator=g, device=DEV).to(dtype), torch.randn(2, N, K, generator=g, device=DEV).to(dtype))
    got = t.gemm_grouped(A, W, o, out_dtype=out)
    assert got.dtype == out
    for e in range(2):
        a, w = A[edges[e]:edges[e + 1]].double(), W[e].double()
        ref = a @ w.t()
        err = (got[edges[e]:edges[e + 1]].double() - ref).abs()
        assert (err <= rounded(ref, 2 * U * K * (a.abs() @ w.abs().t()), out)).all()
    N8 = N // 8 * 8
    dC = torch.randn(rows, N8, generator=g, device=DEV).to(dtype)
    got = t.gemm_grouped_wgrad(dC, A, o, out_dtype=out)
    assert got.dtype == out
    for e in range(2):
        d, a = dC[edges[e]:edges[e + 1]].double().t(), A[edges[e]:edges[e + 1]].double()
        ref = d @ a
        assert ((got[e].double() - ref).abs() <= rounded(ref, 2 * U * a.size(0) * (d.abs() @ a.abs()), out)).all()
