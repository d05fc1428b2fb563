"""Row quantisation of rows whose largest value is near the smallest normal
number, where 1 / scale passes the range of fp32 (below 127 * 2^-128 = 3.7e-37).

Tolerance, with u = 2^-24 and s the row's scale as returned: the inverse of s and
the product with it are off by u each, at most 127.01 * 2.01 u in steps of s; the
sum with one half by 2^-18; rounding by one half.  Together below 0.5 + 2^-15
steps.  s itself is a subnormal of at least 16 bits, off by at most 2^-16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
TOPS = [2.0 ** -126, 1.5 * 2.0 ** -126, 2.0 ** -125, 2e-37, 126.9 * 2.0 ** -128, 127 * 2.0 ** -128, 127.1 * 2.0 ** -128,
        2.0 ** -120, 1e-35]


def T():
    import tensorcoreptx_b200 as t
    return t


def rows_of_size(rows, k, dtype):
    """Rows of all sizes of TOPS in turn, each with its largest value somewhere."""
    g = torch.Generator(device=DEV).manual_seed(rows * 31 + k)
    x = torch.rand(rows, k, generator=g, device=DEV, dtype=torch.float64) * 2 - 1
    x[torch.arange(rows), torch.randint(0, k, (rows,), generator=g, device=DEV)] = 1.0
    top = torch.tensor(TOPS, device=DEV, dtype=torch.float64)[torch.arange(rows, device=DEV) % len(TOPS)]
    return (x * top[:, None]).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k", [(9, 1), (9, 16), (11, 33), (9, 4096), (18, 20000), (603, 520), (603, 8192)])
def test_codes_are_within_half_a_step(rows, k, dtype):
    x = rows_of_size(rows, k, dtype)
    q, s = T().quantize_rows_int8(x)
    top = x.abs().amax(1)
    assert (top >= 2.0 ** -126).all()
    # top / 127 in IEEE single precision, subnormals kept (as the host computes it)
    assert torch.equal(s.cpu(), top.float().cpu() / 127)
    err = (x.double() - q.double() * s.double()[:, None]).abs()
    assert (err <= s.double()[:, None] * (0.5 + 2.0 ** -15)).all()
    assert (err <= top.double()[:, None] / 254 * (1 + 2.0 ** -13)).all()


def test_two_values_of_one_row_keep_their_sizes():
    x = torch.tensor([[2e-37, 2e-38, -2e-37, 0.0]], device=DEV)
    q, s = T().quantize_rows_int8(x)
    assert q.tolist() == [[127, 13, -127, 0]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 9])
def test_linear_int8_of_small_rows(rows, dtype):
    """The product that quantises its own rows agrees with quantising first."""
    x = rows_of_size(rows, 512, dtype)
    g = torch.Generator(device=DEV).manual_seed(rows)
    B = torch.randint(-127, 128, (96, 512), generator=g, device=DEV, dtype=torch.int8)
    sb = torch.rand(96, generator=g, device=DEV) * 1e30
    q, s = T().quantize_rows_int8(x)
    assert torch.equal(T().linear_int8(x, B, sb), T().gemm_int8_scaled(q, B, s, sb, out_dtype=dtype))
    assert (q.float().abs().amax(1) == 127).all() and not (q.float().abs() == 127).all()


def test_checkpoint_gradient_of_small_rows():
    """save="int8": x of 2e-37 against gradients of 1e30; the gradient by W is within the codes' half steps."""
    x = rows_of_size(18, 64, BF16).requires_grad_(True)
    g = torch.Generator(device=DEV).manual_seed(1)
    W = torch.randn(16, 64, generator=g, device=DEV).to(BF16).requires_grad_(True)
    dy = (torch.randn(18, 16, generator=g, device=DEV) * 1e30).to(BF16)
    dW, = torch.autograd.grad(T().linear(x, W, save="int8"), W, dy)
    X, D = x.detach().double(), dy.double()
    step = D.abs().t() @ (X.abs().amax(1, keepdim=True) / 254 * (1 + 2.0 ** -13)).expand_as(X)
    # codes x scale to bf16 (2^-8 relative, 2^-134 absolute), fp32 sums, the result to bf16
    size = D.abs().t() @ X.abs() + step
    rounding = 2.0 ** -7 * 1.01 * size + D.abs().sum(0)[:, None] * 2.0 ** -134
    assert ((dW.double() - D.t() @ X).abs() <= step + rounding).all()
