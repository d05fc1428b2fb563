"""Products whose rows carry structure: int8 rows with a scale each, rows
grouped by expert, and layers that train through them.

* ``quantize_rows_int8``, ``gemm_int8_scaled``, ``linear_int8``: 8-bit
  products with a scale per row (token) and per output channel;
* ``gemm_grouped``, ``gemm_grouped_wgrad``, ``gemm_int8_grouped``,
  ``linear_int8_grouped``: ragged groups of rows, one weight matrix each, the
  groups' bounds on the device;
* ``linear``, ``linear_grouped``: differentiable 16-bit layers, which with
  ``save="int8"`` keep an 8-bit copy of their input for the backward pass.

Like the other entries they check their arguments (``RuntimeError``), return
new tensors on the inputs' device, run asynchronously on that device's current
stream, and can be captured into CUDA graphs.  There is no CPU or library
fallback.  Inputs are contiguous; products need K to be a multiple of 16 (int8)
or 8 (16 bits); the number of rows is arbitrary.

``offsets`` (int32, groups + 1 values on the device) are the ascending row
bounds of the groups: group e is rows ``offsets[e]`` to ``offsets[e + 1] - 1``,
any of them empty.  Rows outside every group (a padded batch) give zeros in a
new result and are left alone in a given one.  Offsets that descend or exceed
the rows are clamped, never followed out of range.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .gemm import _check, _stream_ptr

_TYPES = {torch.float32: nat.TCG_F32, torch.float16: nat.TCG_F16, torch.bfloat16: nat.TCG_BF16}
_HALVES = (torch.float16, torch.bfloat16)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn: str, like: torch.Tensor, *args):
    """nat.lib().<fn>(*args, stream) on like's device and its current stream."""
    f = getattr(nat.lib(), fn)
    if torch.cuda.current_device() == like.get_device():
        st = f(*args, _stream_ptr(like))
    else:
        with torch.cuda.device(like.device):
            st = f(*args, _stream_ptr(like))
    nat.check(fn, st)


def _same_device(first, **others):
    for name, t in others.items():
        _check(t is None or t.device == first.device, f"{name} must be on the same device as the other operands")


def _check_offsets(offsets, groups: int, like):
    _check(offsets.is_cuda and offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous(),
           "offsets must be a contiguous 1-D CUDA int32 tensor")
    _check(offsets.numel() == groups + 1, "offsets must have one entry more than there are groups")
    _check(0 < groups <= nat.TCG_MAX_GROUPS, f"the number of groups must be 1 to {nat.TCG_MAX_GROUPS}")
    _same_device(like, offsets=offsets)


def _check_floats(name: str, t, shape, like):
    _check(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous(),
           f"{name} must be a contiguous CUDA float32 tensor")
    _check(tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}")
    _same_device(like, **{name: t})


def _grouped_out(out, A, M: int, N: int, dtype):
    """(result, zero_rest): a new result whose rows outside the groups become
    zeros, or the given one, whose rows there stay."""
    if out is None:
        return torch.empty((M, N), device=A.device, dtype=dtype), 1
    _check(out.is_cuda and out.is_contiguous() and tuple(out.shape) == (M, N) and out.dtype == dtype,
           f"out must be a contiguous CUDA tensor of shape {(M, N)} and type {dtype}")
    _same_device(A, out=out)
    return out, 0


# --------------------------------------------------------- int8 with scales --

def quantize_rows_int8(x: torch.Tensor):
    """Absmax quantisation of each row (the last axis) of a float32, float16 or
    bfloat16 tensor: codes int8 of x's shape and scales float32 of its leading
    shape, scale = max|x| / 127 and codes rounded half away from zero, as
    quantize_absmax_int8 does per tensor.  A row of zeros has scale 0; a row
    with an infinity or a NaN gets a scale that is not finite."""
    _check(x.is_cuda and x.dtype in _TYPES and x.is_contiguous() and x.dim() >= 1,
           "x must be a contiguous CUDA float32, float16 or bfloat16 tensor with at least one axis")
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call("tcg_quantize_rows_s8", x, x.data_ptr(), _TYPES[x.dtype], codes.data_ptr(), scales.data_ptr(),
          scales.numel(), x.size(-1))
    return codes, scales


def gemm_int8_scaled(A: torch.Tensor, BT: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                     bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """C[M,N] = (A[M,K] int8 x BT[N,K]^T int8) * scale_a[M] * scale_b[N] (+
    bias[N]), float32 scales and bias, rounded once to out_dtype (float16,
    bfloat16 or float32).  3-D inputs are batches, with scale_a [b,M] and
    scale_b and bias [b,N]."""
    _check(A.is_cuda and BT.is_cuda, "A and BT must be CUDA tensors")
    _check(A.dtype == torch.int8 and BT.dtype == torch.int8, "A and BT must be int8")
    _check(A.dim() == BT.dim() and A.dim() in (2, 3), "A and BT must be 2-D")
    _check(A.dim() == 2 or A.size(0) == BT.size(0), "A and BT must have the same batch count")
    _check(A.size(-1) == BT.size(-1), "A cols must equal BT cols (both = K)")
    _check(A.is_contiguous() and BT.is_contiguous(), "A and BT must be contiguous")
    _check(out_dtype in _TYPES, "out_dtype must be float16, bfloat16 or float32")
    _same_device(A, BT=BT)
    lead, M, N, K = A.shape[:-2], A.size(-2), BT.size(-2), A.size(-1)
    _check_floats("scale_a", scale_a, lead + (M,), A)
    _check_floats("scale_b", scale_b, lead + (N,), A)
    if bias is not None:
        _check_floats("bias", bias, lead + (N,), A)
    C = torch.empty(lead + (M, N), dtype=out_dtype, device=A.device)
    _call("tcg_gemm_s8_scaled", A, A.data_ptr(), BT.data_ptr(), C.data_ptr(), _TYPES[out_dtype], M, N, K,
          A.size(0) if A.dim() == 3 else 1, scale_a.data_ptr(), scale_b.data_ptr(), _ptr(bias))
    return C


def _linear_int8(x, BT, offsets, scale_b, bias, out, fn):
    groups, N, K = (BT.size(0) if offsets is not None else 1), BT.size(-2), BT.size(-1)
    _check(x.dtype in _TYPES, "x must be float32, float16 or bfloat16")
    _check(BT.dtype == torch.int8, "BT must be int8")
    _check(x.size(-1) == K, "x cols must equal BT cols (both = K)")
    _check(x.is_contiguous() and BT.is_contiguous(), "x and BT must be contiguous")
    _same_device(x, BT=BT)
    _check_floats("scale_b", scale_b, BT.shape[:-1], x)
    if bias is not None:
        _check_floats("bias", bias, BT.shape[:-1], x)
    M = x.numel() // K if K else 0
    _check(K > 0, "K must not be 0")
    if offsets is None:
        C, rest = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device), 0
    else:
        C, rest = _grouped_out(out, x, M, N, x.dtype)
    if C.numel() == 0:
        return C
    need = ((M * K + 255) & ~255) + ((4 * M + 255) & ~255)  # tcg_linear_s8_workspace_size
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _call("tcg_linear_s8_grouped", x, x.data_ptr(), _TYPES[x.dtype], BT.data_ptr(), C.data_ptr(), _TYPES[x.dtype],
          _ptr(offsets), groups, M, N, K, scale_b.data_ptr(), _ptr(bias), rest, ws.data_ptr(), need)
    return C


def linear_int8(x: torch.Tensor, BT: torch.Tensor, scale_b: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """y[..., N] in x's type = x[..., K] quantised per row (quantize_rows_int8)
    times BT[N,K] int8 with scale_b[N] per channel, plus bias[N]: one call from
    activations to activations (gemm_int8_scaled between)."""
    _check(x.is_cuda and BT.is_cuda, "x and BT must be CUDA tensors")
    _check(x.dim() >= 1 and BT.dim() == 2, "BT must be 2-D")
    return _linear_int8(x, BT, None, scale_b, bias, None, "linear_int8")


def linear_int8_grouped(x: torch.Tensor, BT: torch.Tensor, offsets: torch.Tensor, scale_b: torch.Tensor,
                        bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """As linear_int8 for grouped rows x[M,K]: group e meets BT[e] of
    BT[E,N,K], with scale_b and bias [E,N]."""
    _check(x.is_cuda and BT.is_cuda, "x and BT must be CUDA tensors")
    _check(x.dim() == 2 and BT.dim() == 3, "x must be 2-D and BT 3-D")
    _check_offsets(offsets, BT.size(0), x)
    return _linear_int8(x, BT, offsets, scale_b, bias, out, "linear_int8_grouped")


def gemm_int8_grouped(A: torch.Tensor, BT: torch.Tensor, offsets: torch.Tensor, scale_a: torch.Tensor,
                      scale_b: torch.Tensor, bias: torch.Tensor | None = None,
                      out_dtype: torch.dtype = torch.float16, out: torch.Tensor | None = None) -> torch.Tensor:
    """As gemm_int8_scaled for grouped rows A[M,K]: group e meets BT[e] of
    BT[E,N,K], with scale_a [M], scale_b and bias [E,N]."""
    _check(A.is_cuda and BT.is_cuda, "A and BT must be CUDA tensors")
    _check(A.dtype == torch.int8 and BT.dtype == torch.int8, "A and BT must be int8")
    _check(A.dim() == 2 and BT.dim() == 3, "A must be 2-D and BT 3-D")
    _check(A.size(-1) == BT.size(-1), "A cols must equal BT cols (both = K)")
    _check(A.is_contiguous() and BT.is_contiguous(), "A and BT must be contiguous")
    _check(out_dtype in _TYPES, "out_dtype must be float16, bfloat16 or float32")
    _same_device(A, BT=BT)
    E, N, K = BT.shape
    M = A.size(0)
    _check_offsets(offsets, E, A)
    _check_floats("scale_a", scale_a, (M,), A)
    _check_floats("scale_b", scale_b, (E, N), A)
    if bias is not None:
        _check_floats("bias", bias, (E, N), A)
    C, rest = _grouped_out(out, A, M, N, out_dtype)
    _call("tcg_gemm_s8_grouped", A, A.data_ptr(), BT.data_ptr(), C.data_ptr(), _TYPES[out_dtype], offsets.data_ptr(),
          E, M, N, K, scale_a.data_ptr(), scale_b.data_ptr(), _ptr(bias), rest)
    return C


# ------------------------------------------------------- 16-bit, by groups --

def _product(A, B, offsets, b_layout, C, rest):
    """C = A x B per group through tcg_gemm_16_grouped (arguments checked)."""
    groups = B.size(0) if B.dim() == 3 else 1
    K, N = A.size(-1), C.size(-1)
    M = A.numel() // K if K else 0
    _call("tcg_gemm_16_grouped", A, A.data_ptr(), B.data_ptr(), _TYPES[A.dtype], C.data_ptr(), _TYPES[C.dtype],
          _ptr(offsets), groups, M, N, K, nat.TCG_B_NK if b_layout == "nk" else nat.TCG_B_KN, rest)
    return C


def gemm_grouped(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, b_layout: str = "nk",
                 out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """C[M,N] = rows of A[M,K] (float16 or bfloat16) times their group's matrix
    of B: [E,N,K] (b_layout="nk") or [E,K,N] ("kn"), fp32 sums, rounded once to
    out_dtype (A's type, or float32)."""
    _check(A.is_cuda and B.is_cuda, "A and B must be CUDA tensors")
    _check(A.dtype in _HALVES and B.dtype == A.dtype, "A and B must both be float16 or both bfloat16")
    _check(A.dim() == 2 and B.dim() == 3, "A must be 2-D and B 3-D")
    _check(b_layout in ("nk", "kn"), "b_layout must be 'nk' or 'kn'")
    N, K = (B.size(1), B.size(2)) if b_layout == "nk" else (B.size(2), B.size(1))
    _check(A.size(1) == K, "A cols must equal K of B")
    _check(A.is_contiguous() and B.is_contiguous(), "A and B must be contiguous")
    out_dtype = A.dtype if out_dtype is None else out_dtype
    _check(out_dtype in _TYPES, "out_dtype must be float16, bfloat16 or float32")
    _same_device(A, B=B)
    _check_offsets(offsets, B.size(0), A)
    C, rest = _grouped_out(out, A, A.size(0), N, out_dtype)
    return _product(A, B, offsets, b_layout, C, rest)


def _wgrad(dC, A, scale_a, offsets, groups, out_dtype):
    """dB[groups,N,K] through tcg_gemm_16_grouped_wgrad (arguments checked)."""
    N, K = dC.size(-1), A.size(-1)
    M = dC.numel() // N if N else 0
    dB = torch.empty((groups, N, K), dtype=out_dtype, device=dC.device)
    _call("tcg_gemm_16_grouped_wgrad", dC, dC.data_ptr(), A.data_ptr(), _ptr(scale_a), _TYPES[dC.dtype],
          dB.data_ptr(), _TYPES[out_dtype], _ptr(offsets), groups, M, N, K)
    return dB


def gemm_grouped_wgrad(dC: torch.Tensor, A: torch.Tensor, offsets: torch.Tensor,
                       scale_a: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dB[E,N,K], the gradient of gemm_grouped by B ("nk"): for each group the
    sum over its rows m of dC[m,N] (float16 or bfloat16) outer A[m,K], zero for
    an empty group; fp32 sums, rounded once to out_dtype (dC's type, or
    float32).  A has dC's type, or is the int8 codes of quantize_rows_int8 with
    their scales as scale_a[M].  (Swapping dC and A gives the "kn" gradient.)"""
    _check(dC.is_cuda and A.is_cuda, "dC and A must be CUDA tensors")
    _check(dC.dtype in _HALVES, "dC must be float16 or bfloat16")
    _check(A.dtype == (dC.dtype if scale_a is None else torch.int8),
           "A must have dC's type, or be int8 with scale_a given")
    _check(dC.dim() == 2 and A.dim() == 2 and dC.size(0) == A.size(0), "dC and A must be 2-D with the same rows")
    _check(dC.is_contiguous() and A.is_contiguous(), "dC and A must be contiguous")
    out_dtype = dC.dtype if out_dtype is None else out_dtype
    _check(out_dtype in _TYPES, "out_dtype must be float16, bfloat16 or float32")
    _same_device(dC, A=A)
    groups = offsets.numel() - 1
    _check_offsets(offsets, groups, dC)
    if scale_a is not None:
        _check_floats("scale_a", scale_a, (A.size(0),), dC)
    return _wgrad(dC, A, scale_a, offsets, groups, out_dtype)


# ------------------------------------------------------------------ layers --

class _Linear(torch.autograd.Function):
    """y = x W^T per group.  Backward: dx = dy W (the same product with W's
    other layout), dW = dy^T x from x or from its int8 codes and scales."""

    @staticmethod
    def forward(ctx, x, W, offsets, save):
        y = torch.empty(x.shape[:-1] + (W.size(-2),), dtype=x.dtype, device=x.device)
        _product(x, W, offsets, "nk", y, 1)
        codes = scales = None
        if ctx.needs_input_grad[1]:
            if save == "int8":
                codes, scales = quantize_rows_int8(x)
                x = None
        else:
            x = None
        ctx.save_for_backward(x, codes, scales, W if ctx.needs_input_grad[0] else None, offsets)
        ctx.weight_shape = W.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, codes, scales, W, offsets = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dW = None
        if W is not None:
            dx = torch.empty(dy.shape[:-1] + (W.size(-1),), dtype=dy.dtype, device=dy.device)
            _product(dy, W, offsets, "kn", dx, 1)
        if ctx.needs_input_grad[1]:
            groups = ctx.weight_shape[0] if len(ctx.weight_shape) == 3 else 1
            dW = _wgrad(dy, codes if x is None else x, scales, offsets, groups, dy.dtype).view(ctx.weight_shape)
        return dx, dW, None, None


def _check_linear(x, W, save):
    _check(x.is_cuda and W.is_cuda, "x and W must be CUDA tensors")
    _check(x.dtype in _HALVES and W.dtype == x.dtype, "x and W must both be float16 or both bfloat16")
    _check(save in ("input", "int8"), "save must be 'input' or 'int8'")
    _check(x.size(-1) == W.size(-1), "x cols must equal W cols (both = K)")
    _check(x.is_contiguous() and W.is_contiguous(), "x and W must be contiguous")
    _check(W.size(-1) % (16 if save == "int8" else 8) == 0, "K must be a multiple of 8 (16 with save='int8')")
    _check(W.size(-2) % 8 == 0, "N must be a multiple of 8")
    _check(W.numel() > 0, "W must not be empty")
    _same_device(x, W=W)


def linear(x: torch.Tensor, W: torch.Tensor, save: str = "input") -> torch.Tensor:
    """y[..., N] = x[..., K] W[N,K]^T (float16 or bfloat16, fp32 sums),
    differentiable by x and W.  save="int8" keeps x for the backward pass as
    int8 codes with a scale per row, half of its bytes: the output and x's
    gradient are unchanged, W's gradient is that of the codes."""
    _check(x.dim() >= 1 and W.dim() == 2, "W must be 2-D")
    _check_linear(x, W, save)
    return _Linear.apply(x, W, None, save)


def linear_grouped(x: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, save: str = "input") -> torch.Tensor:
    """As linear for grouped rows x[M,K]: group e meets W[e] of W[E,N,K].  Rows
    outside every group give zero outputs and get zero gradients."""
    _check(x.dim() == 2 and W.dim() == 3, "x must be 2-D and W 3-D")
    _check_linear(x, W, save)
    _check_offsets(offsets, W.size(0), x)
    return _Linear.apply(x, W, offsets, save)


def set_rows_tile(rows: int, split: int = 0) -> None:
    """Force the tile (16, 32, 64, 128 or 256 rows) and the number of CTAs that
    share a tile's sum (1, 2, 4, 8) of these products; 0 restores the choice."""
    nat.lib().tcg_set_rows_tile(int(rows), int(split))
