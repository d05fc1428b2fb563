"""Products whose rows carry structure: int8 rows with a scale each, rows
grouped by expert, and layers that train through them.

* ``quantize_rows_int8``, ``dequantize_rows_int8``, ``gemm_int8_scaled``,
  ``linear_int8``: 8-bit products with a scale per row (token) and per output channel;
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
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# Small calls are bound by the host, so what every call passes through stays
# short: checks build their message only when they fail, and results are made
# with Tensor.new_empty / empty_like (a third of torch.empty's time here).

def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn: str, like: torch.Tensor, *args):
    """nat.lib().<fn>(*args, stream) on like's device and its current stream."""
    f = getattr(nat.lib(), fn)
    if _current_device() == like.get_device():
        st = f(*args, _stream_ptr(like))
    else:
        with torch.cuda.device(like.device):
            st = f(*args, _stream_ptr(like))
    if st != nat.TCG_SUCCESS:
        nat.check(fn, st)


def _same_device(like, name, t):
    if t is not None and t.get_device() != like.get_device():
        raise RuntimeError(f"{name} must be on the same device as the other operands")


def _check_offsets(offsets, groups: int, like):
    if not (offsets.is_cuda and offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous()):
        raise RuntimeError("offsets must be a contiguous 1-D CUDA int32 tensor")
    _check(offsets.numel() == groups + 1, "offsets must have one entry more than there are groups")
    if not 0 < groups <= nat.TCG_MAX_GROUPS:
        raise RuntimeError(f"the number of groups must be 1 to {nat.TCG_MAX_GROUPS}")
    _same_device(like, "offsets", offsets)


def _check_floats(name: str, t, shape, like):
    if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
        raise RuntimeError(f"{name} must be a contiguous CUDA float32 tensor")
    if t.shape != shape:
        raise RuntimeError(f"{name} must have shape {tuple(shape)}")
    _same_device(like, name, t)


def _grouped_out(out, A, M: int, N: int, dtype):
    """(result, zero_rest): a new result whose rows outside the groups become
    zeros, or the given one, whose rows there stay."""
    if out is None:
        return A.new_empty((M, N), dtype=dtype), 1
    if not (out.is_cuda and out.is_contiguous() and out.shape == (M, N) and out.dtype == dtype):
        raise RuntimeError(f"out must be a contiguous CUDA tensor of shape {(M, N)} and type {dtype}")
    _same_device(A, "out", out)
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
    codes = torch.empty_like(x, dtype=torch.int8)
    scales = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _call("tcg_quantize_rows_s8", x, x.data_ptr(), _TYPES[x.dtype], codes.data_ptr(), scales.data_ptr(),
          scales.numel(), x.size(-1))
    return codes, scales


def _dequantize(codes, scales, dtype):
    out = torch.empty_like(codes, dtype=dtype)
    _call("tcg_dequantize_rows_s8", codes, codes.data_ptr(), scales.data_ptr(), out.data_ptr(), _TYPES[dtype],
          scales.numel(), codes.size(-1))
    return out


def dequantize_rows_int8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float16):
    """The way back from quantize_rows_int8: codes times their row's scale in
    fp32, rounded once to dtype (float16, bfloat16 or float32)."""
    _check(codes.is_cuda and codes.dtype == torch.int8 and codes.is_contiguous() and codes.dim() >= 1,
           "codes must be a contiguous CUDA int8 tensor with at least one axis")
    _check_floats("scales", scales, codes.shape[:-1], codes)
    _check(dtype in _TYPES, "dtype must be float16, bfloat16 or float32")
    return _dequantize(codes, scales, dtype)


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
    _same_device(A, "BT", BT)
    lead, M, N, K = A.shape[:-2], A.size(-2), BT.size(-2), A.size(-1)
    _check_floats("scale_a", scale_a, lead + (M,), A)
    _check_floats("scale_b", scale_b, lead + (N,), A)
    if bias is not None:
        _check_floats("bias", bias, lead + (N,), A)
    C = A.new_empty(lead + (M, N), dtype=out_dtype)
    _call("tcg_gemm_s8_scaled", A, A.data_ptr(), BT.data_ptr(), C.data_ptr(), _TYPES[out_dtype], M, N, K,
          A.size(0) if A.dim() == 3 else 1, scale_a.data_ptr(), scale_b.data_ptr(), _ptr(bias))
    return C


def _linear_int8(x, BT, offsets, scale_b, bias, out):
    groups, N, K = (BT.size(0) if offsets is not None else 1), BT.size(-2), BT.size(-1)
    _check(x.dtype in _TYPES, "x must be float32, float16 or bfloat16")
    _check(BT.dtype == torch.int8, "BT must be int8")
    _check(x.size(-1) == K, "x cols must equal BT cols (both = K)")
    _check(x.is_contiguous() and BT.is_contiguous(), "x and BT must be contiguous")
    _same_device(x, "BT", BT)
    _check_floats("scale_b", scale_b, BT.shape[:-1], x)
    if bias is not None:
        _check_floats("bias", bias, BT.shape[:-1], x)
    M = x.numel() // K if K else 0
    _check(K > 0, "K must not be 0")
    if offsets is None:
        C, rest = x.new_empty(x.shape[:-1] + (N,)), 0
    else:
        C, rest = _grouped_out(out, x, M, N, x.dtype)
    if C.numel() == 0:
        return C
    need = ((M * K + 255) & ~255) + ((4 * M + 255) & ~255)  # tcg_linear_s8_workspace_size
    ws = x.new_empty(need, dtype=torch.uint8)
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
    return _linear_int8(x, BT, None, scale_b, bias, None)


def linear_int8_grouped(x: torch.Tensor, BT: torch.Tensor, offsets: torch.Tensor, scale_b: torch.Tensor,
                        bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """As linear_int8 for grouped rows x[M,K]: group e meets BT[e] of
    BT[E,N,K], with scale_b and bias [E,N]."""
    _check(x.is_cuda and BT.is_cuda, "x and BT must be CUDA tensors")
    _check(x.dim() == 2 and BT.dim() == 3, "x must be 2-D and BT 3-D")
    _check_offsets(offsets, BT.size(0), x)
    return _linear_int8(x, BT, offsets, scale_b, bias, out)


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
    _same_device(A, "BT", BT)
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
    _same_device(A, "B", B)
    _check_offsets(offsets, B.size(0), A)
    C, rest = _grouped_out(out, A, A.size(0), N, out_dtype)
    return _product(A, B, offsets, b_layout, C, rest)


def _wgrad(dC, A, scale_a, offsets, groups, out_dtype):
    """dB[groups,N,K] through tcg_gemm_16_grouped_wgrad (arguments checked).
    Codes are widened into a buffer of the call first: every tile of dB along N
    reads all of A, so widening them on the way into the product (32 times over
    for N = 8192) measured 515 us where this takes 390 + 20 (8192 rows, N 8192,
    K 4096)."""
    if scale_a is not None:
        A = _dequantize(A, scale_a, dC.dtype)
    N, K = dC.size(-1), A.size(-1)
    M = dC.numel() // N if N else 0
    dB = dC.new_empty((groups, N, K), dtype=out_dtype)
    _call("tcg_gemm_16_grouped_wgrad", dC, dC.data_ptr(), A.data_ptr(), _TYPES[dC.dtype], dB.data_ptr(),
          _TYPES[out_dtype], _ptr(offsets), groups, M, N, K)
    return dB


def gemm_grouped_wgrad(dC: torch.Tensor, A: torch.Tensor, offsets: torch.Tensor,
                       scale_a: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dB[E,N,K], the gradient of gemm_grouped by B ("nk"): for each group the
    sum over its rows m of dC[m,N] (float16 or bfloat16) outer A[m,K], zero for
    an empty group; fp32 sums, rounded once to out_dtype (dC's type, or
    float32).  A has dC's type, or is the int8 codes of quantize_rows_int8 with
    their scales as scale_a[M], which stand for code * scale rounded to dC's
    type (a buffer of that size lives during the call).  (Swapping dC and A gives the "kn" gradient.)"""
    _check(dC.is_cuda and A.is_cuda, "dC and A must be CUDA tensors")
    _check(dC.dtype in _HALVES, "dC must be float16 or bfloat16")
    _check(A.dtype == (dC.dtype if scale_a is None else torch.int8),
           "A must have dC's type, or be int8 with scale_a given")
    _check(dC.dim() == 2 and A.dim() == 2 and dC.size(0) == A.size(0), "dC and A must be 2-D with the same rows")
    _check(dC.is_contiguous() and A.is_contiguous(), "dC and A must be contiguous")
    out_dtype = dC.dtype if out_dtype is None else out_dtype
    _check(out_dtype in _TYPES, "out_dtype must be float16, bfloat16 or float32")
    _same_device(dC, "A", A)
    groups = offsets.numel() - 1
    _check_offsets(offsets, groups, dC)
    if scale_a is not None:
        _check_floats("scale_a", scale_a, (A.size(0),), dC)
    return _wgrad(dC, A, scale_a, offsets, groups, out_dtype)


# ------------------------------------------------------------------ layers --

def _forward(x, W, offsets):
    return _product(x, W, offsets, "nk", x.new_empty(x.shape[:-1] + (W.size(-2),)), 1)


def _backward(ctx, dy):
    x, scales, W, offsets = ctx.saved_tensors
    dy = dy.contiguous()
    dx = dW = None
    if W is not None:
        dx = _product(dy, W, offsets, "kn", dy.new_empty(dy.shape[:-1] + (W.size(-1),)), 1)
    if x is not None:
        shape = ctx.weight_shape
        dW = _wgrad(dy, x, scales, offsets, shape[0] if len(shape) == 3 else 1, dy.dtype)
        if len(shape) == 2:
            dW = dW.view(shape)
    return dx, dW, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


class _Linear(torch.autograd.Function):
    """y = x W^T per group.  Backward: dx = dy W (the same product with W's
    other layout), dW = dy^T x from x or from its int8 codes and scales.  What
    one input's gradient alone needs is kept only where that is asked for."""

    @staticmethod
    def forward(ctx, x, W, offsets, eight):
        y = _forward(x, W, offsets)
        need_x, need_W = ctx.needs_input_grad[:2]
        scales = None
        if not need_W:
            x = None
        elif eight:
            x, scales = quantize_rows_int8(x)
        ctx.weight_shape = W.shape
        ctx.save_for_backward(x, scales, W if need_x else None, offsets)
        return y

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses a second differentiation costs microseconds
        # and matters only where this one is recorded)
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _apply(x, W, offsets, save):
    if torch.is_grad_enabled() and (x.requires_grad or W.requires_grad):
        return _Linear.apply(x, W, offsets, save == "int8")
    return _forward(x, W, offsets)


def _check_linear(x, W, save):
    _check(x.is_cuda and W.is_cuda, "x and W must be CUDA tensors")
    _check(x.dtype in _HALVES and W.dtype == x.dtype, "x and W must both be float16 or both bfloat16")
    _check(save in ("input", "int8"), "save must be 'input' or 'int8'")
    _check(x.size(-1) == W.size(-1), "x cols must equal W cols (both = K)")
    _check(x.is_contiguous() and W.is_contiguous(), "x and W must be contiguous")
    _check(W.size(-1) % 8 == 0, "K must be a multiple of 8")
    _check(W.size(-2) % 8 == 0, "N must be a multiple of 8")
    _check(W.numel() > 0, "W must not be empty")
    _same_device(x, "W", W)


def linear(x: torch.Tensor, W: torch.Tensor, save: str = "input") -> torch.Tensor:
    """y[..., N] = x[..., K] W[N,K]^T (float16 or bfloat16, fp32 sums),
    differentiable by x and W.  save="int8" keeps x for the backward pass as
    int8 codes with a scale per row, half of its bytes (the backward pass widens
    one layer's codes at a time): the output and x's gradient are unchanged, W's
    gradient is that of the codes."""
    _check(x.dim() >= 1 and W.dim() == 2, "W must be 2-D")
    _check_linear(x, W, save)
    return _apply(x, W, None, save)


def linear_grouped(x: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, save: str = "input") -> torch.Tensor:
    """As linear for grouped rows x[M,K]: group e meets W[e] of W[E,N,K].  Rows
    outside every group give zero outputs and get zero gradients."""
    _check(x.dim() == 2 and W.dim() == 3, "x must be 2-D and W 3-D")
    _check_linear(x, W, save)
    _check_offsets(offsets, W.size(0), x)
    return _apply(x, W, offsets, save)


def set_rows_tile(rows: int, split: int = 0) -> None:
    """Force the tile (16, 32, 64, 128 or 256 rows) and the number of CTAs that
    share a tile's sum (1, 2, 4, 8) of these products; 0 restores the choice."""
    nat.lib().tcg_set_rows_tile(int(rows), int(split))
