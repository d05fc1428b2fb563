"""Products whose rows carry structure: int8 rows with a scale each, rows
grouped by expert, and layers that train through them.

* ``quantize_rows_int8``, ``dequantize_rows_int8``, ``gemm_int8_scaled``,
  ``linear_int8``: 8-bit products with a scale per row (token) and per output channel;
* ``gemm_grouped``, ``gemm_grouped_wgrad``, ``gemm_int8_grouped``,
  ``linear_int8_grouped``: ragged groups of rows, one weight matrix each, the
  groups' bounds on the device;
* ``linear``, ``linear_grouped``: differentiable 16-bit layers, which with
  ``save="int8"`` keep an 8-bit copy of their input for the backward pass.

Only the layers differentiate; the results of the others, like those of the
package's dense products, carry no gradient to inputs that require one.

Like the other entries they check their arguments (``RuntimeError``), return
new tensors on the inputs' device, run asynchronously on that device's current
stream, and can be captured into CUDA graphs.  There is no CPU or library
fallback.  Inputs are contiguous; products need K to be a multiple of 16 (int8,
at most 131056, so that the int32 sums are exact) or 8 (16 bits); the number of rows is arbitrary.

``offsets`` (int32, groups + 1 values on the device) are the ascending row
bounds of the groups: group e is rows ``offsets[e]`` to ``offsets[e + 1] - 1``,
any of them empty.  Rows outside every group (a padded batch) give zeros in a
new result and are left alone in a given one (``out``, which overlaps no input
and, as with torch's own ``out=``, requires no gradient and counts as changed in
place).  Offsets that descend or exceed the rows are clamped, never followed out
of range.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .gemm import _check, _stream_ptr

_TYPES = {torch.float32: nat.TCG_F32, torch.float16: nat.TCG_F16, torch.bfloat16: nat.TCG_BF16}
_HALVES = (torch.float16, torch.bfloat16)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# The calls that are bound by the host when they are small (quantize_rows_int8,
# linear_int8, gemm_grouped, linear and their like) go through the torch binding,
# csrc/tcg_torch.cpp, checks included; the others through ctypes.

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


def _overlap(a, b) -> bool:
    """Whether two contiguous tensors share memory."""
    return (a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() and
            b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def _grouped_out(out, A, inputs, M: int, N: int, dtype):
    """(result, zero_rest): a new result whose rows outside the groups become
    zeros, or the given one, whose rows there stay."""
    if out is None:
        return A.new_empty((M, N), dtype=dtype), 1
    if not (out.is_cuda and out.is_contiguous() and out.shape == (M, N) and out.dtype == dtype):
        raise RuntimeError(f"out must be a contiguous CUDA tensor of shape {(M, N)} and type {dtype}")
    _same_device(A, "out", out)
    _check(not any(_overlap(out, t) for t in inputs if t is not None), "out must not overlap the inputs")
    _check(not (torch.is_grad_enabled() and out.requires_grad), "out must not require grad")
    _check(torch.is_inference_mode_enabled() or not out.is_inference(),
           "out must not be an inference tensor outside inference mode")
    torch.autograd.graph.increment_version(out)  # autograd: what was saved of it is stale
    return out, 0


# --------------------------------------------------------- int8 with scales --

def quantize_rows_int8(x: torch.Tensor):
    """Absmax quantisation of each row (the last axis) of a float32, float16 or
    bfloat16 tensor: codes int8 of x's shape and scales float32 of its leading
    shape, scale = max|x| / 127 and codes rounded half away from zero, as
    quantize_absmax_int8 does per tensor.  codes times scale are within half a
    step, max|x| / 254, of x as long as max|x| is a normal fp32 number or 0 (in a
    row of subnormal values, below 1.2e-38, they are 0 and +-max|x|).  A row of
    zeros has scale 0; a row with an infinity or a NaN gets a scale that is not
    finite."""
    return nat.torch_binding().quantize_rows(x)


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


def linear_int8(x: torch.Tensor, BT: torch.Tensor, scale_b: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """y[..., N] in x's type = x[..., K] quantised per row (quantize_rows_int8)
    times BT[N,K] int8 with scale_b[N] per channel, plus bias[N]: one call from
    activations to activations (gemm_int8_scaled between)."""
    return nat.torch_binding().linear_int8(x, BT, None, scale_b, bias, None)


def linear_int8_grouped(x: torch.Tensor, BT: torch.Tensor, offsets: torch.Tensor, scale_b: torch.Tensor,
                        bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """As linear_int8 for grouped rows x[M,K]: group e meets BT[e] of
    BT[E,N,K], with scale_b and bias [E,N]."""
    return nat.torch_binding().linear_int8(x, BT, offsets, scale_b, bias, out)


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
    C, rest = _grouped_out(out, A, (A, BT, offsets, scale_a, scale_b, bias), M, N, out_dtype)
    _call("tcg_gemm_s8_grouped", A, A.data_ptr(), BT.data_ptr(), C.data_ptr(), _TYPES[out_dtype], offsets.data_ptr(),
          E, M, N, K, scale_a.data_ptr(), scale_b.data_ptr(), _ptr(bias), rest)
    return C


# ------------------------------------------------------- 16-bit, by groups --

def gemm_grouped(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, b_layout: str = "nk",
                 out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """C[M,N] = rows of A[M,K] (float16 or bfloat16) times their group's matrix
    of B: [E,N,K] (b_layout="nk") or [E,K,N] ("kn"), fp32 sums, rounded once to
    out_dtype (float16, bfloat16 or float32; A's type unless given)."""
    _check(b_layout in ("nk", "kn"), "b_layout must be 'nk' or 'kn'")
    return nat.torch_binding().gemm_grouped(A, B, offsets, b_layout == "nk", out_dtype, out)


def gemm_grouped_wgrad(dC: torch.Tensor, A: torch.Tensor, offsets: torch.Tensor,
                       scale_a: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dB[E,N,K], the gradient of gemm_grouped by B ("nk"): for each group the
    sum over its rows m of dC[m,N] (float16 or bfloat16) outer A[m,K], zero for
    an empty group; fp32 sums, rounded once to out_dtype (float16, bfloat16 or
    float32; dC's type unless given).  A has dC's type, or is the int8 codes of quantize_rows_int8 with
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
        A = _dequantize(A, scale_a, dC.dtype)
    N, K = dC.size(1), A.size(1)
    dB = dC.new_empty((groups, N, K), dtype=out_dtype)
    _call("tcg_gemm_16_grouped_wgrad", dC, dC.data_ptr(), A.data_ptr(), _TYPES[dC.dtype], dB.data_ptr(),
          _TYPES[out_dtype], offsets.data_ptr(), groups, dC.size(0), N, K)
    return dB


# ------------------------------------------------------------------ layers --

def linear(x: torch.Tensor, W: torch.Tensor, save: str = "input") -> torch.Tensor:
    """y[..., N] = x[..., K] W[N,K]^T (float16 or bfloat16, fp32 sums),
    differentiable by x and W.  save="int8" keeps x for the backward pass as
    int8 codes with a scale per row, half of its bytes (the backward pass widens
    one layer's codes at a time): the output and x's gradient are unchanged, W's
    gradient is that of code * scale rounded to x's type (half a step of that
    type on top of the codes' half step)."""
    _check(save in ("input", "int8"), "save must be 'input' or 'int8'")
    return nat.torch_binding().linear(x, W, None, save == "int8")


def linear_grouped(x: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, save: str = "input") -> torch.Tensor:
    """As linear for grouped rows x[M,K]: group e meets W[e] of W[E,N,K].  Rows
    outside every group give zero outputs and get zero gradients."""
    _check(save in ("input", "int8"), "save must be 'input' or 'int8'")
    return nat.torch_binding().linear(x, W, offsets, save == "int8")


def set_rows_tile(rows: int, split: int = 0) -> None:
    """Force the tile (16, 32, 64, 128 or 256 rows) and the number of CTAs that
    share a tile's sum (1, 2, 4, 8) of these products; 0 restores the choice."""
    nat.lib().tcg_set_rows_tile(int(rows), int(split))
