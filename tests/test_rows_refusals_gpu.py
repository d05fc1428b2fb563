"""The Python surface's refusals of CUDA tensors for the row-scaled and grouped
products: each raises before anything is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def z(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype, device=DEV)


def refuse(match, f, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        f(*args, **kw)


def test_quantize_and_int8_products():
    import tensorcoreptx_b200 as T
    i8, f32 = torch.int8, torch.float32
    o = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    refuse("contiguous", T.quantize_rows_int8, z(8, 8).t()[:, ::2])
    refuse("float32, float16", T.quantize_rows_int8, z(4, 8, dtype=i8))
    refuse("at least one axis", T.quantize_rows_int8, z())
    refuse("CUDA int8", T.dequantize_rows_int8, z(4, 8), z(4, dtype=f32))
    refuse("scales must have shape", T.dequantize_rows_int8, z(4, 8, dtype=i8), z(8, dtype=f32))
    refuse("dtype must be", T.dequantize_rows_int8, z(4, 8, dtype=i8), z(4, dtype=f32), i8)
    a, b, sa, sb = z(4, 16, dtype=i8), z(6, 16, dtype=i8), z(4, dtype=f32), z(6, dtype=f32)
    refuse("must be int8", T.gemm_int8_scaled, z(4, 16), b, sa, sb)
    refuse("cols must equal", T.gemm_int8_scaled, a, z(6, 32, dtype=i8), sa, sb)
    refuse("scale_a must have shape", T.gemm_int8_scaled, a, b, sb, sb)
    refuse("scale_b must have shape", T.gemm_int8_scaled, a, b, sa, sa)
    refuse("scale_b must be a contiguous CUDA float32", T.gemm_int8_scaled, a, b, sa, sb.half())
    refuse("bias must have shape", T.gemm_int8_scaled, a, b, sa, sb, sa)
    refuse("out_dtype", T.gemm_int8_scaled, a, b, sa, sb, out_dtype=torch.int8)
    refuse("must be contiguous", T.gemm_int8_scaled, z(16, 4, dtype=i8).t(), b, sa, sb)
    refuse("SHAPE", T.gemm_int8_scaled, z(4, 24, dtype=i8), z(6, 24, dtype=i8), sa, sb)
    refuse("scale_a must be a contiguous CUDA", T.gemm_int8_scaled, a, b, sa.cpu(), sb)
    refuse("x must be float32", T.linear_int8, a, b, sb)
    refuse("K must not be 0", T.linear_int8, z(4, 0), z(6, 0, dtype=i8), sb)
    g = z(2, 6, 16, dtype=i8)
    refuse("BT must be 2-D", T.linear_int8, z(4, 16), g, sb)
    refuse("one entry more", T.linear_int8_grouped, z(4, 16), g, o[:2], z(2, 6, dtype=f32))
    refuse("int32", T.linear_int8_grouped, z(4, 16), g, o.long(), z(2, 6, dtype=f32))
    refuse("int32", T.linear_int8_grouped, z(4, 16), g, o.cpu(), z(2, 6, dtype=f32))
    refuse("scale_b must have shape", T.linear_int8_grouped, z(4, 16), g, o, sb)
    refuse("out must be", T.linear_int8_grouped, z(4, 16), g, o, z(2, 6, dtype=f32), out=z(4, 7))
    refuse("out must be", T.gemm_int8_grouped, a, g, o, sa, z(2, 6, dtype=f32), out=z(4, 6, dtype=f32))
    x = z(4, 32)
    refuse("overlap", T.linear_int8_grouped, x.view(-1)[64:].view(4, 16), g[:, :4].contiguous(), o, z(2, 4, dtype=f32),
           out=x.view(-1)[60:76].view(4, 4))
    buf = z(4 * 16 + 4 * 6 * 2, dtype=i8)
    refuse("overlap", T.gemm_int8_grouped, buf[:64].view(4, 16), g, o, sa, z(2, 6, dtype=f32),
           out=buf[62:110].view(torch.float16).view(4, 6))


def test_16_bit_products_and_layers():
    import tensorcoreptx_b200 as T
    bf = torch.bfloat16
    o = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    a, b = z(4, 16), z(2, 8, 16)
    refuse("both be float16", T.gemm_grouped, a, b.to(bf), o)
    refuse("both be float16", T.gemm_grouped, a.float(), b.float(), o)
    refuse("b_layout", T.gemm_grouped, a, b, o, "mn")
    refuse("cols must equal", T.gemm_grouped, a, b, o, "kn")
    refuse("2-D and B 3-D", T.gemm_grouped, a, b[0], o)
    refuse("must be contiguous", T.gemm_grouped, a, z(2, 16, 8).transpose(1, 2), o)
    refuse("number of groups", T.gemm_grouped, a, z(1025, 8, 16), z(1026, dtype=torch.int32))
    refuse("SHAPE", T.gemm_grouped, z(4, 12), z(2, 8, 12), o)
    refuse("out must be", T.gemm_grouped, a, b, o, out=z(4, 8, dtype=bf))
    refuse("overlap", T.gemm_grouped, a, z(2, 16, 16), o, out=a)
    refuse("ALIGN", T.gemm_grouped, z(65)[1:].view(4, 16), b, o)
    refuse("dC's type", T.gemm_grouped_wgrad, z(4, 8), z(4, 16, dtype=bf), o)
    refuse("dC's type", T.gemm_grouped_wgrad, z(4, 8), z(4, 16), o, scale_a=z(4, dtype=torch.float32))
    refuse("same rows", T.gemm_grouped_wgrad, z(4, 8), z(3, 16), o)
    refuse("SHAPE", T.gemm_grouped_wgrad, z(4, 12), a, o)
    refuse("scale_a must have shape", T.gemm_grouped_wgrad, z(4, 8), z(4, 16, dtype=torch.int8), o,
           scale_a=z(3, dtype=torch.float32))
    refuse("number of groups", T.gemm_grouped_wgrad, z(4, 8), a, o[:1])
    refuse("save must be", T.linear, a, b[0], save="fp8")
    refuse("multiple of 8", T.linear, z(4, 12), z(8, 12))
    refuse("multiple of 8", T.linear, z(4, 20), z(8, 20), save="int8")
    refuse("N must be", T.linear, a, z(12, 16))
    refuse("must not be empty", T.linear, z(4, 0), z(8, 0))
    refuse("must be contiguous", T.linear, z(16, 4).t(), b[0])
