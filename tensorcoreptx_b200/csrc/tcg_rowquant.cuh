// tcg_rowquant.cuh -- the arithmetic of absmax quantisation that the quantising
// kernels (tcg_quant.cuh) and the product that quantises its own rows
// (tcg_fewrows.cuh) share.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tcg {

__device__ __forceinline__ float quant_inv(float absmax, float qmax)
{
    const float scale = __fdiv_rn(absmax, qmax);
    return scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
}

__device__ __forceinline__ int quant_code(float x, float inv, float qmax)
{
    float q = __fmul_rn(x, inv);
    if (q > qmax) q = qmax;
    if (q < -qmax) q = -qmax;
    return __float2int_rz(q >= 0.f ? __fadd_rn(q, 0.5f) : __fsub_rn(q, 0.5f));
}

__device__ __forceinline__ uint32_t quant_word8(float4 v, float inv)
{
    return (static_cast<uint32_t>(quant_code(v.x, inv, 127.f)) & 0xFFu) |
           ((static_cast<uint32_t>(quant_code(v.y, inv, 127.f)) & 0xFFu) << 8) |
           ((static_cast<uint32_t>(quant_code(v.z, inv, 127.f)) & 0xFFu) << 16) |
           ((static_cast<uint32_t>(quant_code(v.w, inv, 127.f)) & 0xFFu) << 24);
}

// How a row's values become codes: code = x * lift * inv, rounded.  The inverse of
// a scale of 2^-128 or less (largest value below 127 * 2^-128 = 3.7e-37) passes
// the range of fp32; rows up to 1e-30 and their scales are therefore taken 2^64
// times as large, which is exact and changes no code where the plain inverse is
// in range.  A row whose largest value is subnormal (below 2^-126) has no scale of
// full precision either; it keeps the plain arithmetic, as the per-tensor quantiser
// has it: its codes are +-127 and 0, a value's sign with the row's largest size.
constexpr float kLift = 0x1p64f;

// scale and inverse are ordinary numbers, or the row is all zeros (padding)
__device__ __forceinline__ bool row_plain(float absmax)
{
    return absmax == 0.f || (absmax > 1e-30f && absmax < 3e38f);
}
__device__ __forceinline__ float row_lift(float absmax)
{
    return absmax >= 0x1p-126f && absmax <= 1e-30f ? kLift : 1.f;
}
__device__ __forceinline__ float row_inv(float absmax)
{
    const float s = __fmul_rn(__fdiv_rn(absmax, 127.f), row_lift(absmax));
    return s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
}

template <class T>
__device__ __forceinline__ float row_value(T v) { return static_cast<float>(v); }

// 16 bytes of a row as floats
template <class T>
struct RowVec {
    static constexpr int kN = 16 / sizeof(T);
    float f[kN];
    __device__ __forceinline__ explicit RowVec(const uint4& v)
    {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < kN; ++i) f[i] = row_value(e[i]);
    }
};

// Largest magnitude, on bit patterns: of fp32 values a word, of 16-bit values
// two lanes of a word (row_magnitude brings both forms to fp32).
template <class T>
__device__ __forceinline__ uint32_t row_absmax(const uint4& v, uint32_t m)
{
    if constexpr (sizeof(T) == 4) {
        return max(max(max(m, v.x & 0x7FFFFFFFu), v.y & 0x7FFFFFFFu), max(v.z & 0x7FFFFFFFu, v.w & 0x7FFFFFFFu));
    } else {
        const uint32_t a = __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu);
        const uint32_t b = __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu);
        return __vmaxu2(m, __vmaxu2(a, b));
    }
}

template <class T>
__device__ __forceinline__ float row_magnitude(uint32_t m)
{
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(m);
    } else {
        const unsigned short h = static_cast<unsigned short>(max(m & 0xFFFFu, m >> 16));
        return row_value(*reinterpret_cast<const T*>(&h));
    }
}

// The signs of a and b in all bits of bytes 0 and 1 (prmt: bit 3 of a selector
// copies the selected byte's sign).
__device__ __forceinline__ uint32_t sign_bytes(float a, float b)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, 0x00FB;" : "=r"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    return r;
}

template <class T>
__device__ __forceinline__ void store_codes(const uint32_t (&w)[RowVec<T>::kN / 4], int8_t* out)
{
    if constexpr (RowVec<T>::kN == 8)
        *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint32_t*>(out) = w[0];
}

// Codes of 16 bytes of a plain row: |x| * inv is at most 127 (1 + 2^-22) and needs
// no lift and no clamp; then the magnitude's code is read from the mantissa of
// (|x| * inv + 0.5) + 2^23, the last sum rounded towards zero, and the signs are
// put in four bytes at a time.  The roundings are those of quant_code, without its
// conversions, compares and selects: 7 instructions a value instead of 16, which
// bound the kernel (bf16 8192 x 4096: 31 us; 17 so, with any_codes in a loop of
// its own -- 20 with both in every unrolled step).
template <class T>
__device__ __forceinline__ void plain_codes(const uint4& v, float inv, int8_t* out)
{
    const RowVec<T> x(v);
    uint32_t w[RowVec<T>::kN / 4];
#pragma unroll
    for (int i = 0; i < RowVec<T>::kN / 4; ++i) {
        const float* f = x.f + 4 * i;
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            u[j] = __float_as_uint(__fadd_rz(__fadd_rn(__fmul_rn(fabsf(f[j]), inv), 0.5f), 8388608.f));
        const uint32_t m = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
        const uint32_t neg = __byte_perm(sign_bytes(f[0], f[1]), sign_bytes(f[2], f[3]), 0x5410);
        const uint32_t minus = (0x80808080u - m) ^ 0x80808080u;  // -m in every byte (m <= 127: no borrow)
        w[i] = (m & ~neg) | (minus & neg);
    }
    store_codes<T>(w, out);
}

// Codes of 16 bytes of any row.
template <class T>
__device__ __forceinline__ void any_codes(const uint4& v, float inv, float lift, int8_t* out)
{
    const RowVec<T> x(v);
    uint32_t w[RowVec<T>::kN / 4];
#pragma unroll
    for (int i = 0; i < RowVec<T>::kN / 4; ++i) {
        const float* f = x.f + 4 * i;
        w[i] = quant_word8(make_float4(f[0] * lift, f[1] * lift, f[2] * lift, f[3] * lift), inv);
    }
    store_codes<T>(w, out);
}

}  // namespace tcg
