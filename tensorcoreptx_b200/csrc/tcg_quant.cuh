// tcg_quant.cuh -- per-tensor absmax quantisation fp32 -> int8 / packed int4 on
// the device: the producers of the integer GEMM's inputs.
//
// Replaces the reference's host loops quantize_absmax (src/data_int8.cu:74-89)
// and quantize_absmax_int4 (src/data_int4.cu:104-127) with three launches:
// an absmax reduction, the elementwise quantisation, and a one-thread kernel
// that publishes the scale.  Every float operation uses an explicitly rounded
// intrinsic (no contraction into FMA), so the codes and the scale are
// bit-identical to the reference's IEEE single-precision host arithmetic:
//   scale = absmax / Q;  inv = scale > 0 ? 1 / scale : 0;
//   q = clamp(x * inv, -Q, Q);  code = (int)(q >= 0 ? q + 0.5 : q - 0.5)
// with Q = 127 (int8) or 7 (int4, two codes per byte, low nibble = even k).
// HBM-bound: one read pass for the absmax, one read + 1/4 (int8) or 1/8
// (int4) write pass for the codes, walking the input backwards so that it
// starts on what the absmax pass left in L2.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcg_ptx.cuh"

namespace tcg {

// |x| max over n floats into *absmax_bits (float bits, must start at +0).
// Non-negative floats order like their bit patterns as signed ints.  Four
// 16-byte loads in flight per thread per step.
__global__ void absmax_kernel(const float* __restrict__ x, long long n, int* __restrict__ absmax_bits)
{
    float m = 0.f;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    const long long n4 = n / 4;
    const float4* x4 = reinterpret_cast<const float4*>(x);
    long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    for (; i + 3 * stride < n4; i += 4 * stride) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = x4[i + u * stride];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            m = fmaxf(m, fmaxf(fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w))));
    }
    for (; i < n4; i += stride) {
        const float4 v = x4[i];
        m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
    }
    for (long long j = n4 * 4 + static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; j < n; j += stride)
        m = fmaxf(m, fabsf(x[j]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __shared__ float wmax[32];
    if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = threadIdx.x < (blockDim.x >> 5) ? wmax[threadIdx.x] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (threadIdx.x == 0) atomicMax(absmax_bits, __float_as_int(m));
    }
}

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

// The quantise passes walk the input from its end: the absmax pass just
// left the end of the input in L2, so the first part of this read hits there.
__device__ __forceinline__ uint32_t quant_word8(float4 v, float inv)
{
    return (static_cast<uint32_t>(quant_code(v.x, inv, 127.f)) & 0xFFu) |
           ((static_cast<uint32_t>(quant_code(v.y, inv, 127.f)) & 0xFFu) << 8) |
           ((static_cast<uint32_t>(quant_code(v.z, inv, 127.f)) & 0xFFu) << 16) |
           ((static_cast<uint32_t>(quant_code(v.w, inv, 127.f)) & 0xFFu) << 24);
}

__global__ void quantize_s8_kernel(const float* __restrict__ x, int8_t* __restrict__ out, long long n,
                                   const int* __restrict__ absmax_bits)
{
    const float inv = quant_inv(__int_as_float(*absmax_bits), 127.f);
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    const long long n4 = n / 4;
    const float4* x4 = reinterpret_cast<const float4*>(x);
    uint32_t* o4 = reinterpret_cast<uint32_t*>(out);
    long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    for (; i + stride < n4; i += 2 * stride) {
        const long long j0 = n4 - 1 - i, j1 = n4 - 1 - (i + stride);
        const float4 v0 = x4[j0];
        const float4 v1 = x4[j1];
        o4[j0] = quant_word8(v0, inv);
        o4[j1] = quant_word8(v1, inv);
    }
    for (; i < n4; i += stride) {
        const long long j = n4 - 1 - i;
        o4[j] = quant_word8(x4[j], inv);
    }
    for (long long j = n4 * 4 + static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; j < n; j += stride)
        out[j] = static_cast<int8_t>(quant_code(x[j], inv, 127.f));
}

__device__ __forceinline__ uint32_t quant_byte4(float2 v, float inv)
{
    const int lo = quant_code(v.x, inv, 7.f);
    const int hi = quant_code(v.y, inv, 7.f);
    return static_cast<uint32_t>((lo & 0x0F) | ((hi & 0x0F) << 4));
}

// rows x cols_k floats -> rows x cols_k/2 bytes; byte = lo | hi << 4 with lo
// the code of the even column.  Eight floats (four output bytes) per step.
__global__ void quantize_s4_kernel(const float* __restrict__ x, int8_t* __restrict__ out, long long n_pairs,
                                   const int* __restrict__ absmax_bits)
{
    const float inv = quant_inv(__int_as_float(*absmax_bits), 7.f);
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    const long long n_g = n_pairs / 4;  // groups of 4 pairs: two float4 in, one 32-bit word out
    const float4* x4 = reinterpret_cast<const float4*>(x);
    uint32_t* o4 = reinterpret_cast<uint32_t*>(out);
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n_g; i += stride) {
        const long long j = n_g - 1 - i;
        const float4 a = x4[2 * j];
        const float4 b = x4[2 * j + 1];
        o4[j] = quant_byte4(make_float2(a.x, a.y), inv) | (quant_byte4(make_float2(a.z, a.w), inv) << 8) |
                (quant_byte4(make_float2(b.x, b.y), inv) << 16) | (quant_byte4(make_float2(b.z, b.w), inv) << 24);
    }
    const float2* x2 = reinterpret_cast<const float2*>(x);
    for (long long j = n_g * 4 + static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; j < n_pairs; j += stride)
        out[j] = static_cast<int8_t>(quant_byte4(x2[j], inv));
}

// ---- one scale per row ----------------------------------------------------
//
// codes[m][k] and scale[m] of each row m of fp32, fp16 or bf16 values, by the
// arithmetic above with Q = 127 and the row's own absmax.  kGroup threads (a
// warp or a block) take a row.  The row is read once: kVecs 16-byte vectors a
// thread stay in registers between the absmax and the codes; what is longer is
// read again, from L2.  A warp holds a row of up to 16 KB that way, with no
// barrier and all of its loads in flight; a block per row is for few or longer
// rows.  A row of zeros has scale 0 and codes 0.  The absmax is taken on the bit
// patterns, where infinity and NaN are the largest: such a row gets a scale that
// is not finite, and codes that dequantise to NaN.
constexpr int kRowThreads = 256;

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

// Codes of 16 bytes.  `plain`: the row's scale and its inverse are ordinary
// numbers, so |x| * inv is at most 127 (1 + 2^-22) and needs no clamp; then the
// magnitude's code is read from the mantissa of (|x| * inv + 0.5) + 2^23, the
// last sum rounded towards zero, and the signs are put in four bytes at a time.
// The roundings are those of quant_code, without its conversions, compares and
// selects: 7 instructions a value instead of 16, which bound the kernel (bf16
// 8192 x 4096: 31 us).
template <class T>
__device__ __forceinline__ void row_codes(const uint4& v, float inv, bool plain, int8_t* out)
{
    const RowVec<T> x(v);
    uint32_t w[RowVec<T>::kN / 4];
#pragma unroll
    for (int i = 0; i < RowVec<T>::kN / 4; ++i) {
        const float* f = x.f + 4 * i;
        if (plain) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                u[j] = __float_as_uint(__fadd_rz(__fadd_rn(__fmul_rn(fabsf(f[j]), inv), 0.5f), 8388608.f));
            const uint32_t m = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
            const uint32_t neg = __byte_perm(sign_bytes(f[0], f[1]), sign_bytes(f[2], f[3]), 0x5410);
            const uint32_t minus = (0x80808080u - m) ^ 0x80808080u;  // -m in every byte (m <= 127: no borrow)
            w[i] = (m & ~neg) | (minus & neg);
        } else {
            w[i] = quant_word8(make_float4(f[0], f[1], f[2], f[3]), inv);
        }
    }
    if constexpr (RowVec<T>::kN == 8)
        *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint32_t*>(out) = w[0];
}

// kVecs = 0: rows that are not whole 16-byte vectors (or a dst that does not
// take their codes in one store)
template <class T, int kGroup, int kVecs>
__global__ void __launch_bounds__(kRowThreads)
    quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ out, float* __restrict__ scale, long long rows,
                         int k)
{
    constexpr int kRows = kRowThreads / kGroup;  // rows per block
    constexpr int kN = RowVec<T>::kN;
    __shared__ uint32_t wmax[kRowThreads / 32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int t = threadIdx.x % kGroup;
    for (long long row0 = static_cast<long long>(blockIdx.x) * kRows; row0 < rows;
         row0 += static_cast<long long>(gridDim.x) * kRows) {
        const long long row = row0 + threadIdx.x / kGroup;
        const bool live = row < rows;
        const T* xr = x + row * k;
        int8_t* orow = out + row * k;
        const int nv = kVecs ? k / kN : 0;
        const uint4* xv = reinterpret_cast<const uint4*>(xr);
        uint4 v[kVecs ? kVecs : 1];
        uint32_t m = 0u;
        if (live && kVecs) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                if (t + u * kGroup < nv) v[u] = xv[t + u * kGroup];
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                if (t + u * kGroup < nv) m = row_absmax<T>(v[u], m);
            for (int i = t + kVecs * kGroup; i < nv; i += kGroup) m = row_absmax<T>(xv[i], m);
        } else if (live) {
            for (int i = t; i < k; i += kGroup) m = max(m, __float_as_uint(row_value(xr[i])) & 0x7FFFFFFFu);
        }
        if constexpr (kVecs > 0) m = __float_as_uint(row_magnitude<T>(m));
        m = __reduce_max_sync(0xffffffffu, m);
        if constexpr (kGroup > 32) {
            __syncthreads();  // the last row's maxima have been read
            if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
            __syncthreads();
            m = wmax[0];
#pragma unroll
            for (int w = 1; w < kRowThreads / 32; ++w) m = max(m, wmax[w]);
        }
        const float absmax = __uint_as_float(m);
        const float inv = quant_inv(absmax, 127.f);
        const bool plain = absmax > 1e-30f && absmax < 3e38f;
        if (!live) continue;
        if (t == 0) scale[row] = __fdiv_rn(absmax, 127.f);
        if constexpr (kVecs > 0) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                if (t + u * kGroup < nv) row_codes<T>(v[u], inv, plain, orow + (t + u * kGroup) * kN);
            for (int i = t + kVecs * kGroup; i < nv; i += kGroup) row_codes<T>(xv[i], inv, plain, orow + i * kN);
        } else {
            for (int i = t; i < k; i += kGroup) orow[i] = static_cast<int8_t>(quant_code(row_value(xr[i]), inv, 127.f));
        }
    }
}

// The way back: code * scale[row] in fp32, rounded once to T (at most half a
// step of T, against the half code step, 2^-8 of the row's largest value, that
// the codes are off by).  kCodes codes a thread and step, whole rows of them
// (kCodes = 16: one 16-byte load) or one by one.  HBM bound: 1 byte read and 2
// (4) written a value.
template <class T>
__device__ __forceinline__ T row_result(float f) { return T(f); }

template <class T, int kCodes>
__global__ void __launch_bounds__(kRowThreads)
    dequantize_rows_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ out,
                           long long rows, int k)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int per_row = k / kCodes;
    const long long total = rows * per_row;
    const long long stride = static_cast<long long>(gridDim.x) * kRowThreads;
    for (long long i = static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += stride) {
        const float s = scale[total <= 0x7fffffffLL ? static_cast<int>(i) / per_row : i / per_row];
        if constexpr (kCodes == 16) {
            const uint4 v = reinterpret_cast<const uint4*>(q)[i];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            alignas(16) T o[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
                o[j] = row_result<T>(static_cast<float>(static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)))) * s);
            uint4* to = reinterpret_cast<uint4*>(out) + i * sizeof(T);
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) to[j] = reinterpret_cast<const uint4*>(o)[j];
        } else {
            out[i] = row_result<T>(static_cast<float>(q[i]) * s);
        }
    }
}

// *scale = absmax / qmax, written over the absmax slot once every quantise
// block has read it (stream order).
__global__ void publish_scale_kernel(float* scale_and_absmax, float qmax)
{
    scale_and_absmax[0] = __fdiv_rn(scale_and_absmax[0], qmax);
}

}  // namespace tcg
