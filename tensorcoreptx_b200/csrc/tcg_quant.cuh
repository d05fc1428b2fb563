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

#include "tcg_ptx.cuh"
#include "tcg_rowquant.cuh"

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

// The quantise passes walk the input from its end: the absmax pass just
// left the end of the input in L2, so the first part of this read hits there.
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
// arithmetic above with Q = 127 and the row's own absmax, lifted as row_lift has it.  kGroup threads
// (a warp or a block) take a row.  The row is read once: kVecs 16-byte vectors a
// thread stay in registers between the absmax and the codes; what is longer is
// read again, from L2.  A warp holds a row of up to 16 KB that way, with no
// barrier and all of its loads in flight; a block per row is for few or longer
// rows.  A row of zeros has scale 0 and codes 0.  The absmax is taken on the bit
// patterns, where infinity and NaN are the largest: such a row gets a scale that
// is not finite, and codes that dequantise to NaN.
constexpr int kRowThreads = 256;

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
        const float inv = row_inv(absmax);
        if (!live) continue;
        if (t == 0) scale[row] = __fdiv_rn(absmax, 127.f);
        const float lift = row_lift(absmax);
        if (kVecs > 0 && row_plain(absmax)) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                if (t + u * kGroup < nv) plain_codes<T>(v[u], inv, orow + (t + u * kGroup) * kN);
            for (int i = t + kVecs * kGroup; i < nv; i += kGroup) plain_codes<T>(xv[i], inv, orow + i * kN);
        } else if (kVecs > 0) {  // (rare: very small, very large or not finite values; read again)
#pragma unroll 1
            for (int i = t; i < nv; i += kGroup) any_codes<T>(xv[i], inv, lift, orow + i * kN);
        } else {
            for (int i = t; i < k; i += kGroup)
                orow[i] = static_cast<int8_t>(quant_code(row_value(xr[i]) * lift, inv, 127.f));
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
