// tcg_fewrows.cuh -- linear_int8 of a few rows in one kernel without tensor
// cores: y[m][n] = (sum_k codes[m][k] * B[n][k]) * scale[m] * scale_b[n] + bias[n]
// with the rows quantised on the way.
//
// The weights' N x K bytes bound it (4096 x 4096: 2.6 us of 16.8 MB), then the
// latency of one launch.  So: a warp takes whole rows of the weights (channels),
// 16 bytes a lane and load, eight loads in flight, the first eight before
// anything else; every block meanwhile quantises all of x into shared memory (by
// the arithmetic and with the results of quantize_rows_kernel; 8 KB of L2 reads a
// row); and the products are four-way byte dot products on 32-bit integers, exact
// in any order, so the result is that of the tensor-core path bit for bit.
// Nothing is split, so nothing has to be exchanged.
// us, against quantize_rows_kernel and a product of tensor-core tiles split over
// up to four CTAs: 4096 x 4096 one row 4.2 (8.8), two 4.8 (8.9), four 7.1 (8.9);
// 8192 x 8192 one 8.9 (12.6), two 10.7 (12.7), three 14.0 (12.5); 1024 x 1024
// one 2.3 (6.9), four 4.9 (6.9); 300 x 8192 three 7.0 (7.7), four 8.5 (7.7).
// Past one row the dot products bound it, hence the limits below; two channels a
// warp halve the reads of the codes (4096 x 4096, four rows 8.5 -> 7.1) and pay
// where there are channels enough for every SM's warps.
#pragma once

#include "tcg_ptx.cuh"
#include "tcg_rowquant.cuh"

namespace tcg {

constexpr int kFewRows = 4;            // most rows
constexpr int kFewThreads = 512;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewCodes = 24576;       // most codes (rows x K): one warp's work per channel
constexpr long long kFewWork = 1LL << 27;  // most products (rows x N x K)
constexpr int kFewPair = 2048;         // channels from which a warp takes two
constexpr int kFewLoads = 8;           // 16-byte loads of weights in flight per lane, of kF channels together

struct FewParams {
    const void* x;
    const int8_t* B;
    void* out;
    const float* scale_b;
    const float* bias;  // or null
    int n, k, out_type; // tcg_dtype
};

template <class T, int kM, int kF>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const FewParams p)
{
    extern __shared__ uint4 few_codes[];  // [kM][k / 16]
    __shared__ uint32_t part[kM][kFewWarps];
    __shared__ float scale[kM], inv[kM], tops[kM];
    constexpr int kN = RowVec<T>::kN;
    constexpr int kU = kFewLoads / kF;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int chunks = p.k / 16;  // of a row of B
    const int stride = static_cast<int>(gridDim.x) * kFewWarps * kF;
    int n = (static_cast<int>(blockIdx.x) * kFewWarps + warp) * kF;  // channels n .. n + kF - 1
    grid_dependency_wait();
    grid_launch_dependents();

    uint4 w[kF][kU];
    const auto load = [&](int row, int c0) {
#pragma unroll
        for (int f = 0; f < kF; ++f) {
            const uint4* b = reinterpret_cast<const uint4*>(p.B + static_cast<long long>(row + f) * p.k);
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int c = c0 + u * 32 + lane;
                w[f][u] = c < chunks && row + f < p.n ? __ldg(b + c) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    if (n < p.n) load(n, 0);

    const uint4* x = static_cast<const uint4*>(p.x);
    const int nv = p.k / kN;  // vectors of a row of x
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        uint32_t top = 0u;
        for (int i = t; i < nv; i += kFewThreads) top = row_absmax<T>(x[static_cast<long long>(m) * nv + i], top);
        top = __reduce_max_sync(0xffffffffu, __float_as_uint(row_magnitude<T>(top)));
        if (lane == 0) part[m][warp] = top;
    }
    __syncthreads();
    if (t < kM) {
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < kFewWarps; ++i) top = max(top, part[t][i]);
        const float absmax = __uint_as_float(top);
        scale[t] = __fdiv_rn(absmax, 127.f);
        inv[t] = row_inv(absmax);
        tops[t] = absmax;
    }
    __syncthreads();
    int8_t* codes = reinterpret_cast<int8_t*>(few_codes);
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const uint4* row = x + static_cast<long long>(m) * nv;
        int8_t* to = codes + static_cast<long long>(m) * p.k;
        if (row_plain(tops[m])) {
            for (int i = t; i < nv; i += kFewThreads) plain_codes<T>(row[i], inv[m], to + i * kN);
        } else {
#pragma unroll 1
            for (int i = t; i < nv; i += kFewThreads) any_codes<T>(row[i], inv[m], row_lift(tops[m]), to + i * kN);
        }
    }
    __syncthreads();

    for (bool loaded = true; n < p.n; n += stride, loaded = false) {
        // lane f * kM + m finishes row m of channel n + f
        const int mine = n + lane / kM;
        const bool live = lane < kF * kM && mine < p.n;
        const float sb = live ? p.scale_b[mine] : 0.f, bias = live && p.bias ? p.bias[mine] : 0.f;
        int sum[kF][kM] = {};
        for (int c0 = 0; c0 < chunks; c0 += 32 * kU) {
            if (!loaded) load(n, c0);
            loaded = false;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int c = min(c0 + u * 32 + lane, chunks - 1);  // (past the row: weights of zero)
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    const uint4 a = few_codes[m * chunks + c];
#pragma unroll
                    for (int f = 0; f < kF; ++f) {
                        int d = sum[f][m];
                        d = __dp4a(static_cast<int>(a.x), static_cast<int>(w[f][u].x), d);
                        d = __dp4a(static_cast<int>(a.y), static_cast<int>(w[f][u].y), d);
                        d = __dp4a(static_cast<int>(a.z), static_cast<int>(w[f][u].z), d);
                        sum[f][m] = __dp4a(static_cast<int>(a.w), static_cast<int>(w[f][u].w), d);
                    }
                }
            }
        }
        int total = 0;
#pragma unroll
        for (int f = 0; f < kF; ++f)
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const int all = __reduce_add_sync(0xffffffffu, sum[f][m]);
                if (lane == f * kM + m) total = all;
            }
        if (live) {
            const int m = lane % kM;
            const float y = fmaf(__int2float_rn(total) * scale[m], sb, bias);
            const long long at = static_cast<long long>(m) * p.n + mine;
            if (p.out_type == 0)
                static_cast<float*>(p.out)[at] = y;
            else if (p.out_type == 1)
                static_cast<__half*>(p.out)[at] = __float2half_rn(y);
            else
                static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
        }
    }
}

}  // namespace tcg
