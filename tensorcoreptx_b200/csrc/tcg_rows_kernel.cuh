// tcg_rows_kernel.cuh -- products whose rows carry structure: rows grouped by
// expert (ragged groups whose bounds are on the device), int8 rows with a
// scale each, and the gradient of such products.
//
// One kernel computes, for every group e, a matrix D_e[p][q] on the tensor
// cores and writes it transposed, out[q][p] with p contiguous:
//
//   rows form    p = an output feature (a row of group e's weights)
//                q = a row of the group             (rows bound[e] .. bound[e+1])
//                sum over the K input features      out[row][feature]
//   weight form  p = an input feature, q = an output feature
//                sum over the rows of the group     out[e][q][p] (a weight gradient)
//
// Putting the rows of the activations on the N side of tcgen05.mma and the
// weights on its M side is what makes ragged groups and single rows cheap:
// N is any multiple of 16, so a group of 3 rows costs a 16-column MMA and not
// a 128-row one; a tile that ends inside a group needs no masked row loop, the
// epilogue just stops at the last column; and one lane of tensor memory is one
// output feature, so a warp's store of one row is 32 consecutive elements and
// per-channel scales are one register a lane.
//
// Two sizes of tile:
//   kSub = 1: 128 features x kBQ rows, one tile per cluster.  The CTAs of a
//     cluster (1, 2, 4 or 8) split the sum between them and add their parts
//     through distributed shared memory, in rank order (the result does not
//     depend on timing).  For few rows, where the weights' bytes bound the
//     product and every SM has to pull on memory.
//   kSub = 2: 256 x 256, persistent CTAs, two M = 128 accumulators that fill
//     the tensor memory.  For many rows, where the tensor cores bound it.
//
// Warps: 0 TMA producer (one thread), 1 MMA issuer, 2..5 epilogue (one per
// tensor-memory lane quarter), and with kConv eight converter warps (see
// conv_tile).  Every wait on an mbarrier is bounded (tcg_wait.cuh).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcg_ptx.cuh"
#include "tcg_wait.cuh"

namespace tcg {

constexpr int kRowsMaxGroups = 1024;

constexpr int kOutF32 = 0, kOutF16 = 1, kOutBF16 = 2;  // tcg_dtype

struct RowsParams {
    void* out;
    const int* offsets;       // groups + 1 row bounds on the device; null: groups of `rows_per_group`
    const float* scale_q;     // int8: one per row
    const float* scale_p;     // int8: one per group and feature
    const float* bias_p;      // int8: one per group and feature, or null
    const float* scale_r;     // kConv: one per row (the rows are the reduction)
    unsigned long long timeout_ns;
    int groups, rows, rows_per_group;
    int P, Q, R;              // features out; weight form: the other features; rows form: length of the sum
    int ptiles, qtiles;       // tiles along P; weight form: along Q
    int band;                 // tiles along q per rasterisation band
    int zero_rest;            // rows form: write zeros into rows outside every group
    int out_type;
    int bf16;                 // 16-bit operands are bf16 (kConv: type of the widened codes)
    int split;                // CTAs per tile (kSub = 1)
    int early;                // the M-side operand and the offsets predate the kernel this one follows
    uint32_t idesc;           // instruction descriptor without N
};

template <int kKind_, bool kPMn_, bool kQMn_, bool kConv_, int kSub_, int kBQ_, int kStages_>
struct RowsTraits {
    static constexpr int kKind = kKind_;
    static constexpr bool kPMn = kPMn_, kQMn = kQMn_, kConv = kConv_;
    static constexpr int kSub = kSub_, kBQ = kBQ_, kStages = kStages_;
    static constexpr bool kWeight = kQMn;               // weight form: the sum runs over a group's rows
    static constexpr int kElem = kKind == kKindF16 ? 2 : 1;
    static constexpr int kBK = 128 / kElem;             // length of the sum per ring stage
    static constexpr int kUmmaK = 32 / kElem;
    static constexpr int kTileP = 128 * kSub;
    static constexpr int kSubBytes = 128 * 128;         // one 128-feature block of a stage
    static constexpr int kPBytes = kSub * kSubBytes;
    static constexpr int kQBytes = kBQ * 128;
    static constexpr int kStageBytes = kPBytes + kQBytes;
    static constexpr int kQBox = kBQ < 64 ? kBQ : 64;   // rows (weight form: columns) per box of the q operand
    static constexpr int kQBoxBytes = kQBox * 128;
    static constexpr int kRawBytes = 128 * kBK;         // kConv: int8 codes of one 128-feature block
    static constexpr int kConvWarps = kConv ? 8 : 0;
    static constexpr int kThreads = 192 + 32 * kConvWarps;
    static constexpr int kTmemCols = kSub * kBQ < 32 ? 32 : kSub * kBQ;
    static constexpr int kRedBytes = kBQ * 512;         // split: 128 x kBQ partial sums
    static constexpr int kBarBytes = 256;
    static constexpr int kRingBytes = kStages * kStageBytes;
    static_assert(!kConv || (kPMn && kQMn && kKind == kKindF16), "converted operand: weight form only");
    static_assert(!kQMn || kKind == kKindF16, "weight form: 16-bit operands");
    static_assert(!kPMn || kKind == kKindF16, "MN-major features: 16-bit operands");
    static_assert(!kQMn || kBQ % 64 == 0, "whole 64-column atoms");
    static_assert(8 * (3 * kStages + 5) + 16 <= kBarBytes, "barrier area");
    static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols <= 512, "TMEM allocation");
    // dynamic shared memory of a launch with `groups` ragged groups
    static constexpr int smem_bytes(int split, int groups_in_table)
    {
        return 1024 + kRingBytes + (split > 1 ? kRedBytes : 0) + kBarBytes + 8 * (groups_in_table + 3);
    }
};

// One tile of work.  `zero`: rows outside every group, written as zeros.
struct RowsItem {
    int e, row0, cnt, p0, q0, nkb, rend;
    bool zero;
};

// Row bounds and running tile counts of the intervals that the offsets cut
// 0 .. rows into: interval 0 before the first group, 1 .. groups the groups,
// groups + 1 behind the last.  Bounds are clamped to be ascending and inside
// the tensor, so no offsets that the device holds can lead out of range.
// One warp; bound and cum have groups + 3 entries.
__device__ __forceinline__ void rows_table(const RowsParams& p, int bq, int* bound, int* cum)
{
    const int lane = threadIdx.x & 31;
    const int n = p.groups + 2;
    int top = 0, sum = 0;
    if (lane == 0) bound[0] = 0, cum[0] = 0;
    for (int base = 0; base < n; base += 32) {
        const int i = base + lane;
        int v = i <= p.groups ? p.offsets[i] : p.rows;
        v = v < 0 ? 0 : (v > p.rows ? p.rows : v);
        v = v < top ? top : v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o && u > v) v = u;
        }
        const int before = __shfl_up_sync(0xffffffffu, v, 1);
        const int cnt = v - (lane == 0 ? top : before);
        const bool group = i >= 1 && i <= p.groups;
        int t = i < n && (group || p.zero_rest) ? (cnt + bq - 1) / bq : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        if (i < n) bound[i + 1] = v, cum[i + 1] = sum + t;
        top = __shfl_sync(0xffffffffu, v, 31);
        sum += __shfl_sync(0xffffffffu, t, 31);
    }
}

template <class C>
__device__ __forceinline__ int rows_total(const RowsParams& p, const int* cum)
{
    if (C::kWeight) return p.groups * p.ptiles * p.qtiles;
    const int tiles =
        p.offsets ? cum[p.groups + 2] : p.groups * ((p.rows_per_group + C::kBQ - 1) / C::kBQ);
    return tiles * p.ptiles;
}

// Work item -> tile.  Items walk a band of `band` q-tiles for all of P before
// the next band, so the tiles in flight share both operands in L2.
template <class C>
__device__ __forceinline__ RowsItem rows_item(const RowsParams& p, int item, int total, const int* bound,
                                              const int* cum)
{
    RowsItem w;
    w.zero = false;
    int e = 0;
    if (C::kWeight) {
        const int per = p.ptiles * p.qtiles;
        e = item / per;
        item -= e * per;
        total = per;
    }
    const int tall = total / p.ptiles;
    const int per_band = p.band * p.ptiles;
    const int b = item / per_band;
    const int r = item - b * per_band;
    const int width = min(p.band, tall - b * p.band);
    const int tq = b * p.band + r % width;
    w.p0 = (r / width) * C::kTileP;
    if (C::kWeight) {
        w.e = e;
        w.q0 = tq * C::kBQ;
        w.cnt = min(C::kBQ, p.Q - w.q0);
        w.row0 = p.offsets ? bound[e + 1] : e * p.rows_per_group;
        w.rend = p.offsets ? bound[e + 2] : (e + 1) * p.rows_per_group;
        w.nkb = (w.rend - w.row0 + C::kBK - 1) / C::kBK;
        return w;
    }
    w.q0 = 0;
    if (p.offsets) {
        int lo = 0, hi = p.groups + 1;  // the last interval whose running count is <= tq
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] <= tq)
                lo = mid;
            else
                hi = mid - 1;
        }
        w.e = lo - 1;
        w.zero = lo == 0 || lo == p.groups + 1;
        w.row0 = bound[lo] + (tq - cum[lo]) * C::kBQ;
        w.rend = bound[lo + 1];
    } else {
        const int per = (p.rows_per_group + C::kBQ - 1) / C::kBQ;
        w.e = tq / per;
        w.row0 = w.e * p.rows_per_group + (tq - w.e * per) * C::kBQ;
        w.rend = (w.e + 1) * p.rows_per_group;
    }
    w.cnt = min(C::kBQ, w.rend - w.row0);
    w.nkb = w.zero ? 0 : (p.R + C::kBK - 1) / C::kBK;
    return w;
}

// 32 accumulator words of one lane (one feature, columns c .. c + 31 of the
// tile) to the output type and out: column j is row j of the output, where the
// warp's 32 lanes write 32 consecutive elements.
template <class C, class T>
__device__ __forceinline__ void store_cols(const uint32_t (&v)[32], T* ptr, long long ld, int n, bool live, float sp,
                                           float bias, float sq_lane)
{
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        float f;
        if constexpr (C::kKind == kKindI8) {
            // the int32 sum, rounded to fp32 once, times both scales, plus the bias
            const float sq = __shfl_sync(0xffffffffu, sq_lane, j);
            f = fmaf(__int2float_rn(static_cast<int>(v[j])) * sq, sp, bias);
        } else {
            f = __uint_as_float(v[j]);
        }
        if (j < n && live) {
            if constexpr (sizeof(T) == 4)
                *ptr = f;
            else
                *ptr = T(f);  // one rounding to nearest, at the end
        }
        ptr += ld;
    }
}

// kConv: one ring stage of int8 codes (64 rows x 128 features per block, rows
// of 128 bytes) into 16-bit values code * scale[row] in the MN-major
// 128-byte-swizzled layout the MMA reads: per block two atoms of 64 features,
// an atom's row r at r * 128 with its 16-byte chunk c at c ^ (r & 7).  The
// product of code and scale is rounded to 16 bits: at most half a step of
// the operand type, against half a code step (2^-8 of the row's largest value)
// that the codes themselves are off by.
// In place: the codes land in the upper half of the stage's P area; each
// thread takes its codes into registers, and after a barrier of the converter
// warps writes them widened.  Eight consecutive threads hold one row; threads
// 4..7 write their two chunks in the other order, so the eight chunks of a
// write lie in different banks.
template <class C>
struct ConvRegs {
    uint4 v[2 * C::kSub];
    float s[2 * C::kSub];
};

// codes of one thread: pass u is 16 codes of row (u & 1) * 32 + ct / 8 of block u / 2
template <class C>
__device__ __forceinline__ void conv_codes(const uint8_t* raw, int ct, ConvRegs<C>& g)
{
#pragma unroll
    for (int u = 0; u < 2 * C::kSub; ++u)
        g.v[u] = *reinterpret_cast<const uint4*>(raw + (u >> 1) * C::kRawBytes + ((u & 1) * 32 + (ct >> 3)) * 128 +
                                                 (ct & 7) * 16);
}

__device__ __forceinline__ float code_float(uint32_t w, int i)
{
    // byte i of w (biased by 128) in the low mantissa bits of 2^23, minus 2^23 + 128: exact
    return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650 | i)) - 8388736.0f;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float a, float b)
{
    if (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <class C, bool kBf16>
__device__ __forceinline__ void conv_write(uint8_t* p_area, int ct, int valid, const ConvRegs<C>& g)
{
    const int c = ct & 7;
#pragma unroll
    for (int u = 0; u < 2 * C::kSub; ++u) {
        const int r = (u & 1) * 32 + (ct >> 3);
        uint4 o[2];
        uint32_t* ow = reinterpret_cast<uint32_t*>(o);
        const uint32_t in[4] = {g.v[u].x ^ 0x80808080u, g.v[u].y ^ 0x80808080u, g.v[u].z ^ 0x80808080u,
                                g.v[u].w ^ 0x80808080u};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ow[2 * i] = pack16<kBf16>(code_float(in[i], 0) * g.s[u], code_float(in[i], 1) * g.s[u]);
            ow[2 * i + 1] = pack16<kBf16>(code_float(in[i], 2) * g.s[u], code_float(in[i], 3) * g.s[u]);
        }
        if (r >= valid) o[0] = o[1] = make_uint4(0, 0, 0, 0);  // rows of the next group
        uint8_t* row = p_area + (u >> 1) * C::kSubBytes + (c >> 2) * 8192 + r * 128;
        const int first = c >> 2;
        *reinterpret_cast<uint4*>(row + (((2 * (c & 3) + first) ^ (r & 7)) << 4)) = first ? o[1] : o[0];
        *reinterpret_cast<uint4*>(row + (((2 * (c & 3) + (first ^ 1)) ^ (r & 7)) << 4)) = first ? o[0] : o[1];
    }
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                const __grid_constant__ RowsParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const int S = C::kSub == 1 ? p.split : 1;
    uint32_t* red = reinterpret_cast<uint32_t*>(smem + C::kRingBytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kRingBytes + (S > 1 ? C::kRedBytes : 0));
    uint64_t* empty = full + C::kStages;
    uint64_t* conv = empty + C::kStages;     // kConv: stage widened (one arrival per converter warp)
    uint64_t* tfull = conv + C::kStages;     // accumulator block h complete
    uint64_t* tempty = tfull + 2;            // accumulator block h read
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int* bound = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + C::kBarBytes);
    int* cum = bound + p.groups + 3;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
            mbar_init(smem_u32(&conv[s]), C::kConvWarps ? C::kConvWarps : 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(smem_u32(&tfull[h]), 1);
            mbar_init(smem_u32(&tempty[h]), 4);
        }
        mbar_init(smem_u32(drain), 1);
        *abort_flag = 0u;
        fence_mbar_init();
        tma_prefetch_desc(&tmP);
        tma_prefetch_desc(&tmQ);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    // Everything above overlaps the previous kernel's tail.  With `early` the
    // kernel before this one wrote only the q operand and its scales, and let
    // this one start after its own wait: features and offsets may be read now.
    if (!p.early) grid_dependency_wait();
    grid_launch_dependents();
    if (p.offsets && warp == 2) rows_table(p, C::kBQ, bound, cum);
    tc_fence_before();
    __syncthreads();
    if (S > 1) cluster_sync_all();  // every CTA of the cluster runs before any writes into another
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t ring = smem_u32(smem);

    const int total = rows_total<C>(p, cum);
    const int first = static_cast<int>(blockIdx.x) / S;
    const int stride = static_cast<int>(gridDim.x) / S;
    // this CTA's share [kb0, kb1) of a tile's k-blocks
    const auto share = [&](const RowsItem& w, int& kb0, int& kb1) {
        kb0 = static_cast<int>(static_cast<long long>(w.nkb) * rank / S);
        kb1 = static_cast<int>(static_cast<long long>(w.nkb) * (rank + 1) / S);
    };
    const auto blocks_of = [&](const RowsItem& w) { return C::kSub == 2 && p.P - w.p0 > 128 ? 2 : 1; };
    // length of the sum inside k-block kb
    const auto valid_of = [&](const RowsItem& w, int kb) {
        const int left = (C::kWeight ? w.rend - w.row0 : p.R) - kb * C::kBK;
        return left < C::kBK ? left : C::kBK;
    };
    uint32_t issued = 0, issued_parity = 0;  // producer: loads in flight, for the abort path

    if (threadIdx.x == 0) {
        // ---------------------------------------------------- producer ----
        int stage = 0;
        uint32_t phase = 0;
        bool aborted = false;
        const auto load_p = [&](const RowsItem& w, int kb, int st, int blocks) {
            const uint32_t dst = ring + st * C::kStageBytes, fb = smem_u32(&full[st]);
            for (int h = 0; h < blocks; ++h) {
                const int f = w.p0 + h * 128;
                if constexpr (C::kConv) {
                    tma_load_3d(dst + C::kSub * C::kRawBytes + h * C::kRawBytes, &tmP, fb, f, w.row0 + kb * C::kBK, 0);
                } else if constexpr (C::kPMn) {
                    const int r = C::kWeight ? w.row0 + kb * C::kBK : kb * C::kBK;
                    const int z = C::kWeight ? 0 : w.e;
                    tma_load_3d(dst + h * C::kSubBytes, &tmP, fb, f, r, z);
                    tma_load_3d(dst + h * C::kSubBytes + 8192, &tmP, fb, f + 64, r, z);
                } else {
                    tma_load_3d(dst + h * C::kSubBytes, &tmP, fb, kb * C::kBK, f, w.e);
                }
            }
        };
        const auto load_q = [&](const RowsItem& w, int kb, int st, int boxes) {
            const uint32_t dst = ring + st * C::kStageBytes + C::kPBytes, fb = smem_u32(&full[st]);
            for (int b = 0; b < boxes; ++b) {
                if constexpr (C::kQMn)
                    tma_load_3d(dst + b * C::kQBoxBytes, &tmQ, fb, w.q0 + b * 64, w.row0 + kb * C::kBK, 0);
                else
                    tma_load_3d(dst + b * C::kQBoxBytes, &tmQ, fb, kb * C::kBK, w.row0 + b * C::kQBox, 0);
            }
        };
        bool waited = !p.early;
        for (int item = first; item < total && !aborted; item += stride) {
            const RowsItem w = rows_item<C>(p, item, total, bound, cum);
            int kb0, kb1;
            share(w, kb0, kb1);
            const int blocks = blocks_of(w);
            const int boxes = (w.cnt + C::kQBox - 1) / C::kQBox;
            const uint32_t tx = static_cast<uint32_t>(blocks * (C::kConv ? C::kRawBytes : C::kSubBytes) +
                                                      boxes * C::kQBoxBytes);
            int kb = kb0;
            if (!waited) {
                // the first ring-full: features now, rows once the kernel before has finished
                const int ahead = kb1 - kb0 < C::kStages ? kb1 - kb0 : C::kStages;
                for (int i = 0; i < ahead; ++i) {
                    mbar_arrive_expect_tx(smem_u32(&full[i]), tx);
                    load_p(w, kb0 + i, i, blocks);
                }
                grid_dependency_wait();
                waited = true;
                for (int i = 0; i < ahead; ++i) {
                    load_q(w, kb0 + i, i, boxes);
                    issued |= 1u << i;
                }
                kb += ahead;
                stage = ahead;
                if (stage == C::kStages) stage = 0, phase = 1u;
            }
            for (; kb < kb1; ++kb) {
                if (!wait_bounded(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.timeout_ns,
                                  (blockIdx.x << 8) | 0x10u | stage)) {
                    aborted = true;
                    break;
                }
                mbar_arrive_expect_tx(smem_u32(&full[stage]), tx);
                load_p(w, kb, stage, blocks);
                load_q(w, kb, stage, boxes);
                issued |= 1u << stage;
                issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                if (++stage == C::kStages) stage = 0, phase ^= 1u;
            }
        }
        if (!waited) grid_dependency_wait();
        // Tail: every stage filled has been released, so no MMA commit arrives
        // on this CTA's barriers after it exits.
        for (int i = 0; i < C::kStages && !aborted; ++i) {
            if (!wait_bounded(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.timeout_ns,
                              (blockIdx.x << 8) | 0x50u | stage))
                break;
            if (++stage == C::kStages) stage = 0, phase ^= 1u;
        }
    } else if (warp == 1) {
        // -------------------------------------------------- MMA issuer ----
        int stage = 0;
        uint32_t phase = 0;
        uint32_t acc_phase = 0;
        bool aborted = false;
        for (int item = first; item < total && !aborted; item += stride) {
            const RowsItem w = rows_item<C>(p, item, total, bound, cum);
            int kb0, kb1;
            share(w, kb0, kb1);
            if (kb0 == kb1) continue;  // nothing to sum: the epilogue writes zeros
            const int blocks = blocks_of(w);
            // columns of the MMA: the tile's rows rounded up to what the instruction takes
            const int n = w.cnt <= 16 ? 16 : (w.cnt + 31) & ~31;
            const uint32_t idesc = p.idesc | (static_cast<uint32_t>(n >> 3) << 17);
            for (int h = 0; h < C::kSub; ++h)
                if (!wait_bounded_warp(smem_u32(&tempty[h]), acc_phase ^ 1u, abort_flag, p.timeout_ns,
                                       (blockIdx.x << 8) | 0x20u | h)) {
                    aborted = true;
                    break;
                }
            if (aborted) break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_bounded_warp(smem_u32(&full[stage]), phase, abort_flag, p.timeout_ns,
                                       (blockIdx.x << 8) | 0x30u | stage)) {
                    aborted = true;
                    break;
                }
                if (C::kConv && !wait_bounded_warp(smem_u32(&conv[stage]), phase, abort_flag, p.timeout_ns,
                                                   (blockIdx.x << 8) | 0x38u | stage)) {
                    aborted = true;
                    break;
                }
                const int valid = valid_of(w, kb);
                const int ksteps = (valid + C::kUmmaK - 1) / C::kUmmaK;
                uint8_t* st = smem + stage * C::kStageBytes;
                if (C::kWeight && (valid & 15)) {
                    // The sum ends inside an MMA step: the step's remaining
                    // rows belong to the next group and are overwritten with
                    // zeros, in both operands (0 x NaN would not be 0).
                    const int extra = 16 - (valid & 15);
                    const int atoms = (C::kConv ? 0 : 2 * blocks) + (n + 63) / 64;
                    for (int i = lane; i < atoms * extra * 8; i += 32) {
                        const int a = i / (extra * 8), r = valid + (i / 8) % extra;
                        const int pa = C::kConv ? 0 : 2 * blocks;
                        uint8_t* atom = a < pa ? st + a * 8192 : st + C::kPBytes + (a - pa) * 8192;
                        *reinterpret_cast<uint4*>(atom + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t pa = smem_u32(st), qa = pa + C::kPBytes;
                    for (int k = 0; k < ksteps; ++k) {
                        const uint64_t qd = C::kQMn ? smem_desc_sw128(qa + k * C::kUmmaK * 128, 8192, 1024)
                                                    : smem_desc_sw128(qa + k * 32, 16, 1024);
                        for (int h = 0; h < blocks; ++h) {
                            const uint32_t ph = pa + h * C::kSubBytes;
                            const uint64_t pd = C::kPMn ? smem_desc_sw128(ph + k * C::kUmmaK * 128, 8192, 1024)
                                                        : smem_desc_sw128(ph + k * 32, 16, 1024);
                            umma<C::kKind>(tmem_base + h * C::kBQ, pd, qd, idesc, kb > kb0 || k > 0 ? 1u : 0u);
                        }
                    }
                    umma_commit(smem_u32(&empty[stage]));
                }
                __syncwarp();
                if (++stage == C::kStages) stage = 0, phase ^= 1u;
            }
            if (aborted) break;
            if (lane == 0)
                for (int h = 0; h < C::kSub; ++h) umma_commit(smem_u32(&tfull[h]));
            __syncwarp();
            acc_phase ^= 1u;
        }
    } else if (warp >= 2 && warp < 6) {
        // ---------------------------------------------------- epilogue ----
        const int quarter = warp & 3;
        uint32_t acc_phase = 0;
        bool lost = false;
        if (p.early) grid_dependency_wait();  // the rows' scales, and the output's last readers
        for (int item = first; item < total && !lost; item += stride) {
            const RowsItem w = rows_item<C>(p, item, total, bound, cum);
            int kb0, kb1;
            share(w, kb0, kb1);
            const bool empty_sum = kb0 == kb1;
            for (int h = 0; h < C::kSub; ++h) {
                const int f = w.p0 + h * 128 + quarter * 32 + lane;  // this lane's feature
                const bool live = f < p.P;
                if (!empty_sum) {
                    if (!wait_bounded_warp(smem_u32(&tfull[h]), acc_phase, abort_flag, p.timeout_ns,
                                           (blockIdx.x << 8) | 0x40u | h)) {
                        lost = true;
                        break;
                    }
                    tc_fence_after();
                }
                float sp = 0.f, bias = 0.f;
                if (C::kKind == kKindI8 && S == 1 && live && !w.zero) {
                    const long long at = static_cast<long long>(w.e) * p.P + f;
                    sp = p.scale_p[at];
                    if (p.bias_p) bias = p.bias_p[at];
                }
                const long long row = C::kWeight ? static_cast<long long>(w.e) * p.Q + w.q0 : w.row0;
                const uint32_t t_addr =
                    tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(h * C::kBQ);
#pragma unroll 1
                for (int c = 0; c < w.cnt; c += 32) {
                    uint32_t v[32];
                    if (empty_sum) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0u;
                    } else {
                        tmem_ld_32x32b_x32(t_addr + c, v);
                        tmem_ld_wait();
                    }
                    const int n = w.cnt - c < 32 ? w.cnt - c : 32;
                    if (C::kSub == 1 && S > 1) {
                        // this CTA's part of column c + j to the CTA that
                        // finishes that column: [source rank][column][feature]
                        const int per = C::kBQ / S;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (j < n) {
                                const int d = (c + j) / per, cl = (c + j) - d * per;
                                const uint32_t at =
                                    smem_u32(red + (rank * per + cl) * 128 + quarter * 32 + lane);
                                st_cluster_u32(mapa_shared(at, d), v[j]);
                            }
                        }
                        continue;
                    }
                    float sq = 0.f;
                    if (C::kKind == kKindI8 && !w.zero && lane < n) sq = p.scale_q[w.row0 + c + lane];
                    const long long at = (row + c) * p.P + f;
                    if (p.out_type == kOutF32)
                        store_cols<C>(v, static_cast<float*>(p.out) + at, p.P, n, live, sp, bias, sq);
                    else if (p.out_type == kOutF16)
                        store_cols<C>(v, static_cast<__half*>(p.out) + at, p.P, n, live, sp, bias, sq);
                    else
                        store_cols<C>(v, static_cast<__nv_bfloat16*>(p.out) + at, p.P, n, live, sp, bias, sq);
                }
                if (!empty_sum) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&tempty[h]));
                }
            }
            if (!empty_sum) acc_phase ^= 1u;
        }
    } else if (C::kConv && warp >= 6) {
        // -------------------------------------------------- converters ----
        // Every wait's outcome goes through a barrier-AND of the converter
        // warps, so they give up together.
        const int ct = static_cast<int>(threadIdx.x) - 192;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int item = first; item < total && ok; item += stride) {
            const RowsItem w = rows_item<C>(p, item, total, bound, cum);
            int kb0, kb1;
            share(w, kb0, kb1);
            for (int kb = kb0; kb < kb1; ++kb) {
                ConvRegs<C> g;
                const int valid = valid_of(w, kb);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = u * 32 + (ct >> 3);
                    const float s = r < valid ? p.scale_r[w.row0 + kb * C::kBK + r] : 0.f;
#pragma unroll
                    for (int b = 0; b < C::kSub; ++b) g.s[2 * b + u] = s;
                }
                const bool landed = wait_bounded_warp(smem_u32(&full[stage]), phase, abort_flag, p.timeout_ns,
                                                      (blockIdx.x << 8) | 0xA0u | stage);
                uint8_t* st = smem + stage * C::kStageBytes;
                if (landed) conv_codes<C>(st + C::kSub * C::kRawBytes, ct, g);
                ok = named_barrier_and(1, 32 * C::kConvWarps, landed);
                if (!ok) break;
                if (p.bf16)
                    conv_write<C, true>(st, ct, valid, g);
                else
                    conv_write<C, false>(st, ct, valid, g);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&conv[stage]));
                if (++stage == C::kStages) stage = 0, phase ^= 1u;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // Some role gave up.  Before shared and tensor memory are released,
        // let this CTA's own copies land and its MMAs retire.
        if (threadIdx.x == 0)
            for (int s = 0; s < C::kStages; ++s)
                if (issued & (1u << s)) drain_wait(smem_u32(&full[s]), (issued_parity >> s) & 1u);
        if (threadIdx.x == 32) {
            umma_commit(smem_u32(drain));
            drain_wait(smem_u32(drain), 0);
        }
        __syncwarp();
        __syncthreads();
    }
    if (C::kSub == 1 && S > 1) {
        cluster_sync_all();  // every part has arrived
        if (first < total && !*abort_flag) {
            // this CTA's columns of the tile: the parts in rank order
            const RowsItem w = rows_item<C>(p, first, total, bound, cum);
            const int per = C::kBQ / S;
            const int f = w.p0 + (static_cast<int>(threadIdx.x) & 127);
            if (threadIdx.x < 128 && f < p.P) {
                float sp = 0.f, bias = 0.f;
                if (C::kKind == kKindI8 && !w.zero) {
                    const long long at = static_cast<long long>(w.e) * p.P + f;
                    sp = p.scale_p[at];
                    if (p.bias_p) bias = p.bias_p[at];
                }
                if (p.early) grid_dependency_wait();
                const long long row0 = C::kWeight ? static_cast<long long>(w.e) * p.Q + w.q0 : w.row0;
                for (int cl = 0; cl < per; ++cl) {
                    const int c = rank * per + cl;
                    if (c >= w.cnt) break;
                    float x;
                    if constexpr (C::kKind == kKindI8) {
                        int sum = 0;
                        for (int s = 0; s < S; ++s)
                            sum += static_cast<int>(red[(s * per + cl) * 128 + threadIdx.x]);
                        const float sq = w.zero ? 0.f : p.scale_q[w.row0 + c];
                        x = fmaf(__int2float_rn(sum) * sq, sp, bias);
                    } else {
                        x = 0.f;
                        for (int s = 0; s < S; ++s)
                            x += __uint_as_float(red[(s * per + cl) * 128 + threadIdx.x]);
                    }
                    const long long at = (row0 + c) * p.P + f;
                    if (p.out_type == kOutF32)
                        static_cast<float*>(p.out)[at] = x;
                    else if (p.out_type == kOutF16)
                        static_cast<__half*>(p.out)[at] = __float2half_rn(x);
                    else
                        static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
                }
            }
        }
    }
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
}

}  // namespace tcg
