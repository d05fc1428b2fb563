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
//   kSub = 1: 128 features x kBQ rows, one tile per cluster, for few rows, where
//     the weights' bytes bound the product and every SM has to pull on memory.
//     The CTAs of a cluster (1, 2, 4 or 8) split the sum between them and add
//     their parts through distributed shared memory, in rank order (the result
//     does not depend on timing).  fp32 results are summed in chunks of 128 to
//     512: the tensor cores drop the bits that do not fit when they add to an
//     accumulator, an error that grows with the length of the chain (rms of the
//     result's: 2.5e-6 at K = 2048, an fp32 product 0.8e-6; 0.65e-6 in chunks of
//     512, 0.34e-6 of 256, 0.19e-6 of 128, added with one rounding each).
//   kSub = 2: 256 x 256, two M = 128 accumulators that fill the tensor memory,
//     for many rows, where the tensor cores bound the product.  Persistent CTAs
//     take every so manieth tile; or, where the number of tiles is known at
//     launch and tiles are long, there is a CTA per tile and running CTAs take
//     over those that have not started (cluster launch control).
//
// Warps: 0 TMA producer, 1 MMA issuer, 2..9 epilogue (two per tensor-memory lane
// quarter).  Every wait on an mbarrier is bounded (tcg_wait.cuh).
//
// What bounds it (B200): few rows, start and exchange, then the weights' bytes
// (eight rows of 4096 x 4096 int8, quantising included, 8.5 us where the bytes are
// 2.6; experts' weights of 64 x 2048 x 4096 int8 at 6.0 TB/s of 6.5); many rows,
// the tensor cores, under the power limit after some ms: int8 16384 x 8192 x 8192
// 714 us (3.08 POPS), 820 sustained; bf16 8192 x 8192 x 4096 366 us (1.50 PFLOP/s),
// 422 sustained (the library's product 350 and 406).
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
    unsigned long long timeout_ns;
    int groups, rows, rows_per_group;
    int P, Q, R;              // features out; weight form: the other features; rows form: length of the sum
    int ptiles, qtiles;       // tiles along P; weight form: along Q
    int band_log2;            // kSub = 2: tiles along q per rasterisation band
    uint32_t per_band_inv, ptiles_inv, per_group_inv;  // div_by: band * ptiles, ptiles, tiles per group
    int zero_rest;            // rows form: write zeros into rows outside every group
    int aligned_out;          // output rows are whole 16-byte vectors, 16-byte aligned
    int out_type;
    int split_log2;           // kSub = 1: 1, 2, 4 or 8 CTAs per tile
    int stages;               // ring depth
    int chunk;                // kChunks: k-blocks that the tensor cores add up in one go
    int p_whole, q_whole;     // MN-major operands of whole 64-element atoms: one copy a tile and stage
    int dynamic;              // kSub = 2: a CTA per item, running ones taking over those not started
    int early;                // the M-side operand and the offsets predate the kernel this one follows
    uint32_t idesc;           // instruction descriptor without N
};

template <int kKind_, bool kPMn_, bool kQMn_, int kSub_, int kBQ_>
struct RowsTraits {
    static constexpr int kKind = kKind_;
    static constexpr bool kPMn = kPMn_, kQMn = kQMn_;
    static constexpr int kSub = kSub_, kBQ = kBQ_;
    static constexpr bool kWeight = kQMn;               // weight form: the sum runs over a group's rows
    // kSub = 2: each group of epilogue warps takes one block, whole, so that its
    // reads of the accumulator overlap the other's stores.  Pays where stores are
    // most of a tile, in the gradients (16 groups, 300 rows x 2048 x 2048 59.5 ->
    // 49.2 us, 16384 x 4096 x 2048 224 -> 217); both groups on each block free it
    // sooner, which the rows form prefers (int8 8192 x 4096 x 512 58 against 66).
    static constexpr bool kOwnBlock = kWeight && kSub_ == 2;
    static constexpr int kElem = kKind == kKindF16 ? 2 : 1;
    static constexpr int kBK = 128 / kElem;             // length of the sum per ring stage
    static constexpr int kUmmaK = 32 / kElem;
    static constexpr int kTileP = 128 * kSub;
    static constexpr int kSubBytes = 128 * kBK * kElem; // one 128-feature block of a stage
    static constexpr int kPBytes = kSub * kSubBytes;
    static constexpr int kQBytes = kBQ * kBK * kElem;
    static constexpr int kStageBytes = kPBytes + kQBytes;
    static constexpr int kAtomBytes = 128 * kBK;        // MN-major: 64 elements of kBK rows
    static constexpr int kQBox = kBQ < 64 ? kBQ : 64;   // rows (weight form: columns) per box of the q operand
    static constexpr int kQBoxBytes = kQBox * kBK * kElem;
    static constexpr int kEpiWarps = 8;                 // two per quarter of the tensor memory's lanes
    static constexpr int kThreads = 32 * (2 + kEpiWarps);
    static constexpr int kPerSm = kSub == 1 ? 2 : 1;  // CTAs per SM that registers are kept for
    // kSub = 1 with fp32 sums: two accumulators that take chunks of the sum in turn
    static constexpr bool kChunks = kSub == 1 && kKind == kKindF16;
    static constexpr int kTmemCols = kChunks ? (kBQ < 32 ? 64 : 2 * kBQ) : (kSub * kBQ < 32 ? 32 : kSub * kBQ);
    static constexpr int kRedBytes = kBQ * 512;         // split: 128 x kBQ partial sums
    static constexpr int kMaxStages = 12;
    static constexpr int kRing = 4;                     // kSub = 2: items on their way to the other roles
    static constexpr int kBarBytes = 384;
    static constexpr int kScaleBytes = 1024;            // scales of the rows being written out
    // two blocks of 32 x 128 results on their way out; one tile a CTA: in the ring, which is idle by then
    static constexpr int kOutBytes = 8192;
    static constexpr int kOutArea = kSub == 2 ? 2 * kOutBytes : 0;
    static_assert(!kQMn || kKind == kKindF16, "weight form: 16-bit operands");
    static_assert(!kPMn || kKind == kKindF16, "MN-major features: 16-bit operands");
    static_assert(!kQMn || kBQ % 64 == 0, "whole 64-column atoms");
    static_assert(8 * (2 * kMaxStages + 6 + 2 * kRing) + 8 + 4 * kRing + 16 <= kBarBytes - 16, "barrier area");
    static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols <= 512, "TMEM allocation");
    // the epilogue reads 32 columns at a time, from the start of the last accumulator too
    static_assert((kChunks || kSub == 2 ? kBQ : 0) + (kBQ < 32 ? 32 : kBQ) <= kTmemCols, "reads inside the allocation");
    // dynamic shared memory of a launch with a table of `groups` groups
    static constexpr int smem_bytes(int stages, int split, int groups)
    {
        return 1024 + stages * kStageBytes + kOutArea + (split > 1 ? kRedBytes : 0) + kScaleBytes + kBarBytes +
               8 * (groups + 3);
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

// a / d for 0 <= a < 2^31 with inv = div_inverse(d): the product with the
// rounded-up reciprocal is at most one too large.
__host__ __device__ constexpr uint32_t div_inverse(uint32_t d)
{
    return d <= 1 ? 0u : static_cast<uint32_t>((0x100000000ull + d - 1) / d);
}
__device__ __forceinline__ int div_by(int a, int d, uint32_t inv)
{
    if (d <= 1) return a;
    int q = static_cast<int>(__umulhi(static_cast<uint32_t>(a), inv));
    if (q * d > a) --q;
    return q;
}

// Tiles along q (weight form: of every group together).
template <class C>
__device__ __forceinline__ int rows_qtiles(const RowsParams& p, const int* cum)
{
    if (C::kWeight) return p.groups * p.qtiles;
    return p.offsets ? cum[p.groups + 2] : p.groups * p.qtiles;
}

// The tile at p-tile pt and q-tile tq (weight form: tq of group e).
template <class C>
__device__ __forceinline__ RowsItem rows_tile(const RowsParams& p, int pt, int tq, int e, const int* bound,
                                              const int* cum)
{
    RowsItem w;
    w.zero = false;
    w.p0 = pt * C::kTileP;
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
        w.e = div_by(tq, p.qtiles, p.per_group_inv);
        w.row0 = w.e * p.rows_per_group + (tq - w.e * p.qtiles) * C::kBQ;
        w.rend = (w.e + 1) * p.rows_per_group;
    }
    w.cnt = min(C::kBQ, w.rend - w.row0);
    w.nkb = w.zero ? 0 : (p.R + C::kBK - 1) / C::kBK;
    return w;
}

// The same tile with every field broadcast, so that the compiler knows what
// the producer and the MMA issuer compute from it to be uniform.
__device__ __forceinline__ RowsItem uniform(RowsItem w)
{
    const unsigned all = 0xffffffffu;
    w.e = __shfl_sync(all, w.e, 0);
    w.row0 = __shfl_sync(all, w.row0, 0);
    w.cnt = __shfl_sync(all, w.cnt, 0);
    w.p0 = __shfl_sync(all, w.p0, 0);
    w.q0 = __shfl_sync(all, w.q0, 0);
    w.nkb = __shfl_sync(all, w.nkb, 0);
    w.rend = __shfl_sync(all, w.rend, 0);
    return w;
}

// Work item of a persistent CTA (kSub = 2) -> tile.  Items walk a band of
// 2^band_log2 q-tiles for all of P before the next band, so the tiles in
// flight share both operands in L2; a last, narrower band goes row by row.
template <class C>
__device__ __forceinline__ RowsItem rows_item(const RowsParams& p, int item, int qtiles, const int* bound,
                                              const int* cum)
{
    int e = 0;
    if (C::kWeight) {
        const int per = p.ptiles * p.qtiles;
        e = div_by(item, per, p.per_group_inv);
        item -= e * per;
        qtiles = p.qtiles;
    }
    const int per_band = p.ptiles << p.band_log2;
    const int b = div_by(item, per_band, p.per_band_inv);
    const int r = item - b * per_band;
    int tq = b << p.band_log2, pt;
    if (tq + (1 << p.band_log2) <= qtiles) {
        tq += r & ((1 << p.band_log2) - 1);
        pt = r >> p.band_log2;
    } else {
        const int j = div_by(r, p.ptiles, p.ptiles_inv);
        tq += j;
        pt = r - j * p.ptiles;
    }
    return rows_tile<C>(p, pt, tq, e, bound, cum);
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

// Results of 32 columns (rows of the output) x 128 features, held by the four
// warps of one epilogue group as one feature a lane, out to memory with whole
// 128-byte lines a warp: through 8 KB of shared memory, 16 x 128 words at a
// time -- for 16-bit results a word is one feature of two rows.  (Straight from
// the registers a warp's store is 64 bytes of one row.  With whole lines and
// the accumulators freed early, see below: bf16 8192 x 8192 x 4096 394 -> 368 us,
// weight gradients of 16 groups of 1024 rows, 4096 x 2048, 257 -> 228.)
struct OutBlock {
    void* out;
    long long row;   // first row
    int ld;          // elements
    int f;           // first feature of the block
    int n;           // rows of the block that exist
    int features;    // features of the block that exist (<= 128)
    bool aligned;    // rows are whole 16-byte vectors, 16-byte aligned
};

__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// two rows' values of one feature per word, each rounded once
__device__ __forceinline__ void pack_block(const float (&x)[32], bool bf16, uint32_t (&w)[16])
{
    if (bf16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack16<true>(x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack16<false>(x[2 * j], x[2 * j + 1]);
    }
}

__device__ __forceinline__ void store_block16(const uint32_t (&w)[16], const OutBlock& o, uint32_t* stage, int quarter,
                                              int lane, int barrier)
{
#pragma unroll
    for (int j = 0; j < 16; ++j) stage[j * 128 + quarter * 32 + lane] = w[j];
    group_sync(barrier);
    unsigned short* out = static_cast<unsigned short*>(o.out) + o.row * o.ld + o.f;
    const int e = (lane & 15) * 8;  // 16 lanes a row pair, eight features a lane
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int pair = quarter * 4 + i * 2 + (lane >> 4);
        const uint4 a = *reinterpret_cast<const uint4*>(stage + pair * 128 + e);
        const uint4 b = *reinterpret_cast<const uint4*>(stage + pair * 128 + e + 4);
        unsigned short* row = out + static_cast<long long>(2 * pair) * o.ld + e;
        if (e < o.features && 2 * pair < o.n)
            *reinterpret_cast<uint4*>(row) =
                make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410),
                           __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
        if (e < o.features && 2 * pair + 1 < o.n)
            *reinterpret_cast<uint4*>(row + o.ld) =
                make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632),
                           __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
    }
    group_sync(barrier);
}

// Rows that are not whole 16-byte vectors: straight from the registers, 64
// bytes of a row per warp and store.  (Putting rows of odd length together
// from aligned words in shared memory measured slower: int8 1777 x 4099 x 4096
// 38 against 29 us.)
__device__ __forceinline__ void store_rows16(const uint32_t (&w)[16], const OutBlock& o, int quarter, int lane)
{
    const int e = quarter * 32 + lane;
    const bool live = e < o.features;
    unsigned short* ptr = static_cast<unsigned short*>(o.out) + o.row * o.ld + o.f + e;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        if (2 * j < o.n && live) ptr[0] = static_cast<unsigned short>(w[j]);
        if (2 * j + 1 < o.n && live) ptr[o.ld] = static_cast<unsigned short>(w[j] >> 16);
        ptr += 2 * static_cast<long long>(o.ld);
    }
}

__device__ __forceinline__ void store_block32(const float (&x)[32], const OutBlock& o, uint32_t* stage, int quarter,
                                              int lane, int barrier)
{
    float* out = static_cast<float*>(o.out) + o.row * o.ld + o.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < 16; ++j) stage[j * 128 + quarter * 32 + lane] = __float_as_uint(x[16 * half + j]);
        group_sync(barrier);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = quarter * 4 + i;
            float* row = out + static_cast<long long>(16 * half + r) * o.ld;
            if (16 * half + r >= o.n) continue;
            if (o.aligned) {
                if (lane * 4 < o.features)
                    *reinterpret_cast<uint4*>(row + lane * 4) =
                        *reinterpret_cast<const uint4*>(stage + r * 128 + lane * 4);
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (lane + 32 * u < o.features) row[lane + 32 * u] = __uint_as_float(stage[r * 128 + lane + 32 * u]);
            }
        }
        group_sync(barrier);
    }
}

// Split sums.  Columns c .. c + n - 1 of this CTA's part (one lane = feature
// f) to the CTAs that finish them: CTA d finishes columns d * kBQ / S onwards.
// There the parts lie as [source rank][group of V columns][feature][V], V = 4
// (2 for two columns a CTA): one 16-byte store per four columns and lane, and
// a warp's stores are contiguous.
template <class C>
__device__ __forceinline__ void push_part(const uint32_t (&v)[32], uint32_t* red, int rank, int split_log2, int c,
                                          int n, int f)
{
    const int per = C::kBQ >> split_log2;
    const int per_log2 = 31 - __clz(per);
#pragma unroll
    for (int j = 0; j < (C::kBQ < 32 ? C::kBQ : 32); j += 4) {
        if (j >= n) break;
        const int d = (c + j) >> per_log2, cl = (c + j) & (per - 1);
        if (per >= 4) {
            const uint32_t at = smem_u32(red + (rank * per + cl) * 128 + f * 4);
            st_cluster_v4(mapa_shared(at, d), v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else {
            const uint32_t at = smem_u32(red + rank * 256 + f * 2);
            st_cluster_v2(mapa_shared(at, d), v[j], v[j + 1]);
            st_cluster_v2(mapa_shared(at, d + 1), v[j + 2], v[j + 3]);
        }
    }
}

// This CTA's columns of the tile: the parts added in rank order, scaled, and
// stored; two threads per feature f, V columns at a time in turn (g).
template <class C, int V, class T>
__device__ __forceinline__ void finish_parts(const RowsParams& p, const RowsItem& w, const uint32_t* red,
                                             const float* scale, int rank, int f, int g, float sp, float bias)
{
    const int S = 1 << p.split_log2;
    const int per = C::kBQ >> p.split_log2;
    const bool live = w.p0 + f < p.P;
    const long long row0 = (C::kWeight ? static_cast<long long>(w.e) * p.Q + w.q0 : w.row0) + rank * per;
    const int n = min(per, w.cnt - rank * per);
    T* ptr = static_cast<T*>(p.out) + (row0 + g * V) * p.P + w.p0 + f;
    const uint32_t* part = red + f * V;
#pragma unroll 2
    for (int cl = g * V; cl < n; cl += 2 * V) {
        float x[V];
        if constexpr (C::kKind == kKindI8) {
            int sum[V] = {};
#pragma unroll 2
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += static_cast<int>(part[(s * per + cl) * 128 + i]);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = fmaf(__int2float_rn(sum[i]) * scale[cl + i], sp, bias);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = 0.f;
#pragma unroll 2
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] += __uint_as_float(part[(s * per + cl) * 128 + i]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (cl + i < n && live) *ptr = T(x[i]);
            ptr += p.P;
        }
        ptr += static_cast<long long>(V) * p.P;
    }
}

template <class C, class T>
__device__ __forceinline__ void finish(const RowsParams& p, const RowsItem& w, const uint32_t* red, const float* scale,
                                       int rank, int t, float sp, float bias)
{
    if ((C::kBQ >> p.split_log2) >= 4)
        finish_parts<C, 4, T>(p, w, red, scale, rank, t & 127, t >> 7, sp, bias);
    else
        finish_parts<C, 2, T>(p, w, red, scale, rank, t & 127, t >> 7, sp, bias);
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, C::kPerSm)
    rows_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                const __grid_constant__ CUtensorMap tmQb, const __grid_constant__ RowsParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const int S = C::kSub == 1 ? 1 << p.split_log2 : 1;
    const int stages = p.stages;
    uint8_t* out_area = C::kSub == 2 ? smem + stages * C::kStageBytes : smem;
    uint32_t* red = reinterpret_cast<uint32_t*>(smem + stages * C::kStageBytes + C::kOutArea);
    float* scales = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(red) + (S > 1 ? C::kRedBytes : 0));
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(scales) + C::kScaleBytes);
    uint64_t* empty = full + C::kMaxStages;
    uint64_t* tfull = empty + C::kMaxStages;  // accumulator block h complete
    uint64_t* tempty = tfull + 2;            // accumulator block h read
    uint64_t* drain = tempty + 2;
    uint64_t* qfull = drain + 1;             // item published
    uint64_t* qempty = qfull + C::kRing;     // item read by the MMA issuer and every epilogue warp
    uint64_t* clcbar = qempty + C::kRing;    // cluster launch control has answered
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(clcbar + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    volatile int* ring_item = reinterpret_cast<volatile int*>(tmem_slot + 2);
    const uint32_t clc_answer = smem_u32(reinterpret_cast<uint8_t*>(full) + C::kBarBytes - 16);  // 16-byte aligned
    int* bound = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + C::kBarBytes);
    int* cum = bound + p.groups + 3;  // (used, and room for it, with offsets only)

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // (uniform to the compiler)
    const int lane = threadIdx.x & 31;
    const int rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;

    if (warp == 0) {
        // one stage's barriers a lane; then the others
        if (lane < stages) {
            mbar_init(smem_u32(&full[lane]), 1);
            mbar_init(smem_u32(&empty[lane]), 1);
        } else if (lane >= 16 && lane < 18) {
            mbar_init(smem_u32(&tfull[lane - 16]), 1);
            mbar_init(smem_u32(&tempty[lane - 16]), C::kOwnBlock ? C::kEpiWarps / 2 : C::kEpiWarps);
        } else if (lane == 18) {
            mbar_init(smem_u32(drain), 1);
            mbar_init(smem_u32(clcbar), 1);
            *abort_flag = 0u;
        } else if (lane >= 24 && lane < 24 + C::kRing) {
            mbar_init(smem_u32(&qfull[lane - 24]), 1);
            mbar_init(smem_u32(&qempty[lane - 24]), 1 + C::kEpiWarps);
        } else if (lane == 19) {
            tma_prefetch_desc(&tmP);
        } else if (lane == 20) {
            tma_prefetch_desc(&tmQ);
        } else if (lane == 21) {
            tma_prefetch_desc(&tmQb);
        }
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    // Everything above overlaps the previous kernel's tail.  With `early` the
    // kernel before this one wrote only the q operand and its scales, and let
    // this one start after its own wait: features and offsets may be read now.
    if (!p.early) grid_dependency_wait();
    // (by the warp that allocates: the next kernel's CTAs take what tensor memory
    // is left only once every CTA here has its own, so neither waits for the other)
    if (warp == 1) grid_launch_dependents();
    if (p.offsets && warp == 2) rows_table(p, C::kBQ, bound, cum);
    tc_fence_before();
    __syncthreads();
    if (S > 1) cluster_arrive();  // every CTA of the cluster runs before any writes into another (push_part)
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t ring = smem_u32(smem);

    // kSub = 1: one tile a CTA, by its place in the grid (x: q-tile and rank, y:
    // p-tile, z: group of the weight form); kSub = 2: items from here on.
    const int qtiles = rows_qtiles<C>(p, cum);
    const int tq1 = static_cast<int>(blockIdx.x) >> p.split_log2;
    const int first = C::kSub == 1 ? 0 : static_cast<int>(blockIdx.x);
    const int stride = C::kSub == 1 ? 1 : static_cast<int>(gridDim.x);
    const int total = C::kSub == 1 ? ((C::kWeight ? p.qtiles : qtiles) > tq1 ? 1 : 0) : qtiles * p.ptiles;
    const auto tile_of = [&](int item) {
        if constexpr (C::kSub == 1)
            return rows_tile<C>(p, static_cast<int>(blockIdx.y), tq1, static_cast<int>(blockIdx.z), bound, cum);
        else
            return rows_item<C>(p, item, qtiles, bound, cum);
    };
    // Items reach the MMA issuer and the epilogue like this.  Static: every
    // stride-th item.  Dynamic: whatever the producer has published (-1 at the
    // end; a wait that gave up ends the role too).
    const bool dynamic = C::kSub == 2 && p.dynamic;
    int q = 0;
    uint32_t qph = 0;
    const auto next_item = [&](int item) {
        if (!dynamic) {
            item = item < 0 ? first : item + stride;
            return item < total ? item : -1;
        }
        if (!wait_bounded_warp(smem_u32(&qfull[q]), qph, abort_flag, p.timeout_ns, (blockIdx.x << 8) | 0x70u | q))
            return -1;
        item = ring_item[q];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&qempty[q]));
        if (++q == C::kRing) q = 0, qph ^= 1u;
        return item;
    };
    // this CTA's share [kb0, kb1) of a tile's k-blocks
    const auto share = [&](const RowsItem& w, int& kb0, int& kb1) {
        kb0 = C::kSub == 1 ? (w.nkb * rank) >> p.split_log2 : 0;
        kb1 = C::kSub == 1 ? (w.nkb * (rank + 1)) >> p.split_log2 : w.nkb;
    };
    const auto blocks_of = [&](const RowsItem& w) { return C::kSub == 2 && p.P - w.p0 > 128 ? 2 : 1; };
    // length of the sum inside k-block kb
    const auto valid_of = [&](const RowsItem& w, int kb) {
        const int left = (C::kWeight ? w.rend - w.row0 : p.R) - kb * C::kBK;
        return left < C::kBK ? left : C::kBK;
    };
    uint32_t issued = 0, issued_parity = 0;  // producer: loads in flight, for the abort path

    if (warp == 0) {
        // ---------------------------------------------------- producer ----
        int stage = 0;
        uint32_t phase = 0;
        bool aborted = false;
        // One copy per operand and stage wherever the layout allows.
        const auto load_p = [&](const RowsItem& w, int kb, int st, int blocks) {
            const uint32_t dst = ring + st * C::kStageBytes, fb = smem_u32(&full[st]);
            if constexpr (C::kPMn) {
                const int r = C::kWeight ? w.row0 + kb * C::kBK : kb * C::kBK;
                const int z = C::kWeight ? 0 : w.e;
                if (p.p_whole)
                    tma_load_4d(dst, &tmP, fb, 0, r, w.p0 / 64, z);
                else
                    for (int a = 0; a < 2 * blocks; ++a)
                        tma_load_4d(dst + a * C::kAtomBytes, &tmP, fb, w.p0 + a * 64, r, 0, z);
            } else {
                tma_load_4d(dst, &tmP, fb, kb * C::kBK, w.p0, 0, w.e);
            }
        };
        const auto load_q = [&](const RowsItem& w, int kb, int st, int boxes) {
            const uint32_t dst = ring + st * C::kStageBytes + C::kPBytes, fb = smem_u32(&full[st]);
            if constexpr (C::kQMn) {
                if (p.q_whole)
                    tma_load_4d(dst, &tmQ, fb, 0, w.row0 + kb * C::kBK, w.q0 / 64, 0);
                else
                    for (int b = 0; b < boxes; ++b)
                        tma_load_4d(dst + b * C::kAtomBytes, &tmQ, fb, w.q0 + b * 64, w.row0 + kb * C::kBK, 0, 0);
            } else {
                if (boxes * C::kQBox == C::kBQ)
                    tma_load_4d(dst, &tmQ, fb, kb * C::kBK, w.row0, 0, 0);
                else
                    for (int b = 0; b < boxes; ++b)
                        tma_load_4d(dst + b * C::kQBoxBytes, &tmQb, fb, kb * C::kBK, w.row0 + b * C::kQBox, 0, 0);
            }
        };
        bool waited = !p.early;
        bool asked = false;  // an answer of cluster launch control is on its way
        uint32_t clc_phase = 0;
        // The item after `item` (-1: none).  Dynamic: publish that one and ask
        // for the CTA to take over; the answer is read after its loads.
        const auto publish = [&](int item) {
            if (!wait_bounded_warp(smem_u32(&qempty[q]), qph ^ 1u, abort_flag, p.timeout_ns,
                                   (blockIdx.x << 8) | 0x78u | q))
                return false;
            if (elect_one()) {
                ring_item[q] = item;
                mbar_arrive(smem_u32(&qfull[q]));
            }
            __syncwarp();
            if (++q == C::kRing) q = 0, qph ^= 1u;
            return true;
        };
        for (int item = first < total ? first : -1; !aborted;) {
            if (dynamic && !publish(item)) {
                aborted = true;
                break;
            }
            if (item < 0) break;
            if (dynamic) {
                if (elect_one()) {
                    mbar_arrive_expect_tx(smem_u32(clcbar), 16);
                    clc_try_cancel(clc_answer, smem_u32(clcbar));
                }
                __syncwarp();
                asked = true;
            }
            const RowsItem w = uniform(tile_of(item));
            int kb0, kb1;
            share(w, kb0, kb1);
            const int blocks = blocks_of(w);
            const int boxes = (w.cnt + C::kQBox - 1) / C::kQBox;
            const int p_bytes = C::kPMn && !p.p_whole ? blocks * C::kSubBytes : C::kPBytes;
            const int q_bytes = C::kQMn && p.q_whole ? C::kQBytes : boxes * C::kQBoxBytes;
            const uint32_t tx = static_cast<uint32_t>(p_bytes + q_bytes);
            int kb = kb0;
            if (!waited) {
                // the first ring-full: features now, rows once the kernel before has finished
                const int ahead = kb1 - kb0 < stages ? kb1 - kb0 : stages;
                if (elect_one())
                    for (int i = 0; i < ahead; ++i) {
                        mbar_arrive_expect_tx(smem_u32(&full[i]), tx);
                        load_p(w, kb0 + i, i, blocks);
                    }
                __syncwarp();
                grid_dependency_wait();
                waited = true;
                if (elect_one())
                    for (int i = 0; i < ahead; ++i) load_q(w, kb0 + i, i, boxes);
                __syncwarp();
                issued = (1u << ahead) - 1u;
                kb += ahead;
                stage = ahead;
                if (stage == stages) stage = 0, phase = 1u;
            }
            for (; kb < kb1; ++kb) {
                if (!wait_bounded_warp(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.timeout_ns,
                                       (blockIdx.x << 8) | 0x10u | stage)) {
                    aborted = true;
                    break;
                }
                if (elect_one()) {
                    mbar_arrive_expect_tx(smem_u32(&full[stage]), tx);
                    load_p(w, kb, stage, blocks);
                    load_q(w, kb, stage, boxes);
                }
                __syncwarp();
                issued |= 1u << stage;
                issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                if (++stage == stages) stage = 0, phase ^= 1u;
            }
            if (aborted) break;
            if (dynamic) {
                if (!wait_bounded_warp(smem_u32(clcbar), clc_phase, abort_flag, p.timeout_ns,
                                       (blockIdx.x << 8) | 0x7Cu)) {
                    aborted = true;
                    break;
                }
                asked = false;
                clc_phase ^= 1u;
                int taken = -1;
                item = clc_query(clc_answer, taken) ? taken : -1;
            } else {
                item = item + stride < total ? item + stride : -1;
            }
        }
        if (asked) drain_wait(smem_u32(clcbar), clc_phase);  // (aborting: the answer lands in this CTA's memory)
        if (!waited) grid_dependency_wait();
        // Tail: every stage filled has been released, so no MMA commit arrives
        // on this CTA's barriers after it exits.
        for (int i = 0; i < stages && !aborted; ++i) {
            if (!wait_bounded_warp(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.timeout_ns,
                                   (blockIdx.x << 8) | 0x50u | stage))
                break;
            if (++stage == stages) stage = 0, phase ^= 1u;
        }
    } else if (warp == 1) {
        // -------------------------------------------------- MMA issuer ----
        int stage = 0;
        uint32_t phase = 0;
        uint32_t acc_phase = 0;
        bool aborted = false;
        const uint64_t pdesc = C::kPMn ? smem_desc_sw128(ring, C::kAtomBytes, 1024) : smem_desc_sw128(ring, 16, 1024);
        const uint64_t qdesc = C::kQMn ? smem_desc_sw128(ring + C::kPBytes, C::kAtomBytes, 1024)
                                       : smem_desc_sw128(ring + C::kPBytes, 16, 1024);
        for (int item = next_item(-1); item >= 0 && !aborted; item = next_item(item)) {
            const RowsItem w = uniform(tile_of(item));
            int kb0, kb1;
            share(w, kb0, kb1);
            if (kb0 == kb1) continue;  // nothing to sum: the epilogue writes zeros
            const int blocks = blocks_of(w);
            // columns of the MMA: the tile's rows rounded up to what the instruction takes
            const int n = w.cnt <= 16 ? 16 : (w.cnt + 31) & ~31;
            const uint32_t idesc = __shfl_sync(0xffffffffu, p.idesc | (static_cast<uint32_t>(n >> 3) << 17), 0);
            // stage st, k-block kb: operands in shared memory
            const auto ready = [&](int st, uint32_t ph) {
                return wait_bounded_warp(smem_u32(&full[st]), ph, abort_flag, p.timeout_ns,
                                         (blockIdx.x << 8) | 0x30u | st);
            };
            // The sum ends inside an MMA step of the last k-block: the step's
            // remaining rows belong to the next group and are overwritten with
            // zeros, in both operands (0 x NaN would not be 0).
            const auto clear_rest = [&](int st, int kb) {
                const int valid = valid_of(w, kb);
                if (!C::kWeight || (valid & 15) == 0) return;
                uint8_t* base = smem + st * C::kStageBytes;
                const int extra = 16 - (valid & 15);
                const int pa = 2 * blocks;
                for (int i = lane; i < (pa + (n + 63) / 64) * extra * 8; i += 32) {
                    const int a = i / (extra * 8), r = valid + (i / 8) % extra;
                    uint8_t* atom = base + (a < pa ? a * C::kAtomBytes : C::kPBytes + (a - pa) * C::kAtomBytes);
                    *reinterpret_cast<uint4*>(atom + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
            };
            // the MMAs of k-block kb in stage st into the accumulator blocks of
            // `mask`; a descriptor's low word is an address in 16-byte units
            const auto issue = [&](int st, int kb, int mask, uint32_t d, bool fresh) {
                tc_fence_after();
                // (broadcasts, so that the compiler knows the operands to be uniform)
                const uint64_t at = static_cast<uint64_t>(__shfl_sync(0xffffffffu, st, 0)) * (C::kStageBytes / 16);
                const int ksteps =
                    __shfl_sync(0xffffffffu, (valid_of(w, kb) + C::kUmmaK - 1) / C::kUmmaK, 0);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < C::kBK / C::kUmmaK; ++k) {
                        if (k >= ksteps) break;
                        const uint64_t qd = qdesc + at + k * (C::kQMn ? C::kUmmaK * 8 : 2);
                        const uint64_t pd = pdesc + at + k * (C::kPMn ? C::kUmmaK * 8 : 2);
                        const uint32_t sum = !fresh || k > 0 ? 1u : 0u;
                        if (mask & 1) umma<C::kKind>(d, pd, qd, idesc, sum);
                        if (C::kSub == 2 && (mask & 2))
                            umma<C::kKind>(d + C::kBQ, pd + C::kSubBytes / 16, qd, idesc, sum);
                    }
                }
                __syncwarp();
            };
            const auto release = [&]() {
                if (elect_one()) umma_commit(smem_u32(&empty[stage]));
                __syncwarp();
                if (++stage == stages) stage = 0, phase ^= 1u;
            };
            const auto complete = [&](int h) {
                if (elect_one()) umma_commit(smem_u32(&tfull[h]));
                __syncwarp();
            };
            if (C::kSub == 2 && !wait_bounded_warp(smem_u32(&tempty[0]), acc_phase ^ 1u, abort_flag, p.timeout_ns,
                                                   (blockIdx.x << 8) | 0x20u))
                break;
            const int mask = blocks == 2 ? 3 : 1;
            int kb = kb0;
            if constexpr (C::kSub == 2) {
                // Both accumulators belong to one tile, so the epilogue has to
                // overlap the MMAs of the other block: while block 1 is still
                // being read, k-blocks go into block 0 only (their stages stay
                // held) and into block 1 once it is free; and the last k-blocks
                // go into block 0 first, so its epilogue starts early.
                const int pre = kb1 - kb0 < stages ? kb1 - kb0 : stages;
                int held = 0, st = stage;
                uint32_t ph = phase;
                const auto next = [&]() {
                    if (++st == stages) st = 0, ph ^= 1u;
                };
                bool free1 = __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&tempty[1]), acc_phase ^ 1u));
                while (!free1 && held < pre) {
                    if (!ready(st, ph)) {
                        aborted = true;
                        break;
                    }
                    if (kb0 + held == kb1 - 1) clear_rest(st, kb0 + held);
                    issue(st, kb0 + held, 1, tmem_base, held == 0);
                    ++held;
                    next();
                    free1 = __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&tempty[1]), acc_phase ^ 1u));
                }
                if (aborted) break;
                if (!free1 && !wait_bounded_warp(smem_u32(&tempty[1]), acc_phase ^ 1u, abort_flag, p.timeout_ns,
                                                 (blockIdx.x << 8) | 0x21u))
                    break;
                for (; kb < kb0 + held; ++kb) {
                    issue(stage, kb, mask & 2, tmem_base, kb == kb0);
                    release();
                }
                const int last = kb1 - kb < stages ? kb1 - kb : stages;
                for (; kb < kb1 - last; ++kb) {
                    if (!ready(stage, phase)) {
                        aborted = true;
                        break;
                    }
                    issue(stage, kb, mask, tmem_base, kb == kb0);
                    release();
                }
                if (aborted) break;
                st = stage;
                ph = phase;
                for (int i = 0; i < last; ++i) {
                    if (!ready(st, ph)) {
                        aborted = true;
                        break;
                    }
                    if (kb + i == kb1 - 1) clear_rest(st, kb + i);
                    issue(st, kb + i, 1, tmem_base, kb + i == kb0);
                    next();
                }
                if (aborted) break;
                complete(0);
                for (; kb < kb1; ++kb) {
                    issue(stage, kb, mask & 2, tmem_base, kb == kb0);
                    release();
                }
                complete(1);
            } else {
                // Chunks of the sum into two accumulators in turn: the epilogue
                // takes one to its registers while the other fills.
                int part = 0;  // k-blocks of the chunk so far
                int buf = 0;
                for (; kb < kb1; ++kb) {
                    if (part == 0 && !wait_bounded_warp(smem_u32(&tempty[buf]), acc_phase ^ 1u, abort_flag,
                                                        p.timeout_ns, (blockIdx.x << 8) | 0x20u | buf)) {
                        aborted = true;
                        break;
                    }
                    if (!ready(stage, phase)) {
                        aborted = true;
                        break;
                    }
                    if (kb == kb1 - 1) clear_rest(stage, kb);
                    issue(stage, kb, 1, tmem_base + buf * C::kBQ, part == 0);
                    release();
                    if (++part == p.chunk || kb == kb1 - 1) {
                        complete(buf);
                        part = 0;
                        buf ^= 1;
                        if (buf == 0) acc_phase ^= 1u;
                    }
                }
                if (aborted) break;
            }
            acc_phase ^= 1u;
        }
    } else if (warp >= 2 && warp < 2 + C::kEpiWarps) {
        // ---------------------------------------------------- epilogue ----
        const int quarter = warp & 3;
        const int group = (warp - 2) >> 2;  // two groups of four warps: 32 columns each in turn, or a block each
        float* warp_scales = scales + (warp - 2) * 32;
        uint32_t* stage_out = reinterpret_cast<uint32_t*>(out_area + group * C::kOutBytes);
        uint32_t acc_phase = 0;
        bool lost = false;
        if (p.early) grid_dependency_wait();  // the rows' scales, and the output's last readers
        if (S > 1) cluster_wait();
        // Dynamic: each warp waits for the item on its own, and on the abort path
        // one may give up where its neighbours still see the item arrive; the
        // group takes an item only if all four have it.
        const auto group_item = [&](int item) {
            item = next_item(item);
            if (dynamic && !named_barrier_and(2 + group, 128, item >= 0)) item = -1;
            return item;
        };
        for (int item = group_item(-1); item >= 0 && !lost; item = group_item(item)) {
            const RowsItem w = tile_of(item);
            int kb0, kb1;
            share(w, kb0, kb1);
            const bool empty_sum = kb0 == kb1;
            const long long row = C::kWeight ? static_cast<long long>(w.e) * p.Q + w.q0 : w.row0;
            float sp = 0.f, bias = 0.f;  // of this lane's feature in the current block
            // wait for accumulator (kSub = 2: block) h; the four warps of a group
            // agree on the outcome: none is left waiting at a barrier that
            // another has given up
            const auto await = [&](int h, uint32_t parity) {
                const bool ok = wait_bounded_warp(smem_u32(&tfull[h]), parity, abort_flag, p.timeout_ns,
                                                  (blockIdx.x << 8) | 0x40u | h);
                if (!named_barrier_and(2 + group, 128, ok)) lost = true;
                tc_fence_after();
            };
            const auto channel = [&](int h) {
                const int f = w.p0 + h * 128 + quarter * 32 + lane;
                if (C::kKind == kKindI8 && S == 1 && f < p.P && !w.zero) {
                    const long long at = static_cast<long long>(w.e) * p.P + f;
                    sp = p.scale_p[at];
                    bias = p.bias_p ? p.bias_p[at] : 0.f;
                }
            };
            // 32 columns of the accumulators from column c on
            const auto load = [&](int c, uint32_t (&v)[32]) {
                tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(c), v);
            };
            const auto rows_scales = [&](int c) {
                if (C::kKind == kKindI8) {  // the rows' scales, for every lane to read
                    __syncwarp();
                    warp_scales[lane] = !w.zero && c + lane < w.cnt ? p.scale_q[w.row0 + c + lane] : 0.f;
                    __syncwarp();
                }
            };
            const auto results = [&](const uint32_t (&v)[32], float (&x)[32]) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    // int8: the int32 sum, rounded to fp32 once, times both scales, plus the bias
                    if (C::kKind == kKindI8)
                        x[j] = fmaf(__int2float_rn(static_cast<int>(v[j])) * warp_scales[j], sp, bias);
                    else
                        x[j] = __uint_as_float(v[j]);
                }
            };
            const auto release = [&](int h) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&tempty[h]));
            };
            const auto block_of = [&](int h, int c) {
                return OutBlock{p.out, row + c, p.P, w.p0 + h * 128, min(32, w.cnt - c),
                                min(128, p.P - w.p0 - h * 128), p.aligned_out != 0};
            };
            const auto store = [&](const float (&x)[32], const OutBlock& o) {
                if (p.out_type == kOutF32) {
                    store_block32(x, o, stage_out, quarter, lane, 2 + group);
                } else {
                    uint32_t words[16];
                    pack_block(x, p.out_type == kOutBF16, words);
                    if (o.aligned)
                        store_block16(words, o, stage_out, quarter, lane, 2 + group);
                    else
                        store_rows16(words, o, quarter, lane);
                }
            };
            if constexpr (C::kSub == 1) {
                // The sum, chunk by chunk, in this thread's registers.
                constexpr int kMine = (C::kBQ + 63) / 64;  // blocks of 32 columns
                uint32_t sum[kMine][32];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[i][j] = 0u;
                channel(0);
                int buf = 0;
                uint32_t parity = 0;
                for (int kb = kb0; kb < kb1;) {
                    await(buf, parity);
                    if (lost) break;
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        const int c = 32 * group + 64 * i;
                        if (c >= w.cnt) continue;
                        uint32_t v[32];
                        load(buf * C::kBQ + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            sum[i][j] = C::kChunks ? __float_as_uint(__uint_as_float(sum[i][j]) + __uint_as_float(v[j]))
                                                   : v[j];
                    }
                    release(buf);
                    if (kb1 - kb <= p.chunk) break;
                    kb += p.chunk;
                    buf ^= 1;
                    if (buf == 0) parity ^= 1u;
                }
                if (lost) break;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int c = 32 * group + 64 * i;
                    if (c >= w.cnt) continue;
                    if (S > 1) {
                        push_part<C>(sum[i], red, rank, p.split_log2, c, min(32, w.cnt - c), quarter * 32 + lane);
                        continue;
                    }
                    float x[32];
                    rows_scales(c);
                    results(sum[i], x);
                    store(x, block_of(0, c));
                }
            } else {
                // In two parts: blocks 0 and 1, of which this group takes every
                // other 32 columns; kOwnBlock: the halves of its block.
                const auto block = [&](int part) { return C::kOwnBlock ? group : part; };
                const auto column = [&](int part, int i) {
                    return C::kOwnBlock ? 128 * part + 32 * i : 32 * group + 64 * i;
                };
                const auto arrived = [&](int part) {
                    if (C::kOwnBlock && part == 1) return;
                    await(block(part), acc_phase);
                    channel(block(part));
                };
                const auto done = [&](int part) {
                    if (!C::kOwnBlock || part == 1) release(block(part));
                };
                if (empty_sum) {
                    // rows outside the groups, a group without rows: zeros
                    const float x[32] = {};
#pragma unroll 1
                    for (int k = 0; k < 8; ++k) {
                        const int c = column(k / 4, k % 4);
                        const OutBlock o = block_of(block(k / 4), c);
                        if (c < w.cnt && o.features > 0) store(x, o);
                    }
                } else if (p.out_type != kOutF32 && p.aligned_out) {
                    // Both parts into registers (128 words a thread) before any
                    // store: the accumulators are free for the next tile after
                    // about 3000 cycles instead of the 11000 that the stores of
                    // all SMs at once take.
                    uint32_t held[2][4][16];
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        if (lost) break;
                        arrived(part);
                        if (lost) break;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = column(part, i);
                            if (c < w.cnt) {
                                uint32_t v[32];
                                float x[32];
                                load(block(part) * C::kBQ + c, v);
                                rows_scales(c);
                                tmem_ld_wait();
                                results(v, x);
                                pack_block(x, p.out_type == kOutBF16, held[part][i]);
                            }
                        }
                        done(part);
                    }
                    if (lost) break;
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = column(part, i);
                            const OutBlock o = block_of(block(part), c);
                            if (c < w.cnt && o.features > 0)
                                store_block16(held[part][i], o, stage_out, quarter, lane, 2 + group);
                        }
                } else {
                    for (int part = 0; part < 2; ++part) {
                        arrived(part);
                        if (lost) break;
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {
                            const int c = column(part, i);
                            const OutBlock o = block_of(block(part), c);
                            if (c >= w.cnt || o.features <= 0) break;  // (uniform) the tile's end, the last tile's second block
                            uint32_t v[32];
                            float x[32];
                            load(block(part) * C::kBQ + c, v);
                            rows_scales(c);
                            tmem_ld_wait();
                            results(v, x);
                            store(x, o);
                        }
                        done(part);
                    }
                }
            }
            if (!empty_sum) acc_phase ^= 1u;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // Some role gave up.  Before shared and tensor memory are released,
        // let this CTA's own copies land and its MMAs retire.
        // (`issued` is zero outside the producer's warp; elect_one picks the same
        // lane of the converged warp that issued the MMAs)
        for (int s = 0; s < stages; ++s)
            if (issued & (1u << s)) drain_wait(smem_u32(&full[s]), (issued_parity >> s) & 1u);
        __syncwarp();
        if (warp == 1) {
            if (elect_one()) {
                umma_commit(smem_u32(drain));
                drain_wait(smem_u32(drain), 0);
            }
        }
        __syncwarp();
        __syncthreads();
    }
    if (C::kSub == 1 && S > 1) {
        const bool work = total > 0 && !*abort_flag;
        RowsItem w;
        float sp = 0.f, bias = 0.f;
        const int per = C::kBQ >> p.split_log2;
        const int t = static_cast<int>(threadIdx.x);
        if (work) {
            w = tile_of(0);
            if (C::kKind == kKindI8) {
                if (t < 256 && w.p0 + (t & 127) < p.P && !w.zero) {
                    const long long at = static_cast<long long>(w.e) * p.P + w.p0 + (t & 127);
                    sp = p.scale_p[at];
                    if (p.bias_p) bias = p.bias_p[at];
                }
                if (p.early) grid_dependency_wait();
                if (t < per)
                    scales[t] = rank * per + t < w.cnt && !w.zero ? p.scale_q[w.row0 + rank * per + t] : 0.f;
            }
        }
        if (warp < 2) cluster_wait();  // (the epilogue's warps have)
        cluster_sync_all();            // every part has arrived
        if (work && t < 256) {
            if (p.out_type == kOutF32)
                finish<C, float>(p, w, red, scales, rank, t, sp, bias);
            else if (p.out_type == kOutF16)
                finish<C, __half>(p, w, red, scales, rank, t, sp, bias);
            else
                finish<C, __nv_bfloat16>(p, w, red, scales, rank, t, sp, bias);
        }
    }
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
}

}  // namespace tcg
