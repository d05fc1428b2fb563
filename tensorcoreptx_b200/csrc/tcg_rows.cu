// tcg_rows.cu -- host side of the row-scaled and grouped products declared in
// include/tcgemm.h: checks of arguments, choice of the tile, tensor maps and
// the launch of rows_kernel (tcg_rows_kernel.cuh) or few_rows_kernel (tcg_fewrows.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "../../include/tcgemm.h"
#include "tcg_fewrows.cuh"
#include "tcg_host.h"
#include "tcg_rows_kernel.cuh"

static_assert(TCG_MAX_GROUPS == tcg::kRowsMaxGroups, "groups of the table in shared memory");
static_assert(TCG_F32 == tcg::kOutF32 && TCG_F16 == tcg::kOutF16 && TCG_BF16 == tcg::kOutBF16, "output types");

namespace {

using namespace tcg;

std::atomic<int> g_rows_tile{0};
std::atomic<int> g_rows_split{0};

// One product, checked and ready to launch.
struct RowsCall {
    const void* pside;      // weights; weight form: the rows' other side
    const void* qside;      // rows; weight form: the gradient by the product's result
    void* out;
    int out_type;
    bool bf16;
    const int32_t* offsets;
    int groups, rows, P, Q, R;
    const float *scale_q, *scale_p, *bias_p;
    int zero_rest;
    int early;
};

struct RowsPlan {
    int bq;     // 16, 32, 64, 128 (kSub = 1) or 256 (kSub = 2)
    int split;
    int chunk;  // k-blocks summed in one go
};

int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Tiles of bq rows along the rows; an upper bound of them where the groups'
// bounds are known to the device only.
long long most_row_tiles(const RowsCall& c, int bq)
{
    if (!c.offsets) return static_cast<long long>(c.groups) * ceil_div(c.rows / c.groups, bq);
    long long parts = c.groups + (c.zero_rest ? 2 : 0);
    if (parts > c.rows) parts = c.rows;
    return (c.rows + parts * (bq - 1)) / bq;
}

// Tile and split: the least of a time model's estimates, in microseconds.  The
// model is a start (launch, first loads, last stores) plus the k-blocks that
// the busiest SM works through, each at a measured rate (B200, 36 shapes of
// 1 to 8192 rows and 1 to 64 groups timed with every tile and split):
//   kSub = 1:  4.0 + k-blocks x 0.20 (tiles of up to 64 rows: the rate at which
//              one CTA's loads and MMAs are issued) or x 0.30 (128 rows: bytes
//              from L2), x tiles per SM, and 1.7 or 2.2 a tile after the first
//              (its start and its stores, of which the CTAs of an SM hide half)
//   split:     5.5 + the same for a share of the k-blocks.  The exchange costs
//              1.5; a second wave of clusters costs far more than it saves (48
//              rows x 10240 x 4096 over 2 CTAs 10.9, over 4 in two waves 14.9),
//              so all clusters have to be resident at once: one CTA per SM, or
//              two with tiles of 16 rows (16 x 10240 x 4096 8.8 against 10.6
//              unsplit) and pairs with tiles of up to 64 (160 CTAs: 48 x 10240 x
//              4096 10.8 against 12.5; 170 x 5000 x 8192 16.4 against 21.7),
//              while more than 148 CTAs in fours find no room for some (180 x
//              3000 x 3008 13.9 against 8.7); clusters of eight CTAs fit few of
//              the GPU's processing clusters (16 of them take two waves), so at
//              most eight of those.
//   kSub = 2:  10 + k-blocks x 0.54 (the tensor cores' rate) for the first whole
//              wave, 4.5 + k-blocks x 0.54 for the others, at least 7 (128 KB of
//              results at the rate at which all SMs write, 14 bytes a cycle each)
// Example: int8 512 x 4096 x 4096 64 rows 13.4 (model 16.3), 128 rows 12.9
// (13.6), 256 rows 29.1 (27.3); 100 x 4096 x 4096: 32 rows 10.8, 64 rows on two
// CTAs 9.0, 128 rows on four 8.5.
RowsPlan choose_plan(const RowsCall& c, bool weight, int kblock, int sms)
{
    const int forced = g_rows_tile.load(), forced_split = g_rows_split.load();
    const double mean = static_cast<double>(c.rows) / c.groups;  // rows per group
    const double kb = weight ? (mean + kblock - 1) / kblock : ceil_div(c.R, kblock);
    const double used = c.groups < c.rows ? c.groups : c.rows;   // groups that can have rows
    // fp32 results of 16-bit sums: in chunks, which the tiles of 256 rows have no
    // room for.  Few rows, where the weights' bytes are the bound, take chunks of
    // 128 (86.5 us against 85.7 unchunked, 64 rows of 32 groups x 4096 x 2048);
    // tiles of more rows 256, or 512 in sums beyond 1024, whose error is that of
    // 256 in a sum of 1024 by an fp32 product's growth with its square root (8
    // groups, 4096 rows x 1536 x 2048: 41.9 us in chunks of 512, 44.3 in 256,
    // 55.6 in 128).
    const bool wide = kblock == 64 && c.out_type == kOutF32;
    const int length = weight ? c.rows : c.R;
    const bool fine = wide && length > 256;
    RowsPlan best{128, 1, 0x7fffffff};
    double least = -1;
    for (int bq = weight ? 128 : 16; bq <= 256; bq *= 2) {
        if (forced && bq != forced && !(weight && forced < 128 && bq == 128)) continue;
        if (!forced && fine && bq == 256) continue;
        const int tile_p = bq == 256 ? 256 : 128;
        double q;  // tiles along q: a ragged group ends half a tile early on average
        if (weight)
            q = static_cast<double>(c.groups) * ceil_div(c.Q, bq);
        else if (!c.offsets)
            q = static_cast<double>(c.groups) * ceil_div(c.rows / c.groups, bq);
        else
            q = std::max(used, static_cast<double>(c.rows) / bq + 0.5 * used);
        const double tiles = q * ceil_div(c.P, tile_p);
        const double bound = weight ? tiles : static_cast<double>(most_row_tiles(c, bq)) * ceil_div(c.P, tile_p);
        for (int split = 1; split <= (bq == 256 ? 1 : 8); split *= 2) {
            if (forced_split && bq != 256 && split != forced_split) continue;
            const int per_sm = bq == 16 || (bq <= 64 && split == 2) ? 2 : 1;
            // (tiles of 128 rows take an SM's shared memory, those of empty CTAs too)
            const double most = bq == 128 ? std::max(tiles, bound) : tiles;
            const bool resident = split == 8 ? most <= 8 : most * split <= per_sm * sms;
            if (split > 1 && !resident && !forced_split) continue;
            const double per = tiles * split / sms;  // tiles that an SM works through
            double t;
            if (bq == 256)
                t = 10.0 + kb * 0.54 + (std::ceil(per) - 1) * std::max(7.0, 4.5 + kb * 0.54);
            else
                t = (split > 1 ? 5.5 : 4.0) + std::max(1.0, per) * kb / split * (bq == 128 ? 0.30 : 0.20) +
                    (split > 1 ? 0.0 : std::max(0.0, per - 1) * (bq == 128 ? 2.2 : 1.7));
            if (least < 0 || t < least) {
                least = t;
                best = RowsPlan{bq, split, !wide ? 0x7fffffff : bq <= 32 ? 2 : length <= 1024 ? 4 : 8};
            }
        }
    }
    return best;
}

template <class C>
tcg_status launch(const RowsCall& c, int split, int chunk, int dev, int sms, cudaStream_t st)
{
    static std::atomic<bool> smem_set[host::kDevices];
    auto kern = rows_kernel<C>;
    constexpr int most = 232448;  // shared memory per CTA
    if (!smem_set[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return host::fail(e);
        smem_set[dev].store(true, std::memory_order_release);
    }

    const CUtensorMapDataType dt = C::kElem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t es = C::kElem, P = c.P, Q = c.Q, R = c.R, M = c.rows, G = c.groups;
    const CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B;
    // An MN-major operand of whole 64-element atoms is seen as {64, rows, atoms,
    // groups}, so that one copy brings a tile's atoms; otherwise (the last atom
    // ends inside a row) as {elements, rows, 1, groups}, a copy per atom.
    const uint32_t bk = C::kBK;
    const bool p_whole = c.P % 64 == 0, q_whole = c.Q % 64 == 0;
    const auto atoms = [&](uint64_t width, uint64_t rows, uint64_t groups, bool whole, uint32_t n) {
        const uint64_t pitch = width * es;
        return whole ? host::Box4{{64, rows, width / 64, groups}, {pitch, 128, rows * pitch}, {64, bk, n}}
                     : host::Box4{{width, rows, 1, groups}, {pitch, rows * pitch, rows * pitch}, {64, bk, 1}};
    };
    const auto k_major = [&](uint64_t rows, uint64_t groups, uint32_t n) {
        const uint64_t pitch = R * es;
        return host::Box4{{R, rows, 1, groups}, {pitch, rows * pitch, rows * pitch}, {bk, n, 1}};
    };
    CUtensorMap mp, mq, mqb;  // mqb: rows in boxes of kQBox, for tiles that are not full
    tcg_status s;
    if (C::kWeight)
        s = host::encode_4d(&mp, dt, c.pside, atoms(P, M, 1, p_whole, 2 * C::kSub), swz);
    else if (C::kPMn)
        s = host::encode_4d(&mp, dt, c.pside, atoms(P, R, G, p_whole, 2 * C::kSub), swz);
    else
        s = host::encode_4d(&mp, dt, c.pside, k_major(P, G, C::kTileP), swz);
    if (s == TCG_SUCCESS)
        s = C::kWeight ? host::encode_4d(&mq, dt, c.qside, atoms(Q, M, 1, q_whole, C::kBQ / 64), swz)
                       : host::encode_4d(&mq, dt, c.qside, k_major(M, 1, C::kBQ), swz);
    mqb = mq;
    if (s == TCG_SUCCESS && !C::kWeight && C::kBQ > C::kQBox)
        s = host::encode_4d(&mqb, dt, c.qside, k_major(M, 1, C::kQBox), swz);
    if (s != TCG_SUCCESS) return s;

    RowsParams p;
    std::memset(&p, 0, sizeof p);
    p.out = c.out;
    p.offsets = c.offsets;
    p.scale_q = c.scale_q;
    p.scale_p = c.scale_p;
    p.bias_p = c.bias_p;
    p.timeout_ns = host::wait_timeout_ns();
    p.groups = c.groups;
    p.rows = c.rows;
    p.rows_per_group = c.rows / c.groups;
    p.P = c.P;
    p.Q = c.Q;
    p.R = c.R;
    p.ptiles = ceil_div(c.P, C::kTileP);
    p.qtiles = ceil_div(C::kWeight ? c.Q : p.rows_per_group, C::kBQ);
    p.zero_rest = c.zero_rest;
    const auto smem_for = [&](int n) { return C::smem_bytes(n, split, c.offsets ? c.groups : 0); };
    const int out_bytes = c.out_type == kOutF32 ? 4 : 2;
    p.aligned_out = (static_cast<long long>(c.P) * out_bytes) % 16 == 0 && (reinterpret_cast<uintptr_t>(c.out) & 15u) == 0;
    p.out_type = c.out_type;
    while ((1 << p.split_log2) < split) ++p.split_log2;
    p.early = c.early;
    p.p_whole = p_whole;
    p.q_whole = q_whole;
    const uint32_t fmt = C::kKind == kKindI8 ? 1u : (c.bf16 ? 1u : 0u);
    p.idesc = make_idesc(C::kKind == kKindI8 ? 2u : 1u, fmt, fmt, C::kQMn, 128, 0) | (C::kPMn ? 1u << 15 : 0u);

    const long long qt = C::kWeight ? static_cast<long long>(c.groups) * p.qtiles : most_row_tiles(c, C::kBQ);
    const long long items = qt * p.ptiles;
    if (items > 0x7fffffffLL / 8 || p.ptiles > 65535) return TCG_ERR_SHAPE;
    // bands about square in elements over the tiles in flight
    while ((4LL << (2 * p.band_log2)) * C::kBQ <= static_cast<long long>(sms) * C::kTileP) ++p.band_log2;
    p.per_band_inv = div_inverse(static_cast<uint32_t>(p.ptiles) << p.band_log2);
    p.ptiles_inv = div_inverse(p.ptiles);
    p.per_group_inv = div_inverse(static_cast<uint32_t>(C::kWeight ? p.ptiles * p.qtiles : p.qtiles));

    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute attr[2];
    std::memset(attr, 0, sizeof attr);
    // A CTA per tile, taken over as they finish, where the exact number of tiles
    // is known (the bound of ragged rows is too high by up to a tile per group
    // and p-tile: empty CTAs would follow) and tiles are long enough for the
    // answer to arrive meanwhile: bf16 8192 x 8192 x 4096 398 -> 373 us, int8
    // 16384 x 8192 x 8192 807 -> 782; but gradients of 16 k-blocks 214 -> 229.
    const int tile_kb = ceil_div(C::kWeight ? c.rows / c.groups : c.R, C::kBK);
    p.dynamic = C::kSub == 2 && items > sms && (C::kWeight || !c.offsets) && tile_kb >= 32;
    if (C::kSub == 2)
        cfg.gridDim = dim3(static_cast<unsigned>(items > sms && !p.dynamic ? sms : items), 1, 1);
    else if (C::kWeight)
        cfg.gridDim = dim3(static_cast<unsigned>(p.qtiles * split), p.ptiles, c.groups);
    else
        cfg.gridDim = dim3(static_cast<unsigned>(qt * split), p.ptiles, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    // Ring depth: all of shared memory for one CTA per SM; half of it, so that
    // one CTA's start and end overlap another's loads, where there are more
    // CTAs than SMs (kSub = 1).
    const int room = C::kSub == 1 && items * split > sms && 2 * smem_for(2) <= most - 2048
                         ? (most - 2048) / 2
                         : most;
    int stages = (room - smem_for(0)) / C::kStageBytes;
    if (stages > C::kMaxStages) stages = C::kMaxStages;
    if (C::kSub == 1 && !C::kWeight)  // no more than a CTA's share of the sum: what is left can start the next kernel
        stages = std::max(2, std::min(stages, ceil_div(ceil_div(c.R, C::kBK), split)));
    p.stages = stages;
    p.chunk = chunk;
    cfg.dynamicSmemBytes = smem_for(stages);
    cfg.stream = st;
    cfg.attrs = attr;
    if (split > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(split);
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (host::dependent_launch()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mp, mq, mqb, p);
    return e == cudaSuccess ? TCG_SUCCESS : host::fail(e);
}

template <int kKind, bool kPMn>
tcg_status run_rows(const RowsCall& c, cudaStream_t st)
{
    int dev, sms;
    const tcg_status s = host::device(&dev, &sms);
    if (s != TCG_SUCCESS) return s;
    const RowsPlan plan = choose_plan(c, false, kKind == kKindF16 ? 64 : 128, sms);
    switch (plan.bq) {
    case 16: return launch<RowsTraits<kKind, kPMn, false, 1, 16>>(c, plan.split, plan.chunk, dev, sms, st);
    case 32: return launch<RowsTraits<kKind, kPMn, false, 1, 32>>(c, plan.split, plan.chunk, dev, sms, st);
    case 64: return launch<RowsTraits<kKind, kPMn, false, 1, 64>>(c, plan.split, plan.chunk, dev, sms, st);
    case 128: return launch<RowsTraits<kKind, kPMn, false, 1, 128>>(c, plan.split, plan.chunk, dev, sms, st);
    default: return launch<RowsTraits<kKind, kPMn, false, 2, 256>>(c, 1, plan.chunk, dev, sms, st);
    }
}

tcg_status run_weight(const RowsCall& c, cudaStream_t st)
{
    int dev, sms;
    const tcg_status s = host::device(&dev, &sms);
    if (s != TCG_SUCCESS) return s;
    const RowsPlan plan = choose_plan(c, true, 64, sms);
    if (plan.bq == 256) return launch<RowsTraits<kKindF16, true, true, 2, 256>>(c, 1, plan.chunk, dev, sms, st);
    return launch<RowsTraits<kKindF16, true, true, 1, 128>>(c, plan.split, plan.chunk, dev, sms, st);
}

template <class T, int kM, int kF>
tcg_status launch_few(const FewParams& p, int sms, cudaStream_t st)
{
    static_assert(kFewCodes <= 40 * 1024, "shared memory without opting in");
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute attr[1];
    std::memset(attr, 0, sizeof attr);
    const int blocks = ceil_div(p.n, kFewWarps * kF);
    cfg.gridDim = dim3(static_cast<unsigned>(blocks < 2 * sms ? blocks : 2 * sms), 1, 1);
    cfg.blockDim = dim3(kFewThreads, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(kM) * p.k;
    cfg.stream = st;
    cfg.attrs = attr;
    if (host::dependent_launch()) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, few_rows_kernel<T, kM, kF>, p);
    return e == cudaSuccess ? TCG_SUCCESS : host::fail(e);
}

template <class T>
tcg_status run_few(const FewParams& p, int rows, cudaStream_t st)
{
    int dev, sms;
    const tcg_status s = host::device(&dev, &sms);
    if (s != TCG_SUCCESS) return s;
    const bool pair = p.n >= kFewPair;
    switch (rows) {
    case 1: return launch_few<T, 1, 1>(p, sms, st);
    case 2: return pair ? launch_few<T, 2, 2>(p, sms, st) : launch_few<T, 2, 1>(p, sms, st);
    case 3: return pair ? launch_few<T, 3, 2>(p, sms, st) : launch_few<T, 3, 1>(p, sms, st);
    default: return pair ? launch_few<T, 4, 2>(p, sms, st) : launch_few<T, 4, 1>(p, sms, st);
    }
}

// Whether few_rows_kernel takes a product of ungrouped rows.
bool few_rows(int M, int N, int K)
{
    return M <= kFewRows && static_cast<long long>(M) * K <= kFewCodes &&
           static_cast<long long>(M) * N * K <= kFewWork;
}

bool is_type(tcg_dtype t) { return t == TCG_F32 || t == TCG_F16 || t == TCG_BF16; }
bool misaligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) % n) != 0; }
unsigned size_of(tcg_dtype t) { return t == TCG_F32 ? 4u : 2u; }
// Longest sum of an int8 product: the int32 sums are exact whatever the codes
// as long as 128 * 128 * K is below 2^31.
constexpr int kMostK8 = 131056;
size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Checks shared by every form; *done: there is no output.
tcg_status check(int M, int N, int K, int groups, const int32_t* offsets, long long out_elems, bool* done)
{
    *done = false;
    if (M < 0 || N < 0 || K < 0 || groups < 0) return TCG_ERR_SHAPE;
    if (out_elems == 0) {
        *done = true;
        return TCG_SUCCESS;
    }
    if (groups == 0 || groups > (offsets ? TCG_MAX_GROUPS : 65535)) return TCG_ERR_SHAPE;  // (table; grid)
    if (!offsets && M % groups != 0) return TCG_ERR_SHAPE;
    if (misaligned(offsets, 4)) return TCG_ERR_ALIGN;
    return TCG_SUCCESS;
}

// The call that multiplies rows of codes A.
RowsCall s8_call(const int8_t* A, const int8_t* B, void* C, tcg_dtype c_type, const int32_t* offsets, int groups, int M,
                 int N, int K, const float* scale_a, const float* scale_b, const float* bias, int zero_rest)
{
    RowsCall c;
    std::memset(&c, 0, sizeof c);
    c.pside = B;
    c.qside = A;
    c.out = C;
    c.out_type = c_type;
    c.offsets = offsets;
    c.groups = groups;
    c.rows = M;
    c.P = N;
    c.R = K;
    c.scale_q = scale_a;
    c.scale_p = scale_b;
    c.bias_p = bias;
    c.zero_rest = zero_rest;
    return c;
}

tcg_status gemm_s8(const int8_t* A, const int8_t* B, void* C, tcg_dtype c_type, const int32_t* offsets, int groups,
                   int M, int N, int K, const float* scale_a, const float* scale_b, const float* bias, int zero_rest,
                   int early, cudaStream_t st)
{
    if (!A || !B || !C || !scale_a || !scale_b) return TCG_ERR_ARG;
    if (K == 0 || K % 16 != 0 || K > kMostK8) return TCG_ERR_SHAPE;
    if (misaligned(A, 16) || misaligned(B, 16) || misaligned(C, size_of(c_type)) || misaligned(scale_a, 4) ||
        misaligned(scale_b, 4) || misaligned(bias, 4))
        return TCG_ERR_ALIGN;
    RowsCall c = s8_call(A, B, C, c_type, offsets, groups, M, N, K, scale_a, scale_b, bias, zero_rest);
    c.early = early && host::dependent_launch();
    return run_rows<kKindI8, false>(c, st);
}

}  // namespace

namespace tcg {
namespace host {

cudaError_t read_rows_error(unsigned long long* word)
{
    return cudaMemcpyFromSymbol(word, tcg::g_tcg_error_word, sizeof *word);
}

cudaError_t clear_rows_error()
{
    const unsigned long long zero = 0;
    return cudaMemcpyToSymbol(tcg::g_tcg_error_word, &zero, sizeof zero);
}

}  // namespace host
}  // namespace tcg

extern "C" {

tcg_status tcg_gemm_s8_grouped(const int8_t* A, const int8_t* B, void* C, tcg_dtype c_type, const int32_t* offsets,
                               int groups, int M, int N, int K, const float* scale_a, const float* scale_b,
                               const float* bias, int zero_rest, void* stream)
{
    if (!is_type(c_type)) return TCG_ERR_ARG;
    bool done;
    const tcg_status s = check(M, N, K, groups, offsets, static_cast<long long>(M) * N, &done);
    if (s != TCG_SUCCESS || done) return s;
    return gemm_s8(A, B, C, c_type, offsets, groups, M, N, K, scale_a, scale_b, bias, zero_rest, 0,
                   static_cast<cudaStream_t>(stream));
}

tcg_status tcg_gemm_s8_scaled(const int8_t* A, const int8_t* B, void* C, tcg_dtype c_type, int M, int N, int K,
                              int batches, const float* scale_a, const float* scale_b, const float* bias,
                              void* stream)
{
    if (M < 0 || batches < 0) return TCG_ERR_SHAPE;
    const long long rows = static_cast<long long>(M) * batches;
    if (rows > 0x7fffffffLL) return TCG_ERR_SHAPE;
    return tcg_gemm_s8_grouped(A, B, C, c_type, nullptr, batches, static_cast<int>(rows), N, K, scale_a, scale_b, bias,
                               0, stream);
}

size_t tcg_linear_s8_workspace_size(int M, int K)
{
    if (M <= 0 || K <= 0) return 0;
    return round256(static_cast<size_t>(M) * K) + round256(static_cast<size_t>(M) * sizeof(float));
}

tcg_status tcg_linear_s8_grouped(const void* x, tcg_dtype x_type, const int8_t* B, void* C, tcg_dtype c_type,
                                 const int32_t* offsets, int groups, int M, int N, int K, const float* scale_b,
                                 const float* bias, int zero_rest, void* workspace, size_t workspace_bytes,
                                 void* stream)
{
    if (!is_type(x_type) || !is_type(c_type)) return TCG_ERR_ARG;
    bool done;
    tcg_status s = check(M, N, K, groups, offsets, static_cast<long long>(M) * N, &done);
    if (s != TCG_SUCCESS || done) return s;
    // everything is checked before the first launch
    if (!x || !B || !C || !scale_b) return TCG_ERR_ARG;
    if (K == 0 || K % 16 != 0 || K > kMostK8) return TCG_ERR_SHAPE;
    if (misaligned(x, size_of(x_type)) || misaligned(B, 16) || misaligned(C, size_of(c_type)) ||
        misaligned(scale_b, 4) || misaligned(bias, 4))
        return TCG_ERR_ALIGN;
    if (!offsets && groups == 1 && few_rows(M, N, K) && !misaligned(x, 16)) {
        const FewParams p{x, B, C, scale_b, bias, N, K, c_type};
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (x_type == TCG_F32) return run_few<float>(p, M, st);
        if (x_type == TCG_F16) return run_few<__half>(p, M, st);
        return run_few<__nv_bfloat16>(p, M, st);
    }
    if (!workspace || workspace_bytes < tcg_linear_s8_workspace_size(M, K)) return TCG_ERR_WORKSPACE;
    if (misaligned(workspace, 256)) return TCG_ERR_ALIGN;
    int8_t* codes = static_cast<int8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(codes + round256(static_cast<size_t>(M) * K));
    s = tcg_quantize_rows_s8(x, x_type, codes, scale, M, K, stream);
    if (s != TCG_SUCCESS) return s;
    return gemm_s8(codes, B, C, c_type, offsets, groups, M, N, K, scale, scale_b, bias, zero_rest, 1,
                   static_cast<cudaStream_t>(stream));
}

tcg_status tcg_linear_s8(const void* x, tcg_dtype x_type, const int8_t* B, void* C, tcg_dtype c_type, int M, int N,
                         int K, const float* scale_b, const float* bias, void* workspace, size_t workspace_bytes,
                         void* stream)
{
    return tcg_linear_s8_grouped(x, x_type, B, C, c_type, nullptr, 1, M, N, K, scale_b, bias, 0, workspace,
                                 workspace_bytes, stream);
}

tcg_status tcg_gemm_16_grouped(const void* A, const void* B, tcg_dtype type, void* C, tcg_dtype c_type,
                               const int32_t* offsets, int groups, int M, int N, int K, tcg_b_layout b_layout,
                               int zero_rest, void* stream)
{
    if ((type != TCG_F16 && type != TCG_BF16) || !is_type(c_type)) return TCG_ERR_ARG;
    if (b_layout != TCG_B_KN && b_layout != TCG_B_NK) return TCG_ERR_ARG;
    bool done;
    const tcg_status s = check(M, N, K, groups, offsets, static_cast<long long>(M) * N, &done);
    if (s != TCG_SUCCESS || done) return s;
    if (!A || !B || !C) return TCG_ERR_ARG;
    if (K == 0 || K % 8 != 0 || (b_layout == TCG_B_KN && N % 8 != 0)) return TCG_ERR_SHAPE;
    if (misaligned(A, 16) || misaligned(B, 16) || misaligned(C, size_of(c_type))) return TCG_ERR_ALIGN;
    RowsCall c;
    std::memset(&c, 0, sizeof c);
    c.pside = B;
    c.qside = A;
    c.out = C;
    c.out_type = c_type;
    c.bf16 = type == TCG_BF16;
    c.offsets = offsets;
    c.groups = groups;
    c.rows = M;
    c.P = N;
    c.R = K;
    c.zero_rest = zero_rest;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return b_layout == TCG_B_NK ? run_rows<kKindF16, false>(c, st) : run_rows<kKindF16, true>(c, st);
}

tcg_status tcg_gemm_16_grouped_wgrad(const void* dC, const void* A, tcg_dtype type, void* dB, tcg_dtype b_type,
                                     const int32_t* offsets, int groups, int M, int N, int K,
                                     void* stream)
{
    if ((type != TCG_F16 && type != TCG_BF16) || !is_type(b_type)) return TCG_ERR_ARG;
    bool done;
    const long long weights = static_cast<long long>(groups < 0 ? 0 : groups) * N;
    const tcg_status s = check(M, N, K, groups, offsets, K > 0 ? weights : 0, &done);
    if (s != TCG_SUCCESS || done) return s;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!dB) return TCG_ERR_ARG;
    if (N % 8 != 0 || K % 8 != 0) return TCG_ERR_SHAPE;
    if (misaligned(dB, size_of(b_type))) return TCG_ERR_ALIGN;
    if (M == 0) {  // no rows at all: every gradient is zero
        const cudaError_t e = cudaMemsetAsync(dB, 0, static_cast<size_t>(weights) * K * size_of(b_type), st);
        return e == cudaSuccess ? TCG_SUCCESS : host::fail(e);
    }
    if (!dC || !A) return TCG_ERR_ARG;
    if (misaligned(dC, 16) || misaligned(A, 16)) return TCG_ERR_ALIGN;
    RowsCall c;
    std::memset(&c, 0, sizeof c);
    c.pside = A;
    c.qside = dC;
    c.out = dB;
    c.out_type = b_type;
    c.bf16 = type == TCG_BF16;
    c.offsets = offsets;
    c.groups = groups;
    c.rows = M;
    c.P = K;
    c.Q = N;
    return run_weight(c, st);
}

void tcg_set_rows_tile(int rows, int split)
{
    const bool tile = rows == 16 || rows == 32 || rows == 64 || rows == 128 || rows == 256;
    const bool parts = split == 1 || split == 2 || split == 4 || split == 8;
    g_rows_tile.store(tile ? rows : 0);
    g_rows_split.store(parts ? split : 0);
}

}  // extern "C"
