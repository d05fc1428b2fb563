// tcg_wait.cuh -- bounded mbarrier waits and the failure word they record,
// shared by every kernel that waits on an mbarrier.
#pragma once

#include "tcg_ptx.cuh"

namespace tcg {

constexpr uint32_t kErrWaitTimeout = 1;  // failure code in the high word

// Failure word, one per device and translation unit (each of the library's
// .cu files has its own; tcg_check_device_error reads them all).
static __device__ unsigned long long g_tcg_error_word = 0ull;

__device__ __forceinline__ void record_failure(volatile uint32_t* abort_flag, uint32_t detail)
{
    *abort_flag = 1u;
    __threadfence_block();
    atomicCAS(&g_tcg_error_word, 0ull,
              (static_cast<unsigned long long>(kErrWaitTimeout) << 32) | detail);
}

// One try_wait; kClusterScope: acquire at cluster scope (data written into
// this CTA's shared memory by the other CTA of its cluster).
template <bool kClusterScope = false>
__device__ __forceinline__ bool try_wait_scoped(uint32_t bar, uint32_t parity)
{
    return kClusterScope ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
}

// Single-thread bounded wait.  true: the phase of `parity` completed.
// false: this CTA is aborting (this wait expired, or another role's did).
template <bool kClusterScope = false>
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                             unsigned long long timeout_ns, uint32_t detail)
{
    if (try_wait_scoped<kClusterScope>(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    while (true) {
        if (try_wait_scoped<kClusterScope>(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_timer_ns() - t0 > timeout_ns) {
            record_failure(abort_flag, detail);
            return false;
        }
    }
}

// Whole-warp bounded wait with a warp-uniform result.  A completed phase is
// sticky until every waiter has arrived for the next one, so once any lane
// sees completion all lanes will.
template <bool kClusterScope = false>
__device__ __forceinline__ bool wait_bounded_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                  unsigned long long timeout_ns, uint32_t detail)
{
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        const bool ok = try_wait_scoped<kClusterScope>(bar, parity);
        if (__all_sync(0xffffffffu, ok)) return true;
        if (__any_sync(0xffffffffu, ok)) continue;
        if (i == 0) t0 = global_timer_ns();
        const bool ab = (*abort_flag != 0u);
        const bool expired = (global_timer_ns() - t0) > timeout_ns;
        const unsigned stop = __ballot_sync(0xffffffffu, ab || expired);
        if (stop) {
            if ((threadIdx.x & 31) == (__ffs(stop) - 1) && !ab) record_failure(abort_flag, detail);
            return false;
        }
    }
}

// Bounded drain wait used only on the abort path (ignores the abort flag).
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity)
{
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (global_timer_ns() - t0 > 200000000ull) return;  // 200 ms
    }
}

}  // namespace tcg
