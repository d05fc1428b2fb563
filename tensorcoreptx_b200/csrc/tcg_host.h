// tcg_host.h -- host-side services that the library's translation units share
// (defined in tcgemm.cu; the rows_error functions in tcg_rows.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/tcgemm.h"

#pragma GCC visibility push(hidden)
namespace tcg {
namespace host {

constexpr int kDevices = 64;

// Record a CUDA error for tcg_last_cuda_error; returns TCG_ERR_CUDA.
tcg_status fail(cudaError_t e);

// The current device (TCG_ERR_UNSUPPORTED unless sm_100), its SM count, and
// the driver's tensor-map encoder resolved.
tcg_status device(int* id, int* sms);

// A 4-D tiled tensor map: extents (innermost first, contiguous), byte strides
// of the outer three, box extents of the inner three (the fourth is 1).
struct Box4 {
    uint64_t d[4], s[3];
    uint32_t box[3];
};
tcg_status encode_4d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, const Box4& b,
                     CUtensorMapSwizzle swz);

bool dependent_launch();               // programmatic dependent launch (TCG_PDL)
unsigned long long wait_timeout_ns();  // tcg_set_wait_timeout_ns

// The failure word of tcg_rows.cu's kernels on this device.
cudaError_t read_rows_error(unsigned long long* word);
cudaError_t clear_rows_error();

}  // namespace host
}  // namespace tcg
#pragma GCC visibility pop
