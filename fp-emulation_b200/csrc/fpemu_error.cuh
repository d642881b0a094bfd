// fpemu_error.cuh -- the record of a kernel's first failure, read back with
// fpemu_device_error() and fpemu_poll_error().  Nothing traps.
#pragma once

#include <cuda_runtime.h>

#include "fpemu_host.h"

namespace fpemu {

struct DeviceError {
    int code;    // FPEMU_ERR_TIMEOUT, ...
    int where;   // which wait or check failed (kWait*, kWhere*)
    int block;   // blockIdx.x of the first failing CTA
    int detail;  // role-specific (unit index, stage, row, ...)
};

enum : int {
    kWhereAdapterIndex = 16,  // a row's adapter id is neither -1 nor an adapter
    kWaitAdapterFull = 17,    // an adapter kernel's warp waiting for a chunk
    kWaitAdapterEmpty = 18,   // its copying warps waiting for a free buffer
};

// First failure wins; `host` is the pinned mirror (null until it is watched).
__device__ __forceinline__ void report_error(DeviceError* err, volatile DeviceError* host, int code, int where,
                                             int detail) {
    if (err != nullptr && atomicCAS(&err->code, 0, code) == 0) {
        err->where = where;
        err->block = (int)blockIdx.x;
        err->detail = detail;
        __threadfence();
        if (host != nullptr) {
            host->where = where;
            host->block = (int)blockIdx.x;
            host->detail = detail;
            __threadfence_system();
            host->code = code;  // last: a non-zero code means the other fields are set
            __threadfence_system();
        }
    }
}

}  // namespace fpemu
