// fpemu_host.h -- host-side helpers shared by the translation units of
// libfpemu.so: error text, device check, and where kernels record a failure.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "fpemu_internal.h"

namespace fpemu {

struct DeviceError;

// Records the detail behind fpemu_last_error() for this host thread; returns `code`.
int fail(int code, const char* fmt, ...);

struct DevInfo {
    int sms = 0;
    int major = 0, minor = 0;
};

// The current device; fails unless it is sm_100.
int device_info(DevInfo* out);

// The driver's encoder of TMA tensor maps (null if the driver has none).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

// How long a kernel's wait may take (FPEMU_WAIT_BUDGET_MS), and the unit at which
// the failure tests' producers stop (FPEMU_TEST_STALL_UNIT; -1: none).
uint64_t wait_budget_ns();
int test_stall_idx();

// Device address of the record that fpemu_device_error() reads, and of its
// host-visible copy (null until fpemu_watch_errors), for the current device.
// Kernels of other translation units get both as arguments.
struct ErrorSink {
    DeviceError* dev;
    DeviceError* host;
};
int error_sink(ErrorSink* out);

}  // namespace fpemu

#define FPEMU_CUDA(expr)                                                                        \
    do {                                                                                        \
        cudaError_t e_ = (expr);                                                                \
        if (e_ != cudaSuccess)                                                                  \
            return fpemu::fail(FPEMU_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_));        \
    } while (0)

#define FPEMU_TRY(expr)                \
    do {                               \
        int s_ = (expr);               \
        if (s_ != FPEMU_OK) return s_; \
    } while (0)
