// status.cuh -- the library's error reporting, shared by the files that
// implement include/talos_cuda.h.
#pragma once

#include <cuda_runtime.h>

#include "../../include/talos_cuda.h"

namespace talos {

// Record the calling thread's error message and return st.
talos_status set_err(talos_status st, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// The streaming multiprocessors of a device (148 if it cannot be asked).
int sm_count_dev(int device);
// Set the attributes of the operators' kernels on a device (once each; it must be current).
talos_status ops_configured(int device);

}  // namespace talos

#define CK(call)                                                                                 \
    do {                                                                                         \
        cudaError_t e_ = (call);                                                                 \
        if (e_ != cudaSuccess)                                                                   \
            return set_err(e_ == cudaErrorMemoryAllocation ? TALOS_ERR_OOM : TALOS_ERR_CUDA,     \
                           "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__,     \
                           __LINE__);                                                            \
    } while (0)

#define TRY(call)                              \
    do {                                       \
        talos_status s_ = (call);              \
        if (s_ != TALOS_OK) return s_;         \
    } while (0)
