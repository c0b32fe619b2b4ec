// dw_host.h -- what the C entry points outside dw_capi.cu share with it: the
// thread's last-error text and the check that the current device is usable.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dwb {

// Remember a CUDA failure for dwb_last_error(); returns DWB_ERR_CUDA.
int record_cuda_failure(const char* what, cudaError_t e);

// DWB_OK when the current device is an sm_100 part this library has kernels for.
int require_device();

// Let a kernel take all of an SM's shared memory and clusters of up to 16 CTAs
// (set once per kernel and device).
cudaError_t allow_large_cta(const void* fn);

inline bool is_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// B200: the persistent and split grids of the host planners are sized for it.
constexpr int kSmCount = 148;

}  // namespace dwb
