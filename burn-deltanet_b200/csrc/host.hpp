// host.hpp — what the C entry points of the library's translation units share on the host side (defined in
// deltacore.cu, which holds the thread's last CUDA error and the per-device facts).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/deltacore.h"

namespace dc {
namespace host {

int cuda_fail(cudaError_t e);   // records `e` for dc_last_cuda_error and returns DC_ECUDA
int check_device();             // DC_OK on an sm_100 device
int sm_count();                 // multiprocessors of the current device

inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }
inline bool valid_dtype(int32_t t) { return t == DC_F32 || t == DC_BF16; }
inline size_t dtype_size(int32_t t) { return t == DC_F32 ? 4 : 2; }
inline int launched() {  // the status of the launch just made
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? DC_OK : cuda_fail(e);
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const char *x = static_cast<const char *>(a), *y = static_cast<const char *>(b);
    return x && y && x < y + nb && y < x + na;
}

}  // namespace host
}  // namespace dc
