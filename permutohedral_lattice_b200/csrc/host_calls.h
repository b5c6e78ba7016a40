// What the host sides of the translation units share: errors, launch counter, shared-memory limits.
#pragma once
#include <cuda_runtime.h>
#include "../../include/pl_lattice.h"
#include "smem_limit.h"

namespace pl {

int cuda_fail(cudaError_t e, const char* where);   // keeps the text for pl_last_cuda_error; returns PL_CUDA_ERROR
void count_launches(int n);
int num_sms();

#define PL_COUNT_LAUNCHES(n) count_launches(n)
#define PL_CUDA(call)                                   \
    do {                                                \
        cudaError_t e_ = (call);                        \
        if (e_ != cudaSuccess) return cuda_fail(e_, #call); \
    } while (0)

#define PL_TRY(call)                     \
    do {                                 \
        const int rc_ = (call);          \
        if (rc_ != PL_OK) return rc_;    \
    } while (0)

// Raises a kernel's dynamic shared-memory limit (and sets its carve-out preference) when this call needs more than any
// call before it on the current device.
template <auto Kernel>
static int ensure_dynamic_smem(size_t bytes, bool max_carveout = false) {
    static SmemLimit limit;
    int dev = -1;
    PL_CUDA(cudaGetDevice(&dev));
    return limit.raise(dev, bytes, [&](size_t n) -> int {
        PL_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)n));
        if (max_carveout)
            PL_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                         cudaSharedmemCarveoutMaxShared));
        return PL_OK;
    });
}

}  // namespace pl
