// What the units of the operators in 8 bits and of experts have of one another.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace atma {
// Reads and clears the status word of the products in 8 bits (non-zero: a bounded wait ran out).
int linear_fp8_status_fetch_and_clear(int* out);

// atma_combine_experts; wide: y is fp32 whatever dtype is.
int combine_experts(const void* y, bool wide, const int32_t* place, const float* weights, const void* add, void* out, int rows, int copies, int D,
                    int dtype, cudaStream_t st);
}
