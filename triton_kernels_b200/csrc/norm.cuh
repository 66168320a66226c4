// The LayerNorm with a learned scale and offset runs on the modulated form's kernels (bandwidth.cu) where rows are
// whole 16-byte pieces; layer_norm.cu has the others.
#pragma once

#include "common.cuh"

namespace fluxb {

// y = h * factor + offset; both given, one vector for all rows, everything 16-byte aligned, cols whole pieces.
int launch_layer_norm_affine(const void* x, const void* factor, const void* offset, void* y, float* mean, float* rstd,
                             int64_t rows, int64_t cols, int64_t x_ld, int64_t y_ld, float eps, int dtype, cudaStream_t st);

}  // namespace fluxb
