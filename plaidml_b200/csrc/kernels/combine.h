// Weighted sums of the experts' rows of each token, and their gradients (combine.cu).
#pragma once

#include <cuda_runtime.h>

#include "pmlb_kernels.h"

namespace pmlb {

cudaError_t launch_combine(const pmlb_combine_desc& d, const void* y, const float* weights, const int32_t* position, void* out,
                           cudaStream_t stream);
cudaError_t launch_combine_grad(const pmlb_combine_desc& d, const void* dout, const void* y, const float* weights,
                                const int32_t* position, const int32_t* source, void* dy, float* dweights, cudaStream_t stream);

}  // namespace pmlb
