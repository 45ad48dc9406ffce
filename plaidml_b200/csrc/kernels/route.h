// Routing of tokens to experts: choice, weights, the experts' order of rows, gradient (route.cu).
#pragma once

#include <cuda_runtime.h>

#include "pmlb_kernels.h"

namespace pmlb {

// The choice and, where the descriptor has rows, the order.
cudaError_t launch_route(const pmlb_route_desc& d, const void* logits, const float* bias, float* weights, int32_t* ids,
                         int32_t* offsets, int32_t* source, int32_t* position, cudaStream_t stream);
cudaError_t launch_route_order(const pmlb_route_desc& d, const int32_t* ids, int32_t* offsets, int32_t* source, int32_t* position,
                               cudaStream_t stream);
cudaError_t launch_route_grad(const pmlb_route_desc& d, const void* logits, const int32_t* ids, const float* dweights, void* dlogits,
                              cudaStream_t stream);

}  // namespace pmlb
