// Quantisation to 8-bit floats by blocks of 128 (quant.cu).
#pragma once

#include <cuda_runtime.h>

#include "pmlb_kernels.h"

namespace pmlb {

cudaError_t launch_quant(const pmlb_quant_desc& d, const void* x, const int32_t* rows, void* q, float* scale, cudaStream_t stream);

}  // namespace pmlb
