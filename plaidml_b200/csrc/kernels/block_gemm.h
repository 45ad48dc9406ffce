// Products of 8-bit floats with a scale for each block of 128 terms (block_gemm.cu).
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "pmlb_kernels.h"

namespace pmlb {

// Returns 0, or a pmlb_status with a message in *err.  `status`: the device word that receives a code if a wait times out.
int block_gemm_launch(const pmlb_block_gemm_desc& d, const void* a, const float* a_scale, const void* b, const float* b_scale,
                      const int32_t* offsets, void* c, int* status, cudaStream_t stream, std::string* err);

}  // namespace pmlb
