// Launcher interface of MXFP4 quantisation and product (implementation: mxfp4_launch.cu).
#pragma once

#include "host_common.h"

namespace beam {

size_t mxfp4_scales_bytes(int rows, int k);
int launch_mxfp4_quantize(const void* x, void* q, void* scales, int rows, int k, int bf16, cudaStream_t stream);
int launch_mxfp4_dequantize(const void* q, const void* scales, void* x, int rows, int k, int type, cudaStream_t stream);
int launch_mxfp4_gemmrc(const void* A, const void* a_scales, const void* B, const void* b_scales, void* C, int m, int n,
                        int k, int bf16, cudaStream_t stream);

}  // namespace beam
