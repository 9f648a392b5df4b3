// Launcher interface of the gated product and of the gradients of rc products (implementation: feedforward_launch.cu).
#pragma once

#include "host_common.h"

namespace beam {

int launch_gated(const void* A, const void* Bg, const void* Bu, void* C, void* G, void* U, int m, int f, int k,
                 int activation, int bf16, cudaStream_t stream);
size_t gated_backward_workspace_bytes(int m, int f, int k);
size_t gemmrc_backward_workspace_bytes(int m, int n, int k);
int launch_gated_backward(const void* dC, const void* A, const void* Bg, const void* Bu, const void* G, const void* U,
                          void* dA, void* dBg, void* dBu, int m, int f, int k, int activation, int bf16,
                          void* workspace, size_t workspace_bytes, cudaStream_t stream);
int launch_gemmrc_backward(const void* dC, const void* A, const void* B, void* dA, void* dB, int m, int n, int k,
                           int bf16, void* workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace beam
