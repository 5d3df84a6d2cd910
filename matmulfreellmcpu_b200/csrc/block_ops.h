// block_ops.h -- argument blocks and launch wrappers of the recurrent-block operators
// (norm_quant.cu, int4_matvec.cu, selective.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/mmfree_cuda.h"

namespace mmfree_cuda {

struct NormQuantArgs {
  void* codes;          // [rows, cols]
  float* scales;        // [rows, parts]
  const void* x;        // [rows, ldx]
  void* residual;       // [rows, ldr] (nullable)
  const float* weight;  // [cols]
  int64_t rows, ldx, ldr;
  int cols, group, parts;
  float eps;
  int type, code_type;
};
cudaError_t launch_norm_quant(const NormQuantArgs& a, cudaStream_t s);

struct Int4Args {
  void* out;              // [M, N]
  const void* x;          // [M, ldx]
  const float* x_scales;  // [M] or [M, parts] (8-bit rows only)
  const uint8_t* codes;   // [N, ldw] bytes
  const void* scales;     // [N, parts]
  const uint8_t* zeros;   // [N, parts] (nullable: 8)
  int64_t ldx, ldw;
  int M, N, K, group, parts;
  bool x_grouped;         // x_scales per group of columns
  int x_type, scale_type, out_type;
};
cudaError_t launch_int4_matvec(const Int4Args& a, int sm_count, cudaStream_t s);

// The sequence errors of causal_conv and selective_scan (kErrRange) since the last call, read
// on `s` (synchronizing it) and cleared; 0 when no such kernel was launched on this device.
cudaError_t take_sequence_flags(cudaStream_t s, uint32_t* flags);

cudaError_t launch_causal_conv(const mmfree_cuda_conv_args& a, cudaStream_t s);
cudaError_t launch_causal_conv_step(const mmfree_cuda_conv_args& a, cudaStream_t s);
cudaError_t launch_selective_scan(const mmfree_cuda_ssm_args& a, int sm_count, cudaStream_t s);
cudaError_t launch_selective_step(const mmfree_cuda_ssm_args& a, cudaStream_t s);

}  // namespace mmfree_cuda
