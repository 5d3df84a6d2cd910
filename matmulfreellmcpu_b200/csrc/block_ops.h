// block_ops.h -- argument blocks and launch wrappers of the recurrent-block operators
// (norm_quant.cu, int4_matvec.cu, selective.cu).
#pragma once

#include <cuda_runtime.h>

#include <atomic>
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

// The errors (kErrRange) of causal_conv and selective_scan (sequence starts and slots) and of
// int4_matvec (zero points) since the last call, read on `s` (synchronizing it) and cleared; 0
// when no such kernel was launched on this device.
cudaError_t take_sequence_flags(cudaStream_t s, uint32_t* flags);
cudaError_t take_zero_point_flags(cudaStream_t s, uint32_t* flags);

// The devices on which a file's kernels were launched.
class LaunchedOn {
 public:
  void mark() {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) bits_.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  }
  bool has(int dev) const { return bits_.load(std::memory_order_relaxed) >> (dev & 63) & 1; }

 private:
  std::atomic<uint64_t> bits_{0};
};

// Reads and clears a __device__ error word of the calling device on `s`, synchronizing it.
inline cudaError_t take_word(uint32_t& symbol, const LaunchedOn& devices, cudaStream_t s, uint32_t* flags) {
  *flags = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || !devices.has(dev)) return e;
  e = cudaMemcpyFromSymbolAsync(flags, symbol, 4, 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess || !*flags) return e;
  const uint32_t zero = 0;
  e = cudaMemcpyToSymbolAsync(symbol, &zero, 4, 0, cudaMemcpyHostToDevice, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

cudaError_t launch_causal_conv(const mmfree_cuda_conv_args& a, cudaStream_t s);
cudaError_t launch_causal_conv_step(const mmfree_cuda_conv_args& a, cudaStream_t s);
cudaError_t launch_selective_scan(const mmfree_cuda_ssm_args& a, int sm_count, cudaStream_t s);
cudaError_t launch_selective_step(const mmfree_cuda_ssm_args& a, cudaStream_t s);

}  // namespace mmfree_cuda
