// int4_matvec.cu -- products of a few rows with 4-bit weights that have a scale (and a zero
// point) for each group of columns.
//
//   out[m, n] = xs[m] * sum_g s[n, g] * sum_{k in g} (u[n, k] - z[n, g]) * x[m, k]
#include "block_ops.h"
#include "common.cuh"
#include "elements.cuh"

#include <cuda_fp8.h>

namespace mmfree_cuda {

namespace {

__device__ __forceinline__ float x_value(const void* x, int type, int64_t i) {
  switch (type) {
    case MMFREE_T_F32: return static_cast<const float*>(x)[i];
    case MMFREE_T_BF16: return to_f32(static_cast<const __nv_bfloat16*>(x)[i]);
    case MMFREE_T_F16: return to_f32(static_cast<const __half*>(x)[i]);
    case MMFREE_T_S8: return static_cast<float>(static_cast<const int8_t*>(x)[i]);
    default: {
      const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(x)[i], __NV_E4M3);
      return __half2float(__half(h));
    }
  }
}

__device__ __forceinline__ float scale_value(const void* p, int type, int64_t i) {
  switch (type) {
    case MMFREE_T_F32: return static_cast<const float*>(p)[i];
    case MMFREE_T_BF16: return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
    default: return to_f32(static_cast<const __half*>(p)[i]);
  }
}

__device__ __forceinline__ void put_out(void* p, int type, int64_t i, float v) {
  switch (type) {
    case MMFREE_T_F32: static_cast<float*>(p)[i] = v; break;
    case MMFREE_T_BF16: static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v); break;
    default: static_cast<__half*>(p)[i] = from_f32<__half>(v); break;
  }
}

// One warp per (weight row, activation row), lanes along the columns of each group.
__global__ void __launch_bounds__(256) int4_simple_kernel(Int4Args a) {
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), m = blockIdx.y, lane = threadIdx.x & 31;
  if (n >= a.N) return;
  float acc = 0.0f;
  for (int g = 0; g < a.parts; ++g) {
    const int64_t at = static_cast<int64_t>(n) * a.parts + g;
    const float z = a.zeros ? static_cast<float>(a.zeros[at]) : 8.0f;
    const int end = min(a.K, (g + 1) * a.group);
    float part = 0.0f;
    for (int k = g * a.group + lane; k < end; k += 32) {
      const int u = a.codes[n * a.ldw + (k >> 1)] >> (4 * (k & 1)) & 15;
      part = fmaf(static_cast<float>(u) - z, x_value(a.x, a.x_type, m * a.ldx + k), part);
    }
    float s = scale_value(a.scales, a.scale_type, at);
    if (a.x_grouped) s *= a.x_scales[static_cast<int64_t>(m) * a.parts + g];
    acc = fmaf(s, part, acc);
  }
  for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
  if (lane == 0) {
    if (a.x_scales && !a.x_grouped) acc *= a.x_scales[m];
    put_out(a.out, a.out_type, static_cast<int64_t>(m) * a.N + n, acc);
  }
}

}  // namespace

cudaError_t launch_int4_matvec(const Int4Args& a, int sm_count, cudaStream_t s) {
  (void)sm_count;
  for (int m0 = 0; m0 < a.M; m0 += 32768) {  // grid.y is 16 bits
    Int4Args b = a;
    const int xs = a.x_type == MMFREE_T_F32 ? 4 : a.x_type >= MMFREE_T_S8 ? 1 : 2;
    b.M = a.M - m0 < 32768 ? a.M - m0 : 32768;
    b.x = static_cast<const char*>(a.x) + m0 * a.ldx * xs;
    if (a.x_scales) b.x_scales = a.x_scales + static_cast<int64_t>(m0) * (a.x_grouped ? a.parts : 1);
    b.out = static_cast<char*>(a.out) + static_cast<int64_t>(m0) * a.N * (a.out_type == MMFREE_T_F32 ? 4 : 2);
    const cudaError_t e = launch_k(int4_simple_kernel, dim3(static_cast<unsigned>(ceil_div(a.N, 8)), b.M), dim3(256), 0, s, false, b);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mmfree_cuda
