// norm_quant.cu -- the residual's addition, its RMS norm and an 8-bit output with scales in
// one pass.
//
//   r = round(residual + x); t = fl32(r * w); m = max |t| over a row or a group of columns
//   int8: code = rne(127 t / m);  e4m3: code = e4m3(t * (448 / m));  scale = m * rstd / limit
//
// The codes are a ratio of two values of the same row, so the norm's factor rstd cancels in
// them and enters the scale alone: the sum of squares and the maximum come from ONE reduction
// (a norm followed by a quantisation needs two, the second waiting for the first).
#include "block_ops.h"
#include "common.cuh"
#include "elements.cuh"

#include <cuda_fp8.h>

namespace mmfree_cuda {

namespace {

constexpr int kCols = 8;  // columns of a thread's chunk

// One int8 code: the exact quotient 127 t / m rounded half to even. The fp32 product t * inv
// is off by less than 127 * 2 * 2^-24 < 2e-5, so unless it lies within 1e-4 of a border
// between two codes it rounds as the exact quotient does; near a border (and where inv is
// not finite) the quotient is taken in 64 bits. A NaN (0 / 0, inf / inf) becomes 0.
__device__ __forceinline__ int code_s8(float t, float inv, float m) {
  const float p = t * inv;
  const float c = rintf(p);
  if (fabsf(p - c) <= 0.4999f) return static_cast<int>(c);
  const double e = rint(static_cast<double>(t) * 127.0 / static_cast<double>(m));
  return e == e ? static_cast<int>(e) : 0;
}

template <typename T, typename Code, int kChunks, bool kVec>
__global__ void __launch_bounds__(1024) norm_quant_kernel(NormQuantArgs a) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  T* res = a.residual ? static_cast<T*>(a.residual) + row * a.ldr : nullptr;
  Code* codes = static_cast<Code*>(a.codes) + row * a.cols;
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5;
  float t[kChunks][kCols];
  float sum = 0.0f;
  uint32_t most[kChunks];  // |t| as its bits: ordered like the values, a NaN above all
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (tid + c * static_cast<int>(blockDim.x)) * kCols;
    const int n = a.cols - col;
    most[c] = 0;
    if (n <= 0) continue;
    load_row<kVec>(x + col, n, t[c]);
    if (res) {
      float r[kCols];
      load_row<kVec>(res + col, n, r);
#pragma unroll
      for (int i = 0; i < kCols; ++i) t[c][i] = to_f32(from_f32<T>(r[i] + t[c][i]));
      store_row<kVec>(res + col, n, t[c]);
    }
    float w[kCols];
    load_row<kVec>(a.weight + col, n, w);
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      sum = fmaf(t[c][i], t[c][i], sum);
      t[c][i] = __fmul_rn(t[c][i], w[i]);
      most[c] = max(most[c], __float_as_uint(t[c][i]) & 0x7FFFFFFFu);
    }
  }
  uint32_t row_most = 0;
  if (a.group == 0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) row_most = max(row_most, most[c]);
    row_most = __reduce_max_sync(0xFFFFFFFFu, row_most);
  } else {
    // a group is 4, 8 or 16 neighbouring lanes' chunks
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      most[c] = max(most[c], __shfl_xor_sync(0xFFFFFFFFu, most[c], 1));
      most[c] = max(most[c], __shfl_xor_sync(0xFFFFFFFFu, most[c], 2));
      if (a.group >= 64) most[c] = max(most[c], __shfl_xor_sync(0xFFFFFFFFu, most[c], 4));
      if (a.group >= 128) most[c] = max(most[c], __shfl_xor_sync(0xFFFFFFFFu, most[c], 8));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (warps > 1) {
    __shared__ float s_sum[32];
    __shared__ uint32_t s_most[32];
    if (lane == 0) {
      s_sum[tid >> 5] = sum;
      s_most[tid >> 5] = row_most;
    }
    __syncthreads();
    // every warp sums all partials in the same order
    sum = lane < warps ? s_sum[lane] : 0.0f;
    row_most = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? s_most[lane] : 0u);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  }
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(a.cols) + a.eps);
  constexpr bool kS8 = sizeof(Code) == 1 && std::is_same<Code, int8_t>::value;
  constexpr float kLimit = kS8 ? 127.0f : 448.0f;
  float* scales = a.scales + row * a.parts;
  if (a.group == 0 && tid == 0) scales[0] = __uint_as_float(row_most) * rstd / kLimit;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (tid + c * static_cast<int>(blockDim.x)) * kCols;
    const int n = a.cols - col;
    if (n <= 0) continue;
    const float m = __uint_as_float(a.group ? most[c] : row_most);
    if (a.group && (col % a.group) == 0) scales[col / a.group] = m * rstd / kLimit;
    const float inv = kLimit / m;
    Pack<uint8_t, kCols> q;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      if constexpr (kS8) {
        q.v[i] = static_cast<uint8_t>(code_s8(t[c][i], inv, m));
      } else {
        float v = t[c][i] * inv;
        if (!(inv < __int_as_float(0x7F800000)))  // m is 0, too small for its reciprocal, or a NaN
          v = m == 0.0f ? 0.0f : static_cast<float>(static_cast<double>(t[c][i]) * 448.0 / static_cast<double>(m));
        q.v[i] = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
      }
    }
    if constexpr (kVec) {
      *reinterpret_cast<Pack<uint8_t, kCols>*>(codes + col) = q;
    } else {
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < n) reinterpret_cast<uint8_t*>(codes)[col + i] = q.v[i];
    }
  }
}

template <typename T, typename Code, bool kVec>
cudaError_t launch_cols(const NormQuantArgs& a, cudaStream_t s) {
  const int chunks = static_cast<int>(ceil_div(a.cols, kCols));
  // a thread holds 1 to 8 chunks of the row in registers
  const int per = chunks <= 256 ? 1 : chunks <= 1024 ? 2 : chunks <= 4096 ? 4 : 8;
  const int threads = static_cast<int>(ceil_div(ceil_div(chunks, per), 32) * 32);
  const dim3 grid(static_cast<unsigned>(a.rows));
  switch (per) {
    case 1: return launch_k(norm_quant_kernel<T, Code, 1, kVec>, grid, dim3(threads), 0, s, false, a);
    case 2: return launch_k(norm_quant_kernel<T, Code, 2, kVec>, grid, dim3(threads), 0, s, false, a);
    case 4: return launch_k(norm_quant_kernel<T, Code, 4, kVec>, grid, dim3(threads), 0, s, false, a);
    default: return launch_k(norm_quant_kernel<T, Code, 8, kVec>, grid, dim3(threads), 0, s, false, a);
  }
}

template <typename T>
cudaError_t launch_type(const NormQuantArgs& a, cudaStream_t s) {
  const bool vec = a.cols % kCols == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) &&
                   (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0 && a.ldx * sizeof(T) % 16 == 0 &&
                   (!a.residual || a.ldr * sizeof(T) % 16 == 0);
  if (a.code_type == MMFREE_T_S8)
    return vec ? launch_cols<T, int8_t, true>(a, s) : launch_cols<T, int8_t, false>(a, s);
  return vec ? launch_cols<T, __nv_fp8_storage_t, true>(a, s) : launch_cols<T, __nv_fp8_storage_t, false>(a, s);
}

}  // namespace

cudaError_t launch_norm_quant(const NormQuantArgs& a, cudaStream_t s) {
  switch (a.type) {
    case MMFREE_T_F32: return launch_type<float>(a, s);
    case MMFREE_T_BF16: return launch_type<__nv_bfloat16>(a, s);
    default: return launch_type<__half>(a, s);
  }
}

}  // namespace mmfree_cuda
