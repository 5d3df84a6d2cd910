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

// Eight columns as they lie in memory, whole or one by one.
template <typename T, bool kVec>
__device__ __forceinline__ void fetch8(const T* p, int n, Words<T, kCols>& w) {
  if constexpr (kVec) {
    w.load(p);
  } else {
    Pack<T, kCols> k;
#pragma unroll
    for (int i = 0; i < kCols; ++i) k.v[i] = i < n ? p[i] : from_f32<T>(0.0f);
    memcpy(&w.w, &k, sizeof(k));
  }
}

// Whether a row's mean of squares is a number that fp32 holds with all its bits.
__device__ __forceinline__ bool in_range(float mean) { return mean >= 0x1p-96f && mean <= 3.402823466e38f; }

// The scales of a CTA's rows once more, from sums and products in 64 bits, where the squares are outside fp32's range (values
// above 1.8e19, a NaN or an infinity) or so small that their rounding counts (without an eps). Behind the last row, where
// nothing else is live, and not inlined: in the rows' loop, which uses all its registers, it made calls 13 to 24% slower.
template <typename T>
__device__ __noinline__ void far_scales(const NormQuantArgs& a, float limit) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();  // the other threads' scales and parts of the residual
#pragma unroll 1
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const r = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : static_cast<const T*>(a.x) + row * a.ldx;
    double sum = 0.0;  // every warp sums the whole row
    for (int i = lane; i < a.cols; i += 32) sum += static_cast<double>(to_f32(r[i])) * to_f32(r[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const double mean = sum / a.cols + static_cast<double>(a.eps);
    // a wider range than in_range's: cols squares, 2^16 at most, may have been out of fp32's where their mean is not
    if (mean >= 0x1p-95 && mean <= 0x1p110) continue;
    const double rstd = 1.0 / sqrt(mean);
    const int group = a.group ? a.group : a.cols;
    for (int part = warp; part < a.parts; part += blockDim.x >> 5) {
      uint32_t most = 0;
      for (int i = part * group + lane; i < min((part + 1) * group, a.cols); i += 32)
        most = max(most, __float_as_uint(__fmul_rn(to_f32(r[i]), a.weight[i])) & 0x7FFFFFFFu);
      const double m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, most));
      if (lane == 0) a.scales[row * a.parts + part] = mean == 0.0 ? 0.0f : static_cast<float>(m * rstd / limit);
    }
  }
}

// A CTA holds a row in registers, kChunks chunks of 8 columns a thread, and walks the rows with a fixed stride; several
// small CTAs an SM cover each other's reductions. Two chunks a thread are the best for most rows: 16384 x 2560 bf16 to
// e4m3 (bound by the issue slots, 60 us, 4.9 TB/s) takes 78 us with one chunk and 75 us with four. Rows of one chunk a
// thread keep the weights, and where the registers allow it the next row is loaded while this one is reduced and stored
// (62.9 us without).
template <typename T, typename Code, int kChunks, bool kVec>
__global__ void __launch_bounds__(kChunks == 8 ? 896 : 512, kChunks == 8 ? 1 : 2) norm_quant_kernel(const __grid_constant__ NormQuantArgs a) {
  constexpr bool kAhead = kChunks * sizeof(T) <= 4, kKeep = kChunks == 1;
  constexpr bool kS8 = std::is_same<Code, int8_t>::value;
  constexpr float kLimit = kS8 ? 127.0f : 448.0f;
  __shared__ __align__(16) float s_sum[2][32];
  __shared__ __align__(16) uint32_t s_most[2][32];
  __shared__ int s_far;  // whether a row was not in range
  if (threadIdx.x == 0) s_far = 0;
  __syncthreads();
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5;
  const bool add = a.residual != nullptr;
  const int parts_shift = a.group ? __ffs(a.group) - 1 : 0;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  Words<T, kCols> next_x[kChunks], next_r[kChunks];
  const auto fetch = [&](int64_t row) {
    const T* const px = static_cast<const T*>(a.x) + row * a.ldx;
    const T* const pr = static_cast<const T*>(a.residual) + (add ? row * a.ldr : 0);
    // whole chunks without a branch between the loads: a thread behind the row's end reads its last chunk
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int at = (tid + c * static_cast<int>(blockDim.x)) * kCols, col = kVec ? min(at, a.cols - kCols) : at;
      fetch8<T, kVec>(px + col, a.cols - col, next_x[c]);
    }
    if (add)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int at = (tid + c * static_cast<int>(blockDim.x)) * kCols, col = kVec ? min(at, a.cols - kCols) : at;
        fetch8<T, kVec>(pr + col, a.cols - col, next_r[c]);
      }
  };
  float w[kCols];
  if constexpr (kKeep) {
    if (tid * kCols < a.cols) load_row<kVec>(a.weight + tid * kCols, a.cols - tid * kCols, w);
  }
  if constexpr (kAhead) fetch(blockIdx.x);
  int buf = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buf ^= 1) {
    if constexpr (!kAhead) fetch(row);
    float t[kChunks][kCols], sum = 0.0f;
    uint32_t most[kChunks];  // |t| as its bits: ordered like the values, a NaN above all
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (tid + c * static_cast<int>(blockDim.x)) * kCols, n = a.cols - col;
      most[c] = 0;
      if (n <= 0) continue;
#pragma unroll
      for (int i = 0; i < kCols; ++i) t[c][i] = next_x[c][i];
      if (add) {
        T* const to = static_cast<T*>(a.residual) + row * a.ldr + col;
#pragma unroll
        for (int i = 0; i < kCols; ++i) t[c][i] += next_r[c][i];
        if constexpr (sizeof(T) == 2) {  // rounded in pairs
          Pack<uint32_t, kCols / 2> words;
#pragma unroll
          for (int i = 0; i < kCols; i += 2) words.v[i / 2] = round2(t[c][i], t[c][i + 1], T{});
          if constexpr (kVec) *reinterpret_cast<Pack<uint32_t, kCols / 2>*>(to) = words;
          else store_row<false>(to, n, t[c]);
        } else {
          store_row<kVec>(to, n, t[c]);
        }
      }
      if constexpr (!kKeep) load_row<kVec>(a.weight + col, n, w);
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        sum = fmaf(t[c][i], t[c][i], sum);
        t[c][i] = __fmul_rn(t[c][i], w[i]);
        most[c] = max(most[c], __float_as_uint(t[c][i]) & 0x7FFFFFFFu);
      }
    }
    if constexpr (kAhead)
      if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
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
      if (lane == 0) {
        s_sum[buf][tid >> 5] = sum;
        s_most[buf][tid >> 5] = row_most;
      }
      __syncthreads();  // one a row: the next row's partials go to the other half
      // every thread sums the warps' partials, in the same order
      sum = 0.0f;
      for (int i = 0; i < warps; ++i) sum += s_sum[buf][i];
      if (a.group == 0) {
        row_most = 0;
        for (int i = 0; i < warps; ++i) row_most = max(row_most, s_most[buf][i]);
      }
    }
    const float mean = fmaf(sum, inv_cols, a.eps);
    const float rstd = rsqrtf(mean);
    if (!in_range(mean)) s_far = 1;
    float* const scales = a.scales + row * a.parts;
    if (a.group == 0 && tid == 0) scales[0] = __uint_as_float(row_most) * rstd * (1.0f / kLimit);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (tid + c * static_cast<int>(blockDim.x)) * kCols, n = a.cols - col;
      if (n <= 0) continue;
      const float m = __uint_as_float(a.group ? most[c] : row_most);
      if (a.group && (col & (a.group - 1)) == 0) scales[col >> parts_shift] = m * rstd * (1.0f / kLimit);
      const float inv = kLimit / m;
      Pack<uint8_t, kCols> q;
      if constexpr (kS8) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) q.v[i] = static_cast<uint8_t>(code_s8(t[c][i], inv, m));
      } else {
        if (inv < __int_as_float(0x7F800000)) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) t[c][i] *= inv;
        } else {  // m is 0, too small for its reciprocal, or a NaN
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            t[c][i] = m == 0.0f ? 0.0f : static_cast<float>(static_cast<double>(t[c][i]) * 448.0 / static_cast<double>(m));
        }
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
          const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(t[c][i], t[c][i + 1]), __NV_SATFINITE, __NV_E4M3);
          q.v[i] = static_cast<uint8_t>(two);
          q.v[i + 1] = static_cast<uint8_t>(two >> 8);
        }
      }
      uint8_t* const codes = static_cast<uint8_t*>(a.codes) + row * a.cols + col;
      if constexpr (kVec) {
        *reinterpret_cast<Pack<uint8_t, kCols>*>(codes) = q;
      } else {
#pragma unroll
        for (int i = 0; i < kCols; ++i)
          if (i < n) codes[i] = q.v[i];
      }
    }
  }
  __syncthreads();
  if (s_far) far_scales<T>(a, kLimit);
}

template <typename T, typename Code, int kChunks, bool kVec>
cudaError_t launch_chunks(const NormQuantArgs& a, int threads, cudaStream_t s) {
  // as many CTAs as the SMs hold at once, each with its share of the rows
  const auto kernel = norm_quant_kernel<T, Code, kChunks, kVec>;
  int64_t grid = a.rows;
  if (grid > 148) {
    int dev = 0, sms = 0, held = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, threads, 0);
    if (e != cudaSuccess) return e;
    if (grid > static_cast<int64_t>(sms) * held) grid = static_cast<int64_t>(sms) * held;
  }
  return launch_k(kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, s, false, a);
}

template <typename T, typename Code, bool kVec>
cudaError_t launch_cols(const NormQuantArgs& a, cudaStream_t s) {
  const int chunks = static_cast<int>(ceil_div(a.cols, kCols));
  // a thread holds 1 to 8 chunks of the row in registers
  const int per = chunks <= 128 ? 1 : chunks <= 1024 ? 2 : chunks <= 2048 ? 4 : 8;
  const int threads = static_cast<int>(ceil_div(ceil_div(chunks, per), 32) * 32);
  switch (per) {
    case 1: return launch_chunks<T, Code, 1, kVec>(a, threads, s);
    case 2: return launch_chunks<T, Code, 2, kVec>(a, threads, s);
    case 4: return launch_chunks<T, Code, 4, kVec>(a, threads, s);
    default: return launch_chunks<T, Code, 8, kVec>(a, threads, s);
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
