// selective.cu -- the short causal convolution and the selective state space scan of packed
// sequences, and both for single tokens.
//
//   conv:  out[t, d] = act(bias[d] + sum_j w[d, j] * in[t - (W - 1) + j, d])
//   scan:  h = exp(delta * A) * h + delta * x * B;  out = (C . h + D * x) * z * sigmoid(z)
//
// States are fp32 in the scan; a convolution's state holds inputs, in the inputs' type.
#include "block_ops.h"
#include "common.cuh"
#include "elements.cuh"

#include <atomic>

namespace mmfree_cuda {

// Bit kErrRange once a sequence start or a slot broke its rules.
__device__ uint32_t g_sequence_error;

namespace {

std::atomic<uint64_t> g_devices{0};  // devices on which one of these kernels was launched

void mark_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) g_devices.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
}

__device__ __forceinline__ void sequence_error() { atomicOr(&g_sequence_error, kErrRange); }

// Rows [b, e) of sequence s; false (and an error) where they are not ascending rows of the call.
__device__ __forceinline__ bool sequence_rows(const int32_t* starts, int64_t tokens, int64_t s, int64_t& b, int64_t& e) {
  b = starts ? starts[s] : 0;
  e = starts ? starts[s + 1] : tokens;
  if (b >= 0 && b <= e && e <= tokens) return true;
  sequence_error();
  return false;
}

// The state of sequence s, or -1: a padded one, or (an error) a slot outside the pool.
__device__ __forceinline__ int64_t sequence_slot(const int32_t* slots, int64_t count, int64_t s) {
  const int64_t at = slots ? slots[s] : s;
  if (at < count) return at < 0 ? -1 : at;
  sequence_error();
  return -1;
}

// ---- causal convolution ----------------------------------------------------------------------

template <int W, int V>
__device__ __forceinline__ void conv_load_taps(const mmfree_cuda_conv_args& a, int64_t d, float (&w)[V][W], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[i][j] = a.weight[(d + i) * W + j];
    bias[i] = a.bias ? a.bias[d + i] : 0.0f;
  }
}

// in: the window's W - 1 older inputs, then the newest; returns the output of each channel.
template <int W, int V>
__device__ __forceinline__ void conv_token(const float (&win)[W - 1][V], const float (&x)[V], const float (&w)[V][W],
                                           const float (&bias)[V], bool silu, float (&y)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float s = bias[i];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) s = fmaf(w[i][j], win[j][i], s);
    s = fmaf(w[i][W - 1], x[i], s);
    y[i] = silu ? silu_f32(s) : s;
  }
}

template <int W, int V>
__device__ __forceinline__ void conv_shift(float (&win)[W - 1][V], const float (&x)[V]) {
#pragma unroll
  for (int j = 0; j + 1 < W - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
#pragma unroll
  for (int i = 0; i < V; ++i) win[W - 2][i] = x[i];
}

// A CTA owns a tile of `rows` tokens for a block of channels. The tile in which a sequence
// begins reads that sequence's old state, writes the new one, and computes every token whose
// window still reaches into the old state, even those behind the tile's end, which the tiles
// there leave out: no other CTA reads a state that this one overwrites.
template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_kernel(mmfree_cuda_conv_args a, int rows) {
  constexpr bool kVec = V > 1;
  const int64_t d = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  if (d >= static_cast<int64_t>(a.channels)) return;
  const int64_t tokens = static_cast<int64_t>(a.tokens), seqs = static_cast<int64_t>(a.seqs);
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * rows, t1 = min(t0 + rows, tokens);
  const T* x = static_cast<const T*>(a.x) + d;
  T* out = static_cast<T*>(a.out) + d;
  const int64_t ldx = static_cast<int64_t>(a.ldx), ldo = static_cast<int64_t>(a.ld_out);
  const bool silu = a.silu != 0;
  // the last sequence that begins at or before t0
  int64_t seq = 0;
  if (a.seq_starts) {
    int64_t lo = 0, hi = seqs;  // starts[lo - 1] <= t0 < starts[hi]
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (a.seq_starts[mid] <= t0) lo = mid + 1; else hi = mid;
    }
    seq = lo > 0 ? lo - 1 : 0;
  }
  float w[V][W], bias[V];
  conv_load_taps<W, V>(a, d, w, bias);
  for (; seq < seqs; ++seq) {
    int64_t b, e;
    if (!sequence_rows(a.seq_starts, tokens, seq, b, e)) continue;
    if (b >= t1) break;
    if (e <= t0 || b == e) continue;
    const int64_t slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), seq);
    if (slot < 0) continue;
    float win[W - 1][V];
    int64_t t, stop;
    if (b >= t0) {
      T* st = a.state ? static_cast<T*>(a.state) + (slot * (W - 1)) * static_cast<int64_t>(a.channels) + d : nullptr;
      const int64_t pitch = static_cast<int64_t>(a.channels);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (st) load_row<kVec>(st + j * pitch, V, win[j]);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) win[j][i] = 0.0f;
      }
      if (st) {
        const int64_t len = e - b;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          // input number len + j of the sequence with its old state in front
          const int64_t k = len + j;
          float v[V];
          if (k >= W - 1) {
            load_row<kVec>(x + (b + k - (W - 1)) * ldx, V, v);
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = 0.0f;
#pragma unroll
            for (int q = 0; q < W - 1; ++q)
              if (q == k)
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = win[q][i];
          }
          store_row<kVec>(st + j * pitch, V, v);
        }
      }
      t = b;
      stop = min(e, max(t1, b + W - 1));
    } else {
      t = max(t0, b + W - 1);
      stop = min(e, t1);
      if (t >= stop) continue;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) load_row<kVec>(x + (t - (W - 1) + j) * ldx, V, win[j]);
    }
    for (; t < stop; ++t) {
      float v[V], y[V];
      load_row<kVec>(x + t * ldx, V, v);
      conv_token<W, V>(win, v, w, bias, silu, y);
      store_row<kVec>(out + t * ldo, V, y);
      conv_shift<W, V>(win, v);
    }
  }
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(mmfree_cuda_conv_args a) {
  constexpr bool kVec = V > 1;
  const int64_t d = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  if (d >= static_cast<int64_t>(a.channels)) return;
  const int64_t s = blockIdx.y, slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), s);
  if (slot < 0) return;
  const int64_t pitch = static_cast<int64_t>(a.channels);
  T* st = a.state ? static_cast<T*>(a.state) + (slot * (W - 1)) * pitch + d : nullptr;
  float win[W - 1][V], v[V], y[V], w[V][W], bias[V];
  load_row<kVec>(static_cast<const T*>(a.x) + s * static_cast<int64_t>(a.ldx) + d, V, v);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    if (st) load_row<kVec>(st + j * pitch, V, win[j]);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = 0.0f;
  }
  conv_load_taps<W, V>(a, d, w, bias);
  conv_token<W, V>(win, v, w, bias, a.silu != 0, y);
  store_row<kVec>(static_cast<T*>(a.out) + s * static_cast<int64_t>(a.ld_out) + d, V, y);
  conv_shift<W, V>(win, v);
  if (st)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<kVec>(st + j * pitch, V, win[j]);
}

template <typename T, int W, int V>
cudaError_t conv_launch(const mmfree_cuda_conv_args& a, bool step, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.channels), 128 * V));
  mark_device();
  if (step) return launch_k(conv_step_kernel<T, W, V>, dim3(blocks, static_cast<unsigned>(a.seqs)), dim3(128), 0, s, false, a);
  int rows = 32;
  while (ceil_div(static_cast<int64_t>(a.tokens), rows) > 65535) rows *= 2;  // grid.y is 16 bits
  const unsigned tiles = static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.tokens), rows));
  return launch_k(conv_kernel<T, W, V>, dim3(blocks, tiles), dim3(128), 0, s, false, a, rows);
}

template <typename T, int V>
cudaError_t conv_width(const mmfree_cuda_conv_args& a, bool step, cudaStream_t s) {
  switch (a.width) {
    case 2: return conv_launch<T, 2, V>(a, step, s);
    case 3: return conv_launch<T, 3, V>(a, step, s);
    case 4: return conv_launch<T, 4, V>(a, step, s);
    // the wider ones hold more taps per channel: one channel per thread
    case 5: return conv_launch<T, 5, 1>(a, step, s);
    case 6: return conv_launch<T, 6, 1>(a, step, s);
    case 7: return conv_launch<T, 7, 1>(a, step, s);
    default: return conv_launch<T, 8, 1>(a, step, s);
  }
}

template <typename T>
cudaError_t conv_type(const mmfree_cuda_conv_args& a, bool step, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);  // channels of a 16-byte access
  const bool vec = a.channels % V == 0 && a.ldx % V == 0 && a.ld_out % V == 0 && aligned16(a.x) && aligned16(a.out) &&
                   aligned16(a.state);
  return vec ? conv_width<T, V>(a, step, s) : conv_width<T, 1>(a, step, s);
}

cudaError_t conv_any(const mmfree_cuda_conv_args& a, bool step, cudaStream_t s) {
  switch (a.type) {
    case MMFREE_T_F32: return conv_type<float>(a, step, s);
    case MMFREE_T_BF16: return conv_type<__nv_bfloat16>(a, step, s);
    default: return conv_type<__half>(a, step, s);
  }
}

// ---- selective scan --------------------------------------------------------------------------

__device__ __forceinline__ float softplus_f32(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

constexpr int kMaxPerLane = MMFREE_CUDA_MAX_STATES / 32;

// `lanes` lanes (a power of two) per (sequence, channel), each holding every lanes-th state.
template <typename T>
__global__ void __launch_bounds__(128) ssm_kernel(mmfree_cuda_ssm_args a, int lanes, bool step) {
  const int64_t channels = static_cast<int64_t>(a.channels), states = static_cast<int64_t>(a.states);
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t d = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes;
  const bool live = d < channels;
  const int64_t dd = live ? d : channels - 1, seq = blockIdx.y;
  int64_t b = seq, e = seq + 1;
  if (!step && !sequence_rows(a.seq_starts, static_cast<int64_t>(a.tokens), seq, b, e)) return;
  if (b == e) return;
  const int64_t slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), seq);
  if (slot < 0) return;
  float* state = a.state ? a.state + (slot * channels + dd) * states : nullptr;
  float h[kMaxPerLane], rate[kMaxPerLane];
#pragma unroll
  for (int j = 0; j < kMaxPerLane; ++j) {
    const int64_t n = lane + j * lanes;
    const bool in = n < states;
    h[j] = in && state ? state[n] : 0.0f;
    rate[j] = in ? a.A[dd * states + n] : 0.0f;
  }
  const int64_t group = dd / (channels / static_cast<int64_t>(a.groups));
  const float skip = a.D ? a.D[dd] : 0.0f, bias = a.dt_bias ? a.dt_bias[dd] : 0.0f;
  for (int64_t t = b; t < e; ++t) {
    const float x = to_f32(static_cast<const T*>(a.x)[t * static_cast<int64_t>(a.ldx) + dd]);
    float delta = to_f32(static_cast<const T*>(a.dt)[t * static_cast<int64_t>(a.ld_dt) + dd]) + bias;
    if (a.dt_softplus) delta = softplus_f32(delta);
    const T* B = static_cast<const T*>(a.B) + t * static_cast<int64_t>(a.ldb) + group * states;
    const T* C = static_cast<const T*>(a.C) + t * static_cast<int64_t>(a.ldc) + group * states;
    float y = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxPerLane; ++j) {
      const int64_t n = lane + j * lanes;
      if (n < states) {
        h[j] = fmaf(expf(delta * rate[j]), h[j], delta * x * to_f32(B[n]));
        y = fmaf(to_f32(C[n]), h[j], y);
      }
    }
    for (int o = lanes >> 1; o; o >>= 1) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
    y = fmaf(skip, x, y);
    if (a.z) y *= silu_f32(to_f32(static_cast<const T*>(a.z)[t * static_cast<int64_t>(a.ldz) + dd]));
    if (live && lane == 0) static_cast<T*>(a.out)[t * static_cast<int64_t>(a.ld_out) + dd] = from_f32<T>(y);
  }
  if (state && live)
#pragma unroll
    for (int j = 0; j < kMaxPerLane; ++j)
      if (lane + j * lanes < states) state[lane + j * lanes] = h[j];
}

cudaError_t ssm_any(const mmfree_cuda_ssm_args& a, bool step, cudaStream_t s) {
  int lanes = 1;
  while (lanes < 32 && lanes < static_cast<int>(a.states)) lanes *= 2;
  const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.channels) * lanes, 128)), static_cast<unsigned>(a.seqs));
  mark_device();
  switch (a.type) {
    case MMFREE_T_F32: return launch_k(ssm_kernel<float>, grid, dim3(128), 0, s, false, a, lanes, step);
    case MMFREE_T_BF16: return launch_k(ssm_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, false, a, lanes, step);
    default: return launch_k(ssm_kernel<__half>, grid, dim3(128), 0, s, false, a, lanes, step);
  }
}

}  // namespace

cudaError_t take_sequence_flags(cudaStream_t s, uint32_t* flags) {
  *flags = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || !(g_devices.load(std::memory_order_relaxed) >> (dev & 63) & 1)) return e;
  e = cudaMemcpyFromSymbolAsync(flags, g_sequence_error, 4, 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess || !*flags) return e;
  const uint32_t zero = 0;
  e = cudaMemcpyToSymbolAsync(g_sequence_error, &zero, 4, 0, cudaMemcpyHostToDevice, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

cudaError_t launch_causal_conv(const mmfree_cuda_conv_args& a, cudaStream_t s) { return conv_any(a, false, s); }
cudaError_t launch_causal_conv_step(const mmfree_cuda_conv_args& a, cudaStream_t s) { return conv_any(a, true, s); }
cudaError_t launch_selective_scan(const mmfree_cuda_ssm_args& a, int, cudaStream_t s) { return ssm_any(a, false, s); }
cudaError_t launch_selective_step(const mmfree_cuda_ssm_args& a, cudaStream_t s) { return ssm_any(a, true, s); }

}  // namespace mmfree_cuda
