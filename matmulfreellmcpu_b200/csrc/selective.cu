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

// ---- tiled scan

// Two fp32 values in one 64-bit register, for the packed FMA (twice the operations an issue slot).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kLog2E = 1.44269504088896341f;

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, with log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3,
// by its series 2 (s + s^3/3 + s^5/5 + ...): the first term left out is below 2^-25 of the sum. Exact to a few
// steps for all v, where log(1 + e) rounded first would lose small e. Two special-function operations.
__device__ __forceinline__ float softplus_fast(float v) {
  const float e = ex2(-fabsf(v) * kLog2E);
  const float s = e * rcp(2.0f + e), q = s * s;
  float p = 1.0f / 15.0f;
  p = fmaf(p, q, 1.0f / 13.0f);
  p = fmaf(p, q, 1.0f / 11.0f);
  p = fmaf(p, q, 1.0f / 9.0f);
  p = fmaf(p, q, 1.0f / 7.0f);
  p = fmaf(p, q, 1.0f / 5.0f);
  p = fmaf(p, q, 1.0f / 3.0f);
  const float l = fmaf(s * q, p, s);
  return fmaf(2.0f, l, fmaxf(v, 0.0f));
}
__device__ __forceinline__ float silu_fast(float v) { return v * rcp(1.0f + ex2(-v * kLog2E)); }

// Sums v[i] over groups of kLanes neighbouring lanes for kSteps values at once: lane l of a group ends with the sum
// of value l % kSteps. Each exchange halves the values a lane holds, so kSteps sums take kSteps - 1 shuffles (and
// one for every doubling of kLanes over kSteps) instead of kSteps * log2(kLanes).
template <int kLanes, int kSteps>
__device__ __forceinline__ float transpose_sum(float (&v)[kSteps], int lane) {
#pragma unroll
  for (int o = 1; o < kSteps; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < kSteps / 2; ++i) {
      if (i >= kSteps / (2 * o)) break;
      // values 2i and 2i + 1 of this level go to the lanes whose bit is clear and set
      const float keep = up ? v[2 * i + 1] : v[2 * i], send = up ? v[2 * i] : v[2 * i + 1];
      v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, o);
    }
  }
  float r = v[0];
#pragma unroll
  for (int o = kSteps; o < kLanes; o <<= 1) r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
  return r;
}

constexpr int kScanThreads = 128;  // of each half of a CTA

// Shared memory of a scan CTA: what the two halves hand over, by tile.
template <int kTile, int kChannels, int kN>
struct ScanShared {
  float2 in[2][kTile][kChannels];    // delta, delta * x
  float2 finish[3][kTile][kChannels];  // D * x, silu(z)
  float y[2][kTile][kChannels];
  float b[2][kTile][kN], c[2][kTile][kN];
};

// One CTA: kScanThreads / kLanes channels of one group and one sequence, in tiles of kTile tokens, by two halves.
// The first half runs the recurrence, kLanes lanes a channel and kStates states a lane. The second half meanwhile
// turns the next tile's x, dt and z into what the recurrence and the outputs need, once per token and channel,
// finishes and stores the previous tile's outputs, and has the tile after the next in flight. They meet at one
// barrier a tile. In one half the two jobs alternated, and each left the issue slots of its latencies unused.
template <typename T, int kLanes, int kStates, int kTile>
__global__ void __launch_bounds__(2 * kScanThreads, 2) scan_kernel(mmfree_cuda_ssm_args a, int blocks_per_group) {
  constexpr int kChannels = kScanThreads / kLanes;           // channels of a CTA
  constexpr int kRows = kScanThreads / kChannels;            // token rows that the second half covers at once
  constexpr int kOwn = (kTile + kRows - 1) / kRows;          // tokens of one of its threads
  constexpr int kN = kLanes * kStates;                       // states, padded
  constexpr int kBC = (kTile * kN + kScanThreads - 1) / kScanThreads;  // elements of B (and of C) it stages
  constexpr int kSteps = kLanes < 8 ? kLanes : 8;            // tokens summed over lanes together
  static_assert(kTile % kSteps == 0, "tile shape");
  extern __shared__ __align__(16) char smem_raw[];
  auto& sh = *reinterpret_cast<ScanShared<kTile, kChannels, kN>*>(smem_raw);

  const int64_t seq = blockIdx.y;
  int64_t b, e;
  if (!sequence_rows(a.seq_starts, static_cast<int64_t>(a.tokens), seq, b, e) || b == e) return;
  const int64_t slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), seq);
  if (slot < 0) return;
  const int tid = threadIdx.x % kScanThreads, states = static_cast<int>(a.states);
  const int64_t channels = static_cast<int64_t>(a.channels), per_group = channels / static_cast<int64_t>(a.groups);
  const int64_t group = blockIdx.x / blocks_per_group;
  const int64_t first = (blockIdx.x - group * blocks_per_group) * kChannels;  // within the group
  const int live = static_cast<int>(min(static_cast<int64_t>(kChannels), per_group - first));
  const int64_t base = group * per_group + first;
  const int tiles = static_cast<int>((e - b + kTile - 1) / kTile);

  if (threadIdx.x < kScanThreads) {
    // ---- the recurrence
    const int lane = tid % kLanes, ch = tid / kLanes;
    const int64_t d = base + min(ch, live - 1);
    float* state = a.state ? a.state + (slot * channels + d) * states : nullptr;
    f32x2 h[kStates / 2], rate[kStates / 2];
#pragma unroll
    for (int j = 0; j < kStates / 2; ++j) {
      float hv[2], rv[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = lane * kStates + 2 * j + i;
        hv[i] = n < states && state ? state[n] : 0.0f;
        rv[i] = n < states ? a.A[d * states + n] * kLog2E : 0.0f;
      }
      h[j] = pack2(hv[0], hv[1]);
      rate[j] = pack2(rv[0], rv[1]);
    }
    __syncthreads();
    for (int tile = 0; tile < tiles; ++tile) {
      const int buf = tile & 1;
      const int left = static_cast<int>(min(static_cast<int64_t>(kTile), e - b - tile * kTile));
      for (int t = 0; t < left; t += kSteps) {
        float y[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const float2 in = sh.in[buf][t + k][ch];
          const f32x2 dd = pack2(in.x, in.x), dx = pack2(in.y, in.y);
          f32x2 sum = pack2(0.0f, 0.0f);
          f32x2 bv[kStates / 2], cv[kStates / 2];
          *reinterpret_cast<Pack<float, kStates>*>(bv) = *reinterpret_cast<const Pack<float, kStates>*>(&sh.b[buf][t + k][lane * kStates]);
          *reinterpret_cast<Pack<float, kStates>*>(cv) = *reinterpret_cast<const Pack<float, kStates>*>(&sh.c[buf][t + k][lane * kStates]);
#pragma unroll
          for (int j = 0; j < kStates / 2; ++j) {
            float lo, hi;
            unpack2(mul2(dd, rate[j]), lo, hi);
            h[j] = fma2(pack2(ex2(lo), ex2(hi)), h[j], mul2(dx, bv[j]));
            sum = fma2(cv[j], h[j], sum);
          }
          float lo, hi;
          unpack2(sum, lo, hi);
          y[k] = lo + hi;
        }
        const float r = transpose_sum<kLanes, kSteps>(y, lane);
        if (lane < kSteps) sh.y[buf][t + lane][ch] = r;
      }
      __syncthreads();
    }
    if (state && ch < live) {
#pragma unroll
      for (int j = 0; j < kStates / 2; ++j) {
        float hv[2];
        unpack2(h[j], hv[0], hv[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (lane * kStates + 2 * j + i < states) state[lane * kStates + 2 * j + i] = hv[i];
      }
    }
    return;
  }

  // ---- loads, per-token work and outputs
  const int ch = tid % kChannels, row = tid / kChannels;
  const int64_t d = base + min(ch, live - 1);
  const float skip = a.D ? a.D[d] : 0.0f, bias = a.dt_bias ? a.dt_bias[d] : 0.0f;
  const bool gate = a.z != nullptr, softplus = a.dt_softplus != 0;
  const int64_t ldx = static_cast<int64_t>(a.ldx), ldt = static_cast<int64_t>(a.ld_dt), ldz = static_cast<int64_t>(a.ldz),
                ldb = static_cast<int64_t>(a.ldb), ldc = static_cast<int64_t>(a.ldc), ldo = static_cast<int64_t>(a.ld_out);
  const T* px = static_cast<const T*>(a.x) + d;
  const T* pt = static_cast<const T*>(a.dt) + d;
  const T* pz = gate ? static_cast<const T*>(a.z) + d : nullptr;
  const T* pb = static_cast<const T*>(a.B) + group * states;
  const T* pc = static_cast<const T*>(a.C) + group * states;
  T* po = static_cast<T*>(a.out) + d;
  T rx[kOwn], rt[kOwn], rz[kOwn], rb[kBC], rc[kBC];
  const auto load = [&](int tile) {
    const int64_t t0 = b + tile * kTile;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int64_t t = min(t0 + row + i * kRows, e - 1);
      rx[i] = px[t * ldx];
      rt[i] = pt[t * ldt];
      if (gate) rz[i] = pz[t * ldz];
    }
#pragma unroll
    for (int i = 0; i < kBC; ++i) {
      const int at = tid + i * kScanThreads, n = min(at % kN, states - 1);
      const int64_t t = min(t0 + at / kN, e - 1);
      rb[i] = pb[t * ldb + n];
      rc[i] = pc[t * ldc + n];
    }
  };
  const auto prepare = [&](int tile) {
    const int buf = tile & 1, fin = tile % 3;
    const int64_t left = e - b - tile * kTile;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int t = row + i * kRows;
      if (kTile % kRows && t >= kTile) break;
      const float x = to_f32(rx[i]);
      float delta = to_f32(rt[i]) + bias;
      if (softplus) delta = softplus_fast(delta);
      // behind the sequence's end: a decay of 1 and no input
      sh.in[buf][t][ch] = t < left ? make_float2(delta, delta * x) : make_float2(0.0f, 0.0f);
      sh.finish[fin][t][ch] = make_float2(skip * x, gate ? silu_fast(to_f32(rz[i])) : 1.0f);
    }
#pragma unroll
    for (int i = 0; i < kBC; ++i) {
      const int at = tid + i * kScanThreads, n = at % kN;
      if (kTile * kN % kScanThreads && at >= kTile * kN) break;
      sh.b[buf][at / kN][n] = n < states ? to_f32(rb[i]) : 0.0f;
      sh.c[buf][at / kN][n] = n < states ? to_f32(rc[i]) : 0.0f;
    }
  };
  const auto finish = [&](int tile) {
    const int buf = tile & 1, fin = tile % 3;
    const int64_t t0 = b + tile * kTile, left = e - t0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int t = row + i * kRows;
      if (t >= left || (kTile % kRows && t >= kTile)) break;
      const float2 f = sh.finish[fin][t][ch];
      if (ch < live) po[(t0 + t) * ldo] = from_f32<T>((sh.y[buf][t][ch] + f.x) * f.y);
    }
  };
  load(0);
  prepare(0);
  if (tiles > 1) load(1);
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {  // the first half is at `tile`
    if (tile + 1 < tiles) prepare(tile + 1);
    if (tile + 2 < tiles) load(tile + 2);
    if (tile > 0) finish(tile - 1);
    __syncthreads();
  }
  finish(tiles - 1);
}

template <typename T, int kLanes, int kStates, int kTile>
cudaError_t scan_launch(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  constexpr int kChannels = kScanThreads / kLanes;
  constexpr size_t kSmem = sizeof(ScanShared<kTile, kChannels, kLanes * kStates>);
  const int blocks = static_cast<int>(ceil_div(static_cast<int64_t>(a.channels / a.groups), kChannels));
  // channel blocks fastest: consecutive CTAs go to different SMs, so every SM gets its share of each sequence
  const dim3 grid(static_cast<unsigned>(blocks * a.groups), static_cast<unsigned>(a.seqs));
  if (kSmem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(scan_kernel<T, kLanes, kStates, kTile>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(kSmem));
    if (e != cudaSuccess) return e;
  }
  return launch_k(scan_kernel<T, kLanes, kStates, kTile>, grid, dim3(2 * kScanThreads), kSmem, s, false, a, blocks);
}

// Lanes of a channel: four states a lane, eight where 32 lanes of four do not reach.
template <typename T>
cudaError_t scan_type(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  if (a.states <= 4) return scan_launch<T, 1, 4, 8>(a, s);
  if (a.states <= 8) return scan_launch<T, 2, 4, 16>(a, s);
  if (a.states <= 16) return scan_launch<T, 4, 4, 32>(a, s);
  if (a.states <= 32) return scan_launch<T, 8, 4, 32>(a, s);
  if (a.states <= 64) return scan_launch<T, 16, 4, 32>(a, s);
  if (a.states <= 128) return scan_launch<T, 32, 4, 32>(a, s);
  return scan_launch<T, 32, 8, 16>(a, s);
}

cudaError_t step_any(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  int lanes = 1;
  while (lanes < 32 && lanes < static_cast<int>(a.states)) lanes *= 2;
  const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.channels) * lanes, 128)), static_cast<unsigned>(a.seqs));
  mark_device();
  switch (a.type) {
    case MMFREE_T_F32: return launch_k(ssm_kernel<float>, grid, dim3(128), 0, s, false, a, lanes, true);
    case MMFREE_T_BF16: return launch_k(ssm_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, false, a, lanes, true);
    default: return launch_k(ssm_kernel<__half>, grid, dim3(128), 0, s, false, a, lanes, true);
  }
}

cudaError_t scan_any(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  mark_device();
  switch (a.type) {
    case MMFREE_T_F32: return scan_type<float>(a, s);
    case MMFREE_T_BF16: return scan_type<__nv_bfloat16>(a, s);
    default: return scan_type<__half>(a, s);
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
cudaError_t launch_selective_scan(const mmfree_cuda_ssm_args& a, int, cudaStream_t s) { return scan_any(a, s); }
cudaError_t launch_selective_step(const mmfree_cuda_ssm_args& a, cudaStream_t s) { return step_any(a, s); }

}  // namespace mmfree_cuda
