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
#include "tcgen05.cuh"

#include <type_traits>

namespace mmfree_cuda {

// Bit kErrRange once a sequence start or a slot broke its rules.
__device__ uint32_t g_sequence_error;

namespace {

LaunchedOn g_devices;

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
  if constexpr (V > 1) {  // 16-byte loads: the channels' taps lie one behind another
    const Pack<float, V * W> p = *reinterpret_cast<const Pack<float, V * W>*>(a.weight + d * W);
#pragma unroll
    for (int i = 0; i < V * W; ++i) w[i / W][i % W] = p.v[i];
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) w[0][j] = a.weight[d * W + j];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i] = a.bias ? a.bias[d + i] : 0.0f;
}

// The output of each channel for the newest input in[W - 1]; in[0] to in[W - 2] are the older ones.
template <int W, int V>
__device__ __forceinline__ void conv_token(const float (*in)[V], const float (&w)[V][W], const float (&bias)[V], bool silu, float (&y)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    y[i] = bias[i];
#pragma unroll
    for (int j = 0; j < W; ++j) y[i] = fmaf(w[i][j], in[j][i], y[i]);
  }
  if (silu)
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = silu_f32(y[i]);
}

// Bound by the bytes in fp32 (16384 x 5120 x 4 taps: 113 us, 6.0 TB/s), by the issue slots and the sigmoid's special
// functions in 16 bits (68 us, 4.9 TB/s). A thread keeps its channels' last inputs in registers.
// A CTA owns a tile of `rows` tokens for a block of channels. The tile in which a sequence
// begins reads that sequence's old state, writes the new one, and computes every token whose
// window still reaches into the old state, even those behind the tile's end, which the tiles
// there leave out: no other CTA reads a state that this one overwrites. The CTAs behind the last tile check every sequence,
// those too that no tile comes to (in the tiles' CTAs the check takes registers in front of the loads, 76 instead of 69 us
// for 16384 x 5120 bf16, or 0.5 us behind them).
template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_kernel(mmfree_cuda_conv_args a, int rows) {
  constexpr bool kVec = V > 1;
  const int64_t d = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  const int64_t tokens = static_cast<int64_t>(a.tokens), seqs = static_cast<int64_t>(a.seqs);
  if (blockIdx.y == gridDim.y - 1) {
    for (int64_t s = blockIdx.x * blockDim.x + threadIdx.x; s < seqs; s += static_cast<int64_t>(gridDim.x) * blockDim.x) {
      int64_t b, e;
      sequence_rows(a.seq_starts, tokens, s, b, e);
      sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), s);
    }
    return;
  }
  if (d >= static_cast<int64_t>(a.channels)) return;
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
    // eight tokens' loads in flight together
    constexpr int kBatch = 8;
    float in[W - 1 + kBatch][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) in[j][i] = win[j][i];
    for (; t + kBatch <= stop; t += kBatch) {
      Words<T, V> raw[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) raw[k].load(x + (t + k) * ldx);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) in[W - 1 + k][i] = raw[k][i];
        conv_token<W, V>(in + k, w, bias, silu, y);
        store_row<kVec>(out + (t + k) * ldo, V, y);
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) in[j][i] = in[kBatch + j][i];
    }
    for (; t < stop; ++t) {
      float y[V];
      load_row<kVec>(x + t * ldx, V, in[W - 1]);
      conv_token<W, V>(in, w, bias, silu, y);
      store_row<kVec>(out + t * ldo, V, y);
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) in[j][i] = in[j + 1][i];
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
  float in[W][V], y[V], w[V][W], bias[V];
  load_row<kVec>(static_cast<const T*>(a.x) + s * static_cast<int64_t>(a.ldx) + d, V, in[W - 1]);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    if (st) load_row<kVec>(st + j * pitch, V, in[j]);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) in[j][i] = 0.0f;
  }
  conv_load_taps<W, V>(a, d, w, bias);
  conv_token<W, V>(in, w, bias, a.silu != 0, y);
  store_row<kVec>(static_cast<T*>(a.out) + s * static_cast<int64_t>(a.ld_out) + d, V, y);
  if (st)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<kVec>(st + j * pitch, V, in[j + 1]);
}

template <typename T, int W, int V>
cudaError_t conv_launch(const mmfree_cuda_conv_args& a, bool step, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.channels), 128 * V));
  g_devices.mark();
  if (step) return launch_k(conv_step_kernel<T, W, V>, dim3(blocks, static_cast<unsigned>(a.seqs)), dim3(128), 0, s, false, a);
  // Tokens of a tile: 64, before which W - 1 are read once more (16384 x 5120 bf16: 68 us; 76 us with tiles of 128),
  // fewer where the tiles would not fill the 148 SMs (300 x 2048: 8.0 us, 14.6 us with 64).
  int rows = 64;
  while (rows > 8 && static_cast<int64_t>(blocks) * ceil_div(static_cast<int64_t>(a.tokens), rows) < 4 * 148) rows /= 2;
  while (ceil_div(static_cast<int64_t>(a.tokens), rows) >= 65535) rows *= 2;  // grid.y is 16 bits
  const unsigned tiles = static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.tokens), rows));
  return launch_k(conv_kernel<T, W, V>, dim3(blocks, tiles + 1), dim3(128), 0, s, false, a, rows);
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
  constexpr int V = 4;  // channels of a thread (with 8 of a 16-bit type, half as many warps: 76 instead of 68 us)
  const auto fits = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) == 0; };
  const bool vec = a.channels % V == 0 && a.ldx % V == 0 && a.ld_out % V == 0 && fits(a.x) && fits(a.out) && fits(a.state) &&
                   aligned16(a.weight);
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

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, with log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3,
// by its series 2 (s + s^3/3 + s^5/5 + ...): the first term left out is below 2^-25 of the sum. For v >= 0 off by a few
// steps; for v < 0 by (6 + |v|) 2^-24 of the value at most, since exp's argument |v| log2(e) is rounded once, and 0 below
// -87.3. (log(1 + e) rounded first would lose small e altogether.) Two special-function operations.
__device__ __forceinline__ float softplus_f32(float v) {
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

// A rate that is infinite (A itself, or its product with log2(e)) counts as the largest finite one: a decay of 0 after any
// step above 1e-36, as its own would be, and of 1, not NaN, where delta is 0, as behind a sequence's end.
__device__ __forceinline__ float finite_rate(float v) { return isinf(v) ? copysignf(3.402823466e38f, v) : v; }

// One token of each of kStreams streams: `lanes` lanes (a power of two) a channel, kStates neighbouring states a lane,
// kVec: read and written by 16 bytes. Bound by its issue slots (78% busy at 256 streams of 4096 x 16: 39 us, 3.6 TB/s) and by
// how many of the state's bytes are in flight together: four streams a thread where there are enough. Every lane repeats its
// channel's softplus and gate.
template <typename T, int kStates, int kStreams, bool kVec>
__global__ void __launch_bounds__(256) step_kernel(mmfree_cuda_ssm_args a, int lanes) {
  const int64_t channels = static_cast<int64_t>(a.channels), seqs = static_cast<int64_t>(a.seqs);
  const int states = static_cast<int>(a.states), lane = threadIdx.x & (lanes - 1);
  const int64_t d = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes, seq0 = static_cast<int64_t>(blockIdx.y) * kStreams;
  const bool live = d < channels;
  const int64_t dd = live ? d : channels - 1;
  const int n = lane * kStates, left = states - n;
  const int64_t group = dd / (channels / static_cast<int64_t>(a.groups));
  // all streams' loads without a branch or a use between them. One behind the last stream reads that one's; a stream that
  // is not there (a negative or bad slot) reads its channel's row of A in place of a state, since no state is its own and
  // the pool may hold none.
  bool there[kStreams];
  float* state[kStreams];
  float h[kStreams][kStates], rate[kStates] = {};
  Words<T, kVec ? kStates : 1> b[kStreams][kVec ? 1 : kStates], c[kStreams][kVec ? 1 : kStates];
  Words<T, 1> x[kStreams], delta[kStreams], z[kStreams];
#pragma unroll
  for (int k = 0; k < kStreams; ++k) {
    const int64_t seq = min(seq0 + k, seqs - 1), slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), seq);
    there[k] = slot >= 0 && seq0 + k < seqs;
    state[k] = (slot < 0 ? const_cast<float*>(a.A) : a.state + slot * channels * states) + dd * states + min(n, states - 1);
  }
#pragma unroll
  for (int k = 0; k < kStreams; ++k) {
    const int64_t seq = min(seq0 + k, seqs - 1);
    const T* const pb = static_cast<const T*>(a.B) + seq * static_cast<int64_t>(a.ldb) + group * states;
    const T* const pc = static_cast<const T*>(a.C) + seq * static_cast<int64_t>(a.ldc) + group * states;
    if constexpr (kVec) {  // a lane behind the last state reads that one's, and stores nothing
      const int at = min(n, states - kStates);
      load_row<true>(state[k] + (at - min(n, states - 1)), kStates, h[k]);
      b[k][0].load(pb + at);
      c[k][0].load(pc + at);
    } else {
#pragma unroll
      for (int i = 0; i < kStates; ++i) {
        const int at = min(n + i, states - 1);
        h[k][i] = state[k][at - min(n, states - 1)];
        b[k][i].load(pb + at);
        c[k][i].load(pc + at);
      }
    }
    x[k].load(static_cast<const T*>(a.x) + seq * static_cast<int64_t>(a.ldx) + dd);
    delta[k].load(static_cast<const T*>(a.dt) + seq * static_cast<int64_t>(a.ld_dt) + dd);
    if (a.z) z[k].load(static_cast<const T*>(a.z) + seq * static_cast<int64_t>(a.ldz) + dd);
  }
  if (left > 0) load_row<kVec>(a.A + dd * states + n, left, rate);
#pragma unroll
  for (int i = 0; i < kStates; ++i) rate[i] = finite_rate(rate[i]);
  const float bias = a.dt_bias ? a.dt_bias[dd] : 0.0f, skip = a.D ? a.D[dd] : 0.0f;
#pragma unroll
  for (int k = 0; k < kStreams; ++k) {
    const float xk = x[k][0];
    float dl = delta[k][0] + bias, y = 0.0f;
    if (a.dt_softplus) dl = softplus_f32(dl);
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
      const float bi = kVec ? b[k][0][kVec ? i : 0] : b[k][kVec ? 0 : i][0], ci = kVec ? c[k][0][kVec ? i : 0] : c[k][kVec ? 0 : i][0];
      h[k][i] = fmaf(ex2(dl * rate[i] * kLog2E), h[k][i], dl * xk * bi);
      if (i < left) y = fmaf(ci, h[k][i], y);
    }
    for (int o = lanes >> 1; o; o >>= 1) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
    if (!live || !there[k]) continue;
    if (left > 0) store_row<kVec>(state[k], left, h[k]);
    if (a.D) y = fmaf(skip, xk, y);  // without D not 0 * x, which may be 0 * infinity
    if (a.z) y *= silu_f32(z[k][0]);
    if (lane == 0) static_cast<T*>(a.out)[(seq0 + k) * static_cast<int64_t>(a.ld_out) + dd] = from_f32<T>(y);
  }
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

// An asynchronous copy of 4, 8 or 16 bytes from global to shared memory.
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(src), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// The state behind a piece: the piece's own, `end`, plus the state h before it times 2^exponent. Token by token an infinite
// state stays infinite and one of 0 stays 0, so they do here, where the whole piece's factor may be 0 or infinite.
__device__ __forceinline__ float past_piece(float h, float exponent, float end) {
  const bool kept = (h == 0.0f || isinf(h)) && isfinite(exponent);
  return fmaf(kept ? 1.0f : ex2(exponent), h, end);
}

// The shape of a scan CTA. kLanes lanes hold the states of kPer neighbouring channels, kStates states of each a lane.
template <typename T, int kLanes_, int kStates_, int kPer_, int kTile_, int kScan_, int kHelpers_, int kCtas_, int kBytes_>
struct ScanShape {
  using Type = T;
  static constexpr int kLanes = kLanes_, kStates = kStates_, kPer = kPer_, kTile = kTile_;
  static constexpr int kScan = kScan_;                          // threads of the recurrence
  static constexpr int kHelpers = kHelpers_;                    // threads that load, prepare and store
  static constexpr int kCtas = kCtas_;                          // CTAs an SM that the registers leave room for
  static constexpr int kBytes = kBytes_;                        // of an access: 16 or 4, copied asynchronously, or 0: one element
  static constexpr bool kVec = kBytes > 0;
  static constexpr bool kMaySplit = kCtas < 4;                  // the shape for short sequences never splits them
  static constexpr int kN = kLanes * kStates;                   // states, padded
  static constexpr int kChannels = kScan / kLanes * kPer;
  static constexpr int kWide = kVec ? kBytes / sizeof(T) : 1;
  static constexpr int V = kWide < kChannels ? kWide : kChannels, VB = kWide < 4 ? kWide : 4;  // channels and states of one access
  static constexpr int kColumns = kChannels / V;                // helper threads along a token
  static constexpr int kRows = kHelpers / kColumns;             // tokens that the helpers cover at once
  static constexpr int kOwn = (kTile + kRows - 1) / kRows;      // tokens of a helper
  static constexpr int kBC = (kTile * kN / VB + kHelpers - 1) / kHelpers;  // vectors of B (and of C) of a helper
  static constexpr int kStages = kVec ? 4 : 1;
  // Places behind the last state hold copies of the first ones, each with its share of C (shares of a half or a quarter,
  // which are exact): with zeros there, an infinite x would bring 0 * infinity into the sum. kN is the power of two next to
  // the number of states (or 4), so that a state has one copy at most, and the only one of a single state has three.
  __device__ static int source(int n, int states, int width) { return n < states ? n : min(n - states, states - width); }
  __device__ static float share(int n, int states) { return states == 1 ? 0.25f : n < kN - states || n >= states ? 0.5f : 1.0f; }
  struct Raw {  // one tile as it lies in memory; every helper reads what it copied itself
    Pack<T, V> x[kOwn][kHelpers], dt[kOwn][kHelpers], z[kOwn][kHelpers];
    Pack<T, VB> b[kBC][kHelpers], c[kBC][kHelpers];
  };
  struct Shared {
    float2 in[2][kTile][kChannels];  // delta, delta * x
    float y[2][kTile][kChannels];
    float b[2][kTile][kN], c[2][kTile][kN];
    float carry[kPer * (kStates + 1)][kScan];  // a piece's last state and sum of deltas, for the pieces behind it
    Raw raw[kStages];
  };
};

// One CTA: a block of channels of one group and one sequence, in tiles of kTile tokens, by two halves. The first
// runs the recurrence. The second, the helpers, meanwhile turns the next tile's x and dt into (delta, delta * x),
// once per token and channel, finishes and stores the previous tile's outputs, and keeps two more tiles in flight
// from memory. They meet at one barrier a tile. In one half the jobs alternated, and each left the issue slots of
// its latencies unused.
// splits > 1: the CTAs of a cluster take a sequence's pieces. A state after a piece is the piece's own, from a state of
// 0, plus the state before it times exp(A * the sum of the piece's deltas): so the pieces between the first and the last
// run without outputs first, then every piece but the first starts from the states and sums of those before it, read
// from their shared memory. Two passes for a sequence, each over 1 / splits of it.
// Bound by the exponentials, one for each token, channel and state: 16 a clock and SM, 385 us with the helpers' for
// 16384 tokens x 5120 channels x 16 states, where the kernel takes 647 us; the special-function unit is busy 60% of the
// time, the rest goes to the two halves' waits for each other and for its latency. An eighth or a quarter of the
// exponentials as polynomials on the multiply-add pipe changed nothing (663 and 693 against 657 us), nor did more CTAs an SM.
// What a turn of the recurrence reads from shared memory bounds it next to the special-function unit (128 bytes of
// registers a clock): kPer channels a lane share one read of B and C.
template <typename S>
__global__ void __launch_bounds__(S::kScan + S::kHelpers, S::kCtas) scan_kernel(mmfree_cuda_ssm_args a, int blocks_per_group, int splits_asked) {
  using T = typename S::Type;
  constexpr int kLanes = S::kLanes, kStates = S::kStates, kPer = S::kPer, kTile = S::kTile, kN = S::kN, V = S::V, VB = S::VB;
  constexpr int kGroup = 4;                                  // tokens of a turn of the recurrence
  constexpr int kSteps = kLanes < kGroup ? kLanes : kGroup;  // tokens summed over lanes together
  constexpr int kPairs = kStates / 2;
  const int splits = S::kMaySplit ? splits_asked : 1;
  static_assert(kTile % kGroup == 0 && sizeof(typename S::Shared) <= 227 * 1024, "tile shape");
  extern __shared__ __align__(16) char smem_raw[];
  auto& sh = *reinterpret_cast<typename S::Shared*>(smem_raw);

  const int64_t seq = blockIdx.y;
  int64_t b, e;
  if (!sequence_rows(a.seq_starts, static_cast<int64_t>(a.tokens), seq, b, e)) return;
  const int64_t slot = sequence_slot(a.slots, static_cast<int64_t>(a.slot_count), seq);  // an empty sequence's is checked too
  if (slot < 0 || b == e) return;
  const int states = static_cast<int>(a.states);
  const int64_t channels = static_cast<int64_t>(a.channels), per_group = channels / static_cast<int64_t>(a.groups);
  const int rank = splits > 1 ? blockIdx.x % splits : 0;
  const int64_t block = blockIdx.x / splits, group = block / blocks_per_group;
  const int64_t first = (block - group * blocks_per_group) * S::kChannels;  // within the group
  const int live = static_cast<int>(min(static_cast<int64_t>(S::kChannels), per_group - first));
  const int64_t base = group * per_group + first;
  // this CTA's piece: at least four tiles, and three pieces or one (two would run one after the other)
  int pieces = 1, length = static_cast<int>(e - b);
  if (splits > 1) {
    pieces = min(splits, length / (4 * kTile));
    if (pieces < 3) pieces = 1;
    const int piece = (length + pieces * kTile - 1) / (pieces * kTile) * kTile;
    pieces = (length + piece - 1) / piece;
    b += min(rank * piece, length);
    length = max(0, min(piece, length - rank * piece));
  }
  const bool mine_first = rank == 0, between = rank > 0 && rank < pieces - 1, behind = rank > 0 && rank < pieces;
  const int tiles = (length + kTile - 1) / kTile;

  if (threadIdx.x < S::kScan) {
    // ---- the recurrence
    const int lane = threadIdx.x % kLanes, ch = threadIdx.x / kLanes * kPer;
    float* const pool = a.state ? a.state + slot * channels * states : nullptr;
    f32x2 h[kPer][kPairs], rate[kPer][kPairs];
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const int64_t d = base + min(ch + c, live - 1);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        float hv[2], rv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = S::source(lane * kStates + 2 * j + i, states, 1);
          hv[i] = pool && mine_first ? pool[d * states + n] : 0.0f;
          rv[i] = finite_rate(a.A[d * states + n] * kLog2E);
        }
        h[c][j] = pack2(hv[0], hv[1]);
        rate[c][j] = pack2(rv[0], rv[1]);
      }
    }
    // the recurrence over `count` turns from token t0 of the tile; the outputs are stored behind the last one, since
    // a store between them would keep the next turn's loads from shared memory behind it
    double deltas[kPer] = {};
    const auto turns = [&](int buf, int t0, auto count, auto outputs) {
      constexpr int kCount = decltype(count)::value;
      constexpr bool kOut = decltype(outputs)::value;
      float part_deltas[kPer] = {};
      float out[kCount][kPer][kGroup / kSteps];
#pragma unroll
      for (int turn = 0; turn < kCount; ++turn) {
        float y[kPer][kGroup];
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          const int t = t0 + turn * kGroup + k;
          const Pack<float, 2 * kPer> in = *reinterpret_cast<const Pack<float, 2 * kPer>*>(&sh.in[buf][t][ch]);
          f32x2 bv[kPairs], cv[kPairs];
          *reinterpret_cast<Pack<float, kStates>*>(bv) = *reinterpret_cast<const Pack<float, kStates>*>(&sh.b[buf][t][lane * kStates]);
          if (kOut) *reinterpret_cast<Pack<float, kStates>*>(cv) = *reinterpret_cast<const Pack<float, kStates>*>(&sh.c[buf][t][lane * kStates]);
#pragma unroll
          for (int c = 0; c < kPer; ++c) {
            if (!kOut) part_deltas[c] += in.v[2 * c];
            const f32x2 dl = pack2(in.v[2 * c], in.v[2 * c]), dx = pack2(in.v[2 * c + 1], in.v[2 * c + 1]);
            f32x2 sum;
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              float lo, hi;
              unpack2(mul2(dl, rate[c][j]), lo, hi);
              h[c][j] = fma2(pack2(ex2(lo), ex2(hi)), h[c][j], mul2(dx, bv[j]));
              if (kOut) sum = j ? fma2(cv[j], h[c][j], sum) : mul2(cv[j], h[c][j]);
            }
            if (!kOut) continue;
            float lo, hi;
            unpack2(sum, lo, hi);
            y[c][k] = lo + hi;
          }
        }
        if (!kOut) continue;
#pragma unroll
        for (int c = 0; c < kPer; ++c)
#pragma unroll
          for (int g = 0; g < kGroup; g += kSteps) {
            float part[kSteps];
#pragma unroll
            for (int k = 0; k < kSteps; ++k) part[k] = y[c][g + k];
            out[turn][c][g / kSteps] = transpose_sum<kLanes, kSteps>(part, lane);
          }
      }
      if (!kOut) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) deltas[c] += part_deltas[c];  // over a piece in 64 bits
      } else if (lane < kSteps)
#pragma unroll
        for (int turn = 0; turn < kCount; ++turn)
#pragma unroll
          for (int g = 0; g < kGroup; g += kSteps) {
            Pack<float, kPer> v;
#pragma unroll
            for (int c = 0; c < kPer; ++c) v.v[c] = out[turn][c][g / kSteps];
            *reinterpret_cast<Pack<float, kPer>*>(&sh.y[buf][t0 + turn * kGroup + g + lane][ch]) = v;
          }
    };
    constexpr int kTurns = kTile / kGroup;
    const auto sweep = [&](auto outputs) {
      __syncthreads();
      for (int tile = 0; tile < tiles; ++tile) {
        const int buf = tile & 1, left = min(kTile, length - tile * kTile);
        if (left > kTile - kGroup) {  // unrolled as a whole, so that loads and exponentials run ahead of the sums
          turns(buf, 0, std::integral_constant<int, kTurns>{}, outputs);
        } else {
#pragma unroll 1
          for (int t = 0; t < left; t += 2 * kGroup) turns(buf, t, std::integral_constant<int, 2>{}, outputs);
        }
        __syncthreads();
      }
    };
    if (between) sweep(std::false_type{});
    // the first piece's outputs before the exchange, the others' behind it (one copy of the code for both)
#pragma unroll 1
    for (int phase = 0; phase < 2; ++phase) {
      if (phase == 0 ? mine_first : behind) sweep(std::true_type{});
      if (phase == 1 || splits == 1) break;
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j)
          unpack2(h[c][j], sh.carry[c * (kStates + 1) + 2 * j][threadIdx.x], sh.carry[c * (kStates + 1) + 2 * j + 1][threadIdx.x]);
        sh.carry[c * (kStates + 1) + kStates][threadIdx.x] = static_cast<float>(deltas[c]);
      }
      cluster_sync();
      if (behind) {
        const auto peer = [&](int value, int q) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map(smem_u32(&sh.carry[value][threadIdx.x]), q)) : "memory");
          return v;
        };
        for (int q = 0; q < rank; ++q)
#pragma unroll
          for (int c = 0; c < kPer; ++c) {
            const float sum = q ? peer(c * (kStates + 1) + kStates, q) : 0.0f;
            const f32x2 sums = pack2(sum, sum);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              const float end_lo = peer(c * (kStates + 1) + 2 * j, q), end_hi = peer(c * (kStates + 1) + 2 * j + 1, q);
              float lo, hi, h_lo, h_hi;
              unpack2(mul2(sums, rate[c][j]), lo, hi);
              unpack2(h[c][j], h_lo, h_hi);
              h[c][j] = q ? pack2(past_piece(h_lo, lo, end_lo), past_piece(h_hi, hi, end_hi)) : pack2(end_lo, end_hi);
            }
          }
      }
    }
    if (splits > 1) cluster_sync();  // before a CTA whose shared memory is read ends
    if (rank != pieces - 1) return;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      if (!pool || ch + c >= live) break;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        float hv[2];
        unpack2(h[c][j], hv[0], hv[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = lane * kStates + 2 * j + i;
          if (n < states) pool[(base + ch + c) * states + n] = hv[i];
        }
      }
    }
    return;
  }

  // ---- the helpers
  constexpr int kOwn = S::kOwn, kRows = S::kRows, kBC = S::kBC, kHelpers = S::kHelpers;
  const int tid = threadIdx.x - S::kScan, ch = tid % S::kColumns * V, row = tid / S::kColumns;
  const bool mine = ch < live;  // whole vectors
  const int64_t d = base + (mine ? ch : 0);
  float skip[V], bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    skip[v] = a.D ? a.D[d + v] : 0.0f;
    bias[v] = a.dt_bias ? a.dt_bias[d + v] : 0.0f;
  }
  const bool gate = a.z != nullptr, skips = a.D != nullptr, softplus = a.dt_softplus != 0;
  const int64_t ldx = static_cast<int64_t>(a.ldx), ldt = static_cast<int64_t>(a.ld_dt), ldz = static_cast<int64_t>(a.ldz),
                ldb = static_cast<int64_t>(a.ldb), ldc = static_cast<int64_t>(a.ldc), ldo = static_cast<int64_t>(a.ld_out);
  const T* px = static_cast<const T*>(a.x) + b * ldx + d;
  const T* pt = static_cast<const T*>(a.dt) + b * ldt + d;
  const T* pz = gate ? static_cast<const T*>(a.z) + b * ldz + d : nullptr;
  const T* pb = static_cast<const T*>(a.B) + group * states + b * ldb;
  const T* pc = static_cast<const T*>(a.C) + group * states + b * ldc;
  T* po = static_cast<T*>(a.out) + b * ldo + d;
  const auto load = [&](int tile) {
    if (tile < tiles) {
      auto& raw = sh.raw[tile % S::kStages];
      const int t0 = tile * kTile, most = length - 1 - t0;  // tokens behind the end read the last one again
      const auto fetch = [](auto* dst, const T* src) {
        if constexpr (S::kVec) copy_async<sizeof(*dst)>(dst, src);
        else dst->v[0] = *src;
      };
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (kTile % kRows && row + i * kRows >= kTile) break;
        const int64_t t = t0 + min(row + i * kRows, most);
        fetch(&raw.x[i][tid], px + t * ldx);
        fetch(&raw.dt[i][tid], pt + t * ldt);
        if (gate) fetch(&raw.z[i][tid], pz + t * ldz);
      }
#pragma unroll
      for (int i = 0; i < kBC; ++i) {
        const int at = (tid + i * kHelpers) * VB, n = S::source(at % kN, states, VB);
        if (kTile * kN / VB % kHelpers && at >= kTile * kN) break;
        const int64_t t = t0 + min(at / kN, most);
        fetch(&raw.b[i][tid], pb + t * ldb + n);
        fetch(&raw.c[i][tid], pc + t * ldc + n);
      }
    }
    if constexpr (S::kVec) copy_commit();
  };
  const auto prepare = [&](int tile) {
    if (tile >= tiles) return;
    const int buf = tile & 1, left = length - tile * kTile;
    const auto& raw = sh.raw[tile % S::kStages];
    // branches around whole arrays: around single elements they would keep the elements' chains one after another
    float delta[kOwn][V], x[kOwn][V];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (kTile % kRows && row + i * kRows >= kTile) break;
      const Pack<T, V> rx = raw.x[i][tid], rt = raw.dt[i][tid];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[i][v] = to_f32(rx.v[v]);
        delta[i][v] = to_f32(rt.v[v]) + bias[v];
      }
    }
    if (softplus) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) delta[i][v] = softplus_f32(delta[i][v]);
    }
    if (left < kTile) {  // behind the sequence's end: a decay of 1 and no input, also where x is not finite
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (row + i * kRows >= left) delta[i][v] = x[i][v] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int t = row + i * kRows;
      if (kTile % kRows && t >= kTile) break;
      Pack<float, 2 * V> in;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        in.v[2 * v] = delta[i][v];
        in.v[2 * v + 1] = delta[i][v] * x[i][v];
      }
      *reinterpret_cast<Pack<float, 2 * V>*>(&sh.in[buf][t][ch]) = in;
    }
#pragma unroll
    for (int i = 0; i < kBC; ++i) {
      const int at = (tid + i * kHelpers) * VB, n = at % kN;
      if (kTile * kN / VB % kHelpers && at >= kTile * kN) break;
      const Pack<T, VB> rb = raw.b[i][tid], rc = raw.c[i][tid];
      Pack<float, VB> vb, vc;
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        vb.v[v] = at / kN < left ? to_f32(rb.v[v]) : 0.0f;  // 0 behind the end too: 0 * inf is not 0
        vc.v[v] = to_f32(rc.v[v]) * S::share(n + v, states);
      }
      *reinterpret_cast<Pack<float, VB>*>(&sh.b[buf][at / kN][n]) = vb;
      *reinterpret_cast<Pack<float, VB>*>(&sh.c[buf][at / kN][n]) = vc;
    }
  };
  const auto finish = [&](int tile) {
    const int buf = tile & 1, t0 = tile * kTile, left = length - t0;
    const auto& raw = sh.raw[tile % S::kStages];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int t = row + i * kRows;
      if ((kTile % kRows && t >= kTile) || t >= left) break;
      Pack<T, V> rx, rz;
      if constexpr (S::kVec) {
        rx = raw.x[i][tid];
        if (gate) rz = raw.z[i][tid];
      } else {
        rx.v[0] = px[(t0 + t) * ldx];
        if (gate) rz.v[0] = pz[(t0 + t) * ldz];
      }
      const Pack<float, V> p = *reinterpret_cast<const Pack<float, V>*>(&sh.y[buf][t][ch]);
      float y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = p.v[v];
      if (skips)  // without D not 0 * x, which may be 0 * infinity
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = fmaf(skip[v], to_f32(rx.v[v]), y[v]);
      if (gate)
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] *= silu_f32(to_f32(rz.v[v]));
      if (mine) store_row<S::kVec>(po + static_cast<int64_t>(t0 + t) * ldo, V, y);
    }
  };
  // before the first half's tile 0: tile 0 prepared; in its tile t: t + 1 prepared, t - 1 finished, then its stage filled
  constexpr int kAhead = S::kStages - 1;
  const auto sweep = [&](bool outputs) {
    load(0);
    if constexpr (S::kVec) {
      load(1);
      load(2);
      copy_wait<kAhead - 1>();
    }
    prepare(0);
    __syncthreads();
    for (int tile = 0; tile < tiles; ++tile) {
      if constexpr (S::kVec) copy_wait<kAhead - 2>();
      else load(tile + 1);
      prepare(tile + 1);
      if (outputs && tile > 0) finish(tile - 1);
      if constexpr (S::kVec) load(tile + kAhead);
      __syncthreads();
    }
    if (outputs) finish(tiles - 1);
  };
#pragma unroll 1
  for (int phase = 0; phase < 2; ++phase) {
    if (phase == 0 ? mine_first || between : behind) sweep(phase == 1 || mine_first);
    if (splits > 1) cluster_sync();
    else break;
  }
}

template <typename S>
cudaError_t scan_launch(const mmfree_cuda_ssm_args& a, int sms, cudaStream_t s) {
  constexpr size_t kSmem = sizeof(typename S::Shared);
  const int blocks = static_cast<int>(ceil_div(static_cast<int64_t>(a.channels / a.groups), S::kChannels));
  // Few CTAs and long sequences: clusters of 8 or 4 split each sequence, as many as two CTAs an SM hold. One sequence of
  // 8192 tokens x 1024 channels (bf16, 32 CTAs): 334 us in one piece, 144 us in 8; 2048 x 2048 (64 CTAs): 86.5 us in one
  // piece, 74.7 us in 4. The host knows the sequences' mean length alone, and goes by it here and in scan_states: a long
  // prompt among many short sequences is not split.
  const int64_t ctas = static_cast<int64_t>(blocks) * static_cast<int64_t>(a.groups * a.seqs);
  const bool long_ones = a.tokens / a.seqs >= 512;
  const int splits = !S::kMaySplit || !long_ones ? 1 : ctas * 4 <= sms ? 8 : ctas * 2 <= sms ? 4 : 1;
  // channel blocks fastest: consecutive CTAs go to different SMs, so every SM gets its share of each sequence
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * a.groups * splits), static_cast<unsigned>(a.seqs));
  cfg.blockDim = dim3(S::kScan + S::kHelpers);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(splits);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  if (kSmem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(scan_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, scan_kernel<S>, a, blocks, splits);
}

template <typename T, int kBytes>
cudaError_t scan_states(const mmfree_cuda_ssm_args& a, int sms, cudaStream_t s) {
  if (a.states <= 4) return scan_launch<ScanShape<T, 1, 4, 1, 8, 128, 128, 2, kBytes>>(a, sms, s);
  if (a.states <= 8) return scan_launch<ScanShape<T, 2, 4, 1, 16, 128, 128, 2, kBytes>>(a, sms, s);
  if (a.states <= 16) {
    // Short sequences on many CTAs: two channels a lane (half the reads of B and C) and tiles of 16 tokens, which leave
    // less behind a sequence's end: 300 tokens in 16 sequences x 2048 channels (fp32) take 14.3 against 16.7 us. Long
    // ones the other way: 16384 tokens in 8 sequences x 5120 channels (bf16) 647 against 657 us, one sequence of
    // 4099 x 4096 160 against 203 us. By the mean length: 63 single tokens and a prompt of 4033 x 4096 (bf16) come here and
    // take 417 us, the prompt alone 164 us.
    if (static_cast<int64_t>(a.channels * a.seqs) >= 32 * 3 * static_cast<int64_t>(sms) && a.tokens / a.seqs < 512)
      return scan_launch<ScanShape<T, 4, 4, 2, 16, 64, 64, 4, kBytes>>(a, sms, s);
    return scan_launch<ScanShape<T, 4, 4, 1, 32, 128, 128, 2, kBytes>>(a, sms, s);
  }
  if (a.states <= 32) return scan_launch<ScanShape<T, 8, 4, 1, 32, 128, 128, 2, kBytes>>(a, sms, s);
  if (a.states <= 64) return scan_launch<ScanShape<T, 16, 4, 1, 32, 128, 128, 2, kBytes>>(a, sms, s);
  if (a.states <= 128) return scan_launch<ScanShape<T, 32, 4, 2, 16, 128, 128, 2, kBytes>>(a, sms, s);
  return scan_launch<ScanShape<T, 32, 8, 1, 8, 128, 128, 2, kBytes>>(a, sms, s);
}

template <typename T>
cudaError_t scan_type(const mmfree_cuda_ssm_args& a, int sms, cudaStream_t s) {
  // whether x, dt, z and out can be accessed by `n` channels, and B and C by up to four states
  const auto fits = [&](size_t n) {
    const size_t m = n < 4 ? n : 4;
    const auto one = [](const void* p, size_t pitch, size_t k) { return reinterpret_cast<uintptr_t>(p) % (k * sizeof(T)) == 0 && pitch % k == 0; };
    return a.channels / a.groups % n == 0 && a.states % m == 0 && one(a.x, a.ldx, n) && one(a.dt, a.ld_dt, n) && one(a.z, a.ldz, n) &&
           one(a.out, a.ld_out, n) && one(a.B, a.ldb, m) && one(a.C, a.ldc, m);
  };
  if (fits(16 / sizeof(T))) return scan_states<T, 16>(a, sms, s);
  return fits(4 / sizeof(T)) ? scan_states<T, 4>(a, sms, s) : scan_states<T, 0>(a, sms, s);
}

template <typename T, int kStates, bool kVec>
cudaError_t step_launch(const mmfree_cuda_ssm_args& a, int lanes, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.channels) * lanes, 256));
  // four streams a thread where one stream a thread would be more threads than the 148 SMs hold at once (4096 x 16
  // states, with slots, captured: 64 streams 11.2 against 14.8 us, 256 streams 39.2 against 53.5 us)
  if (static_cast<int64_t>(blocks) * static_cast<int64_t>(a.seqs) > 148 * 8)
    return launch_k(step_kernel<T, kStates, 4, kVec>, dim3(blocks, static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.seqs), 4))), dim3(256), 0, s, false, a, lanes);
  return launch_k(step_kernel<T, kStates, 1, kVec>, dim3(blocks, static_cast<unsigned>(a.seqs)), dim3(256), 0, s, false, a, lanes);
}

template <typename T>
cudaError_t step_type(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  const int states = static_cast<int>(a.states), per = states <= 128 ? 4 : 8;
  int lanes = 1;
  while (lanes * per < states) lanes *= 2;
  const auto one = [](const void* p, size_t pitch, size_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch * sizeof(T) % bytes == 0;
  };
  const size_t bytes = per * sizeof(T) < 16 ? per * sizeof(T) : 16;
  const bool vec = states % per == 0 && aligned16(a.state) && aligned16(a.A) && one(a.B, a.ldb, bytes) && one(a.C, a.ldc, bytes);
  if (per == 4) return vec ? step_launch<T, 4, true>(a, lanes, s) : step_launch<T, 4, false>(a, lanes, s);
  return vec ? step_launch<T, 8, true>(a, lanes, s) : step_launch<T, 8, false>(a, lanes, s);
}

cudaError_t step_any(const mmfree_cuda_ssm_args& a, cudaStream_t s) {
  g_devices.mark();
  switch (a.type) {
    case MMFREE_T_F32: return step_type<float>(a, s);
    case MMFREE_T_BF16: return step_type<__nv_bfloat16>(a, s);
    default: return step_type<__half>(a, s);
  }
}

cudaError_t scan_any(const mmfree_cuda_ssm_args& a, int sms, cudaStream_t s) {
  g_devices.mark();
  switch (a.type) {
    case MMFREE_T_F32: return scan_type<float>(a, sms, s);
    case MMFREE_T_BF16: return scan_type<__nv_bfloat16>(a, sms, s);
    default: return scan_type<__half>(a, sms, s);
  }
}

}  // namespace

cudaError_t take_sequence_flags(cudaStream_t s, uint32_t* flags) { return take_word(g_sequence_error, g_devices, s, flags); }

cudaError_t launch_causal_conv(const mmfree_cuda_conv_args& a, cudaStream_t s) { return conv_any(a, false, s); }
cudaError_t launch_causal_conv_step(const mmfree_cuda_conv_args& a, cudaStream_t s) { return conv_any(a, true, s); }
cudaError_t launch_selective_scan(const mmfree_cuda_ssm_args& a, int sm_count, cudaStream_t s) { return scan_any(a, sm_count, s); }
cudaError_t launch_selective_step(const mmfree_cuda_ssm_args& a, cudaStream_t s) { return step_any(a, s); }

}  // namespace mmfree_cuda
