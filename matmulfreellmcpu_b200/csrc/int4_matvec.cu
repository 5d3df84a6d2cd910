// int4_matvec.cu -- products of a few rows with 4-bit weights that have a scale (and a zero
// point) for each group of columns.
//
//   out[m, n] = xs[m] * sum_g s[n, g] * sum_{k in g} (u[n, k] - z[n, g]) * x[m, k]
//
// Bound by the weights' bytes: half a byte and one multiply-add per weight and row. In fp32
// registers a weight costs two instructions to unpack and one per row, three times what the
// issue slots allow at the memory's rate, so the products run on the tensor cores (the warp
// instruction m16n8k16: 16 weight rows x 8 activation rows x 16 columns; tcgen05 would need the
// unpacked weights in shared or tensor memory first, an extra trip for operands used once).
// u - z is a small whole number, exact in fp16 and bf16; e4m3 rows are exact in fp16; fp32 rows
// are cut into three bf16 parts of 8 bits each, exactly. The products are therefore exact, summed
// in fp32, and a group's sum is scaled once. For int8 rows the codes stay whole numbers:
// m16n8k32 of u8 codes and s8 rows, summed in 32 bits, and a group's sum of (u - z) x is the sum
// of u x minus z times the sum of x, which an operand of ones gives (one row, 2048 -> 32000: 19.1 us as
// fp16, 14.5 us).
//
// The order of a product's columns is free as long as weights and activations agree, so a lane
// takes 8 consecutive columns of its weight row, one word of the row-major codes: no repacked
// copy of the weights. The words come through shared memory, filled by asynchronous copies two
// turns ahead; rolled loops over it keep the code small (with the words in registers the
// unrolled loops were bound by instruction fetches: 20.4 instead of 15.2 us for 16 fp32 rows,
// 5632 -> 2048).
#include "block_ops.h"
#include "common.cuh"
#include "elements.cuh"
#include "tcgen05.cuh"

#include <cuda_fp8.h>

namespace mmfree_cuda {

// Bit kErrRange once a zero point was above 127 for rows that become bf16 operands.
__device__ uint32_t g_zero_point_error;

namespace {

LaunchedOn g_devices;

constexpr int kWarps = 8;       // of a CTA: they share its weight rows and split the columns
constexpr int kTileK = 256;     // columns of a warp's turn (128 bytes of a weight row)
constexpr int kTurnRuns = kTileK / 32;  // runs: 32 columns, 8 of each of the 4 lanes that share a row
constexpr int kPitch = 36;      // words of a partial-sum row of 32 outputs: keeps its writers on different banks

__device__ __forceinline__ void put_out(void* p, int type, int64_t i, float v) {
  switch (type) {
    case MMFREE_T_F32: static_cast<float*>(p)[i] = v; break;
    case MMFREE_T_BF16: static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v); break;
    default: static_cast<__half*>(p)[i] = from_f32<__half>(v); break;
  }
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t b2_sub(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// How rows of a type become tensor-core operands: kParts operands, pairs of f16 or bf16.
template <int kType>
struct RowType {
  static constexpr bool kBf16 = kType == MMFREE_T_BF16 || kType == MMFREE_T_F32;
  static constexpr int kParts = kType == MMFREE_T_F32 ? 3 : 1;
  static constexpr int kBytes = kType == MMFREE_T_F32 ? 4 : kType >= MMFREE_T_S8 ? 1 : 2;
  static constexpr int kWords = 2 * kBytes;  // of 8 elements
};

// Eight elements of a row from an aligned address.
template <int kType>
__device__ __forceinline__ void load_x(const char* p, uint32_t (&w)[RowType<kType>::kWords]) {
  if constexpr (RowType<kType>::kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < RowType<kType>::kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

// The same from any address, `left` of them inside the row (the others are 0).
template <int kType>
__device__ __forceinline__ void load_x_part(const char* p, int left, uint32_t (&w)[RowType<kType>::kWords]) {
  constexpr int kBytes = RowType<kType>::kBytes;
#pragma unroll
  for (int i = 0; i < RowType<kType>::kWords; ++i) w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= left) break;
    if constexpr (kBytes == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    else if constexpr (kBytes == 2) w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
    else w[i / 4] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(p)[i]) << (8 * (i & 3));
  }
}

// Elements (0, 4), (1, 5), (2, 6) and (3, 7) of eight as pairs: the order in which a word's 4-bit codes come apart.
template <int kType>
__device__ __forceinline__ void split_x(const uint32_t (&w)[RowType<kType>::kWords], uint32_t (&b)[RowType<kType>::kParts][4]) {
  if constexpr (kType == MMFREE_T_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo = w[i], hi = w[i + 4];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        b[p][i] = __byte_perm(lo, hi, 0x7632);  // the upper halves: the leading 8 bits of each, truncated
        if (p < 2) {                            // what is left of each, exact
          lo = __float_as_uint(__uint_as_float(lo) - __uint_as_float(lo & 0xFFFF0000u));
          hi = __float_as_uint(__uint_as_float(hi) - __uint_as_float(hi & 0xFFFF0000u));
        }
      }
    }
  } else if constexpr (RowType<kType>::kBytes == 2) {
    b[0][0] = __byte_perm(w[0], w[2], 0x5410);
    b[0][1] = __byte_perm(w[0], w[2], 0x7632);
    b[0][2] = __byte_perm(w[1], w[3], 0x5410);
    b[0][3] = __byte_perm(w[1], w[3], 0x7632);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t two = static_cast<uint16_t>(__byte_perm(w[0], w[1], i | ((4 + i) << 4)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b[0][i]) : "h"(two));
    }
  }
}

// A word's eight 4-bit codes minus the zero point as four pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <bool kBf16>
__device__ __forceinline__ void split_codes(uint32_t u, uint32_t zero, uint32_t zero16, uint32_t (&p)[4]) {
  if constexpr (kBf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = b2_sub((u >> (4 * i) & 0x000F000Fu) | 0x43004300u, zero);  // 0x430n is 128 + n
  } else {
    // 0x640n is 1024 + n, 0x64n0 is 1024 + 16 n: the second needs no shift, (1024 + 16 n) / 16 - (64 + z) is exact
    p[0] = h2_sub((u & 0x000F000Fu) | 0x64006400u, zero);
    p[1] = h2_fma((u & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, zero16);
    u >>= 8;
    p[2] = h2_sub((u & 0x000F000Fu) | 0x64006400u, zero);
    p[3] = h2_fma((u & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, zero16);
  }
}

template <bool kBf16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of which the first `bytes` are read and the others become 0.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <int kTiles, bool kAligned>
struct Int4Shape {
  static constexpr int kBlocks = 2, kRows = 16 * kBlocks;  // weight rows of a CTA at a time
  static constexpr int kCols = 8 * kTiles;                 // activation rows
  static constexpr int kChunks = kAligned ? 8 : 9;         // 16-byte chunks of a row and turn
  static constexpr int kCtas = kTiles == 4 ? 1 : 2;        // an SM
  static constexpr int kStages = kTiles == 4 ? 3 : 2;
  struct Warp {
    uint4 codes[kStages][kRows][kChunks];
    float scale[kTurnRuns][kRows];
    uint32_t zero[kTurnRuns][kRows];
  };
  struct Shared {
    Warp warp[kWarps];
    float part[kWarps][kCols][kPitch];
    int nan;  // fp32 rows: whether an output was one
  };
};

__device__ __forceinline__ float get_out(const void* p, int type, int64_t i) {
  switch (type) {
    case MMFREE_T_F32: return static_cast<const float*>(p)[i];
    case MMFREE_T_BF16: return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
    default: return to_f32(static_cast<const __half*>(p)[i]);
  }
}

// Outputs of fp32 rows that came out as NaN, once more from the definition in 64 bits, each by the thread that stored it. An
// infinity's first part is the infinity and its second infinity minus infinity, so its row's outputs are all NaN at first;
// telling it apart where rows are cut made calls 8 to 19% slower.
__device__ __forceinline__ void nan_outputs(const Int4Args& a, int splits, int m0, int live) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x % splits;
  for (int64_t n = static_cast<int64_t>(blockIdx.x / splits) * 32 + lane; n < a.N; n += static_cast<int64_t>(gridDim.x / splits) * 32)
    for (int m = rank * kWarps + warp; m < live; m += splits * kWarps) {
      const int64_t at = static_cast<int64_t>(m0 + m) * a.N + n;
      if (!isnan(get_out(a.out, a.out_type, at))) continue;
      const float* const x = static_cast<const float*>(a.x) + static_cast<int64_t>(m0 + m) * a.ldx;
      const uint8_t* const codes = a.codes + n * a.ldw;
      double total = 0.0;
      for (int g = 0; g < a.parts; ++g) {
        const int64_t of = n * a.parts + g;
        const int zero = a.zeros ? a.zeros[of] : 8, stop = min(static_cast<int64_t>(a.K), (g + int64_t(1)) * a.group);
        double part = 0.0;
        for (int k = g * a.group; k < stop; ++k) part += static_cast<double>((codes[k >> 1] >> (4 * (k & 1)) & 15) - zero) * x[k];
        total += part * get_out(a.scales, a.scale_type, of);
        if (isnan(total)) break;  // whatever follows
      }
      put_out(a.out, a.out_type, at, static_cast<float>(total));
    }
}

// A CTA: 32 weight rows and 8 * kTiles activation rows at a time; its warps (and those of the other CTAs of its
// cluster) split the columns into turns of kTileK. The row blocks are walked by a fixed grid.
// kAligned: the rows of the codes start at multiples of 16 bytes. Otherwise the aligned chunks that a row's turn
// touches are copied (a chunk with a byte of the row in it can be read as a whole) and its words put together from
// two, shifted by the row's own offset.
template <int kType, int kTiles, bool kAligned>
__global__ void __launch_bounds__(32 * kWarps, Int4Shape<kTiles, kAligned>::kCtas) int4_kernel(Int4Args a, int splits, int m0, bool xvec, uint32_t group_inverse) {
  using X = RowType<kType>;
  using S = Int4Shape<kTiles, kAligned>;
  constexpr int kBlocks = S::kBlocks, kRows = S::kRows, kCols = S::kCols, kChunks = S::kChunks, kStages = S::kStages;
  extern __shared__ __align__(16) char smem_raw[];
  auto& sh = *reinterpret_cast<typename S::Shared*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  auto& mine = sh.warp[warp];
  const int rank = blockIdx.x % splits, step = gridDim.x / splits;
  const int K = a.K, turns = (K + kTileK - 1) / kTileK, blocks = (a.N + kRows - 1) / kRows, bytes = (K + 1) / 2;
  const int stride = kWarps * splits, first = rank * kWarps + warp;
  const int live = min(kCols, a.M - m0);
  const char* const x = static_cast<const char*>(a.x) + static_cast<int64_t>(m0) * a.ldx * X::kBytes;

  if (kType == MMFREE_T_F32 && threadIdx.x == 0) sh.nan = 0;  // set behind the first block's barrier

  // k / group: columns are below 2^16, where the high word of the product with ceil(2^32 / group) is exact
  const auto group_of = [&](int k) { return static_cast<int>(__umulhi(static_cast<uint32_t>(k), group_inverse)); };

  // the next turn to copy
  int copy_block = blockIdx.x / splits, copy_turn = first, copied = 0;
  const auto copy = [&] {
    if (copy_block < blocks && first < turns) {
      const uint32_t to = smem_u32(&mine.codes[copied % kStages][0][0]);
      const int from = copy_turn * (kTileK / 2), n0 = copy_block * kRows;
      if constexpr (kAligned) {
        // lane: chunk lane % 8 of every fourth row; chunks of a row are exchanged by the row, so that 8 rows' words of
        // one column are on different banks
        const int c = lane & 7, at = from + 16 * c, left = min(max(bytes - at, 0), 16);
        const uint8_t* line = a.codes + (n0 + (lane >> 3)) * a.ldw + (left ? at : 0);
        const int64_t rows4 = 4 * a.ldw;
#pragma unroll
        for (int i = 0; i < kRows / 4; ++i, line += rows4) {
          const int row = (lane >> 3) + 4 * i;
          if (n0 + row >= a.N) break;  // rows behind the last: what the stage held
          copy16(to + (row * 8 + (c ^ (row & 7))) * 16, line, left);
        }
      } else {
        for (int i = lane; i < kRows * kChunks; i += 32) {
          const int row = i / kChunks, c = i % kChunks;
          const uint8_t* const line = a.codes + min(n0 + row, a.N - 1) * a.ldw;
          const uintptr_t at = (reinterpret_cast<uintptr_t>(line + from) & ~uintptr_t(15)) + 16 * c;
          const bool any = at < reinterpret_cast<uintptr_t>(line + bytes);
          copy16(to + i * 16, reinterpret_cast<const void*>(any ? at : reinterpret_cast<uintptr_t>(line) & ~uintptr_t(15)), any ? 16 : 0);
        }
      }
      if ((copy_turn += stride) >= turns) copy_turn = first, copy_block += step;
    }
    ++copied;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // scales and zero points of a turn: lane r has row r's, of up to 8 groups, as they lie in memory
  uint32_t next_scale[kTurnRuns], next_zero[kTurnRuns];
  int next_groups = 0;
  const bool wide_scales = a.scale_type == MMFREE_T_F32;
  const auto fetch = [&](int block, int turn) {
    const int g0 = group_of(turn * kTileK), g1 = min(a.parts - 1, group_of(turn * kTileK + kTileK - 1));
    const int64_t at = static_cast<int64_t>(min(block * kRows + lane, a.N - 1)) * a.parts + g0;
    const char* const p = static_cast<const char*>(a.scales) + at * (wide_scales ? 4 : 2);
    next_groups = g1 - g0 + 1;
#pragma unroll
    for (int i = 0; i < kTurnRuns; ++i) {
      if (i >= next_groups) break;
      next_scale[i] = wide_scales ? reinterpret_cast<const uint32_t*>(p)[i] : reinterpret_cast<const uint16_t*>(p)[i];
      next_zero[i] = a.zeros ? a.zeros[at + i] : 8u;
    }
  };
  const auto keep = [&] {
#pragma unroll
    for (int i = 0; i < kTurnRuns; ++i) {
      if (i >= next_groups) break;
      mine.scale[i][lane] = a.scale_type == MMFREE_T_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(next_scale[i])))
                                                         : __uint_as_float(next_scale[i] << (wide_scales ? 0 : 16));
      if (X::kBf16 && next_zero[i] > 127) atomicOr(&g_zero_point_error, kErrRange);
      // 128 + z (up to z = 127 exact) or 1024 + z twice: 0x4300 + z is 128 + z in bf16, 0x6400 + z is 1024 + z in fp16
      mine.zero[i][lane] = (X::kBf16 ? 0x43004300u : 0x64006400u) + next_zero[i] * 0x10001u;
    }
  };
#pragma unroll
  for (int i = 0; i < kTurnRuns; ++i) next_scale[i] = next_zero[i] = 0;
#pragma unroll
  for (int i = 0; i + 1 < kStages; ++i) copy();
  if (blockIdx.x / splits < blocks && first < turns) fetch(blockIdx.x / splits, first);
  int item = 0;
  for (int block = blockIdx.x / splits; block < blocks; block += step) {
    float total[kBlocks][kTiles][4] = {};
    int offset[kBlocks][2];  // !kAligned: of the rows' first bytes in their chunks
    if constexpr (!kAligned) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          offset[b][h] = static_cast<int>(reinterpret_cast<uintptr_t>(a.codes + min(block * kRows + 16 * b + 8 * h + g, a.N - 1) * a.ldw) & 15);
    }
    for (int turn = first; turn < turns; turn += stride, ++item) {
      __syncwarp();  // every lane is done with the stage that the next copy fills, and with the scales
      copy();
      keep();
      if (turn + stride < turns) fetch(block, turn + stride);
      else if (block + step < blocks) fetch(block + step, first);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint32_t* const words = reinterpret_cast<const uint32_t*>(&mine.codes[item % kStages][0][0]);
      const int k0 = turn * kTileK, runs = min(kTurnRuns, (K - k0 + 31) / 32), g0 = group_of(k0);
      // a whole turn of aligned rows is read without a test (lanes of absent rows read the last one: their columns of
      // the result are not stored)
      const bool whole = xvec && k0 + kTileK <= K;
      const char* xp[kTiles];
#pragma unroll
      for (int c = 0; c < kTiles; ++c) xp[c] = x + (static_cast<int64_t>(min(8 * c + g, live - 1)) * a.ldx + k0 + 8 * t) * X::kBytes;
      int r = 0;
#pragma unroll 1
      for (int group = 0; r < runs; ++group) {
        const int stop = min(runs, ((g0 + group + 1) * a.group - k0) / 32);
        float part[kBlocks][kTiles][4] = {};
        constexpr bool kWhole = kType == MMFREE_T_S8;
        int whole_part[kBlocks][kTiles][4] = {}, xsum[kTiles][4] = {};  // kWhole
        uint32_t zero[kBlocks][2], zero16[kBlocks][2];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            zero[b][h] = mine.zero[group][16 * b + 8 * h + g];
            zero16[b][h] = X::kBf16 ? 0 : h2_sub(0x63806380u, zero[b][h]);  // 960 - (1024 + z)
          }
        const auto word = [&](int b, int h) {
          const int row = 16 * b + 8 * h + g;
          if constexpr (kAligned) return words[row * kChunks * 4 + (((r ^ g) & 7) * 4 + t)];
          const int at = row * kChunks * 4 + r * 4 + t + (offset[b][h] >> 2);
          return __funnelshift_r(words[at], words[min(at + 1, kRows * kChunks * 4 - 1)], 8 * (offset[b][h] & 3));
        };
        const auto run = [&](const uint32_t (&xw)[kTiles][X::kWords]) {
          if constexpr (kWhole) {
            // a word's codes 0, 2, 4, 6 and 1, 3, 5, 7 as bytes, and the row's columns in that order
            uint32_t x0[kTiles], x1[kTiles];
#pragma unroll
            for (int c = 0; c < kTiles; ++c) {
              x0[c] = __byte_perm(xw[c][0], xw[c][1], 0x6420);
              x1[c] = __byte_perm(xw[c][0], xw[c][1], 0x7531);
              mma_u8s8(xsum[c], 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, x0[c], x1[c]);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              const uint32_t u0 = word(b, 0), u1 = word(b, 1), even = 0x0F0F0F0Fu;
#pragma unroll
              for (int c = 0; c < kTiles; ++c)
                mma_u8s8(whole_part[b][c], u0 & even, u1 & even, (u0 >> 4) & even, (u1 >> 4) & even, x0[c], x1[c]);
            }
            return;
          }
          uint32_t xb[kTiles][X::kParts][4];
#pragma unroll
          for (int c = 0; c < kTiles; ++c) split_x<kType>(xw[c], xb[c]);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            uint32_t p[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) split_codes<X::kBf16>(word(b, h), zero[b][h], zero16[b][h], p[h]);
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
              for (int q = 0; q < X::kParts; ++q) {
                mma<X::kBf16>(part[b][c], p[0][0], p[1][0], p[0][1], p[1][1], xb[c][q][0], xb[c][q][1]);
                mma<X::kBf16>(part[b][c], p[0][2], p[1][2], p[0][3], p[1][3], xb[c][q][2], xb[c][q][3]);
              }
          }
        };
        uint32_t xw[kTiles][X::kWords];
        if (whole) {
          // each run's rows are loaded a run ahead
          uint32_t ahead[kTiles][X::kWords];
#pragma unroll
          for (int c = 0; c < kTiles; ++c) load_x<kType>(xp[c] + 32 * X::kBytes * r, ahead[c]);
#pragma unroll 2
          for (; r < stop; ++r) {
            const int next = min(r + 1, kTurnRuns - 1);
#pragma unroll
            for (int c = 0; c < kTiles; ++c) {
#pragma unroll
              for (int i = 0; i < X::kWords; ++i) xw[c][i] = ahead[c][i];
              load_x<kType>(xp[c] + 32 * X::kBytes * next, ahead[c]);
            }
            run(xw);
          }
        } else {
#pragma unroll 1
          for (; r < stop; ++r) {
#pragma unroll
            for (int c = 0; c < kTiles; ++c) load_x_part<kType>(xp[c] + 32 * X::kBytes * r, K - (k0 + 32 * r + 8 * t), xw[c]);
            run(xw);
          }
        }
        // the group's sums, scaled: rows g and g + 8, columns (activation rows) 2 t and 2 t + 1
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
          float xs[2] = {1.0f, 1.0f};
          if (a.x_grouped)
#pragma unroll
            for (int j = 0; j < 2; ++j) xs[j] = a.x_scales[static_cast<int64_t>(m0 + min(8 * c + 2 * t + j, live - 1)) * a.parts + g0 + group];
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
              if constexpr (kWhole)  // the zero point is the low byte of 1024 + z
                part[b][c][j] = static_cast<float>(whole_part[b][c][j] - static_cast<int>(zero[b][j >> 1] & 0xFFu) * xsum[c][j & 1]);
              total[b][c][j] = fmaf(mine.scale[group][16 * b + 8 * (j >> 1) + g], part[b][c][j] * xs[j & 1], total[b][c][j]);
            }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) sh.part[warp][8 * c + 2 * t + (j & 1)][16 * b + 8 * (j >> 1) + g] = total[b][c][j];
    __syncthreads();
    // the warps' sums, always in the same order; in a cluster, into the first warp's place for the other CTAs
    const auto put = [&](int m, float v) {
      const int n = block * kRows + lane;
      if (m >= live || n >= a.N) return;
      if (kType == MMFREE_T_F32 && isnan(v)) sh.nan = 1;
      if (a.x_scales && !a.x_grouped) v *= a.x_scales[m0 + m];
      put_out(a.out, a.out_type, static_cast<int64_t>(m0 + m) * a.N + n, v);
    };
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int m = warp + kWarps * i;
      if (m >= live) break;
      float v = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) v += sh.part[q][m][lane];
      if (splits == 1) put(m, v);
      else sh.part[0][m][lane] = v;  // row m is read by this warp alone before
    }
    if (splits == 1) {
      __syncthreads();
    } else {
      cluster_sync();
      for (int m = rank * kWarps + warp; m < live; m += splits * kWarps) {
        const uint32_t at = smem_u32(&sh.part[0][m][lane]);
        float v = 0.0f;
        for (int q = 0; q < splits; ++q) {
          float o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(cluster_map(at, q)) : "memory");
          v += o;
        }
        put(m, v);
      }
      cluster_sync();  // before a peer's sums are written again, or its CTA ends
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (kType == MMFREE_T_F32)
    if (sh.nan) nan_outputs(a, splits, m0, live);  // set before the last block's barrier
}

template <int kType, int kTiles, bool kAligned>
cudaError_t int4_launch(const Int4Args& a, int sms, int m0, bool xvec, cudaStream_t s) {
  const int blocks = static_cast<int>(ceil_div(a.N, 32)), turns = static_cast<int>(ceil_div(a.K, kTileK));
  // Columns split over a cluster's CTAs as long as that leaves every warp a turn and the CTAs fit the SMs; by the
  // weights' shape alone, so that a row's sums do not depend on how many rows there are.
  int splits = 1;
  while (splits < 8 && blocks * splits * 2 <= 2 * sms && turns > kWarps * splits) splits *= 2;
  using S = Int4Shape<kTiles, kAligned>;
  const int wide = S::kCtas * sms / splits;
  constexpr size_t kSmem = sizeof(typename S::Shared);
  static_assert(S::kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory of the SM");
  const auto kernel = int4_kernel<kType, kTiles, kAligned>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((blocks < wide ? blocks : wide) * splits));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(splits);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  // a group of 2^16 columns or more is the only one
  const uint32_t inverse = a.group < 65536 ? static_cast<uint32_t>(((uint64_t(1) << 32) + a.group - 1) / a.group) : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, splits, m0, xvec, inverse);
}

template <int kType, bool kAligned>
cudaError_t int4_rows(const Int4Args& a, int sms, bool xvec, cudaStream_t s) {
  for (int m0 = 0; m0 < a.M; m0 += 32) {
    const int left = a.M - m0;
    const cudaError_t e = left <= 8    ? int4_launch<kType, 1, kAligned>(a, sms, m0, xvec, s)
                          : left <= 16 ? int4_launch<kType, 2, kAligned>(a, sms, m0, xvec, s)
                                       : int4_launch<kType, 4, kAligned>(a, sms, m0, xvec, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int kType>
cudaError_t int4_type(const Int4Args& a, int sms, cudaStream_t s) {
  const int xb = RowType<kType>::kBytes, chunk = xb == 1 ? 8 : 16;  // bytes of an access to x
  const bool xvec = reinterpret_cast<uintptr_t>(a.x) % chunk == 0 && (a.ldx * xb % chunk == 0 || a.M == 1);
  return aligned16(a.codes) && (a.ldw % 16 == 0 || a.N == 1) ? int4_rows<kType, true>(a, sms, xvec, s) : int4_rows<kType, false>(a, sms, xvec, s);
}

}  // namespace

cudaError_t take_zero_point_flags(cudaStream_t s, uint32_t* flags) { return take_word(g_zero_point_error, g_devices, s, flags); }

cudaError_t launch_int4_matvec(const Int4Args& a, int sm_count, cudaStream_t s) {
  g_devices.mark();
  switch (a.x_type) {
    case MMFREE_T_F32: return int4_type<MMFREE_T_F32>(a, sm_count, s);
    case MMFREE_T_BF16: return int4_type<MMFREE_T_BF16>(a, sm_count, s);
    case MMFREE_T_F16: return int4_type<MMFREE_T_F16>(a, sm_count, s);
    case MMFREE_T_S8: return int4_type<MMFREE_T_S8>(a, sm_count, s);
    default: return int4_type<MMFREE_T_E4M3>(a, sm_count, s);
  }
}

}  // namespace mmfree_cuda
