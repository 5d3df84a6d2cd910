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
// u - z is a small whole number, exact in fp16 and bf16; int8 and e4m3 rows are exact in fp16;
// fp32 rows are cut into three bf16 parts of 8 bits each, exactly. The products are therefore
// exact, summed in fp32, and a group's sum is scaled once.
//
// The order of a product's columns is free as long as weights and activations agree, so a lane
// takes runs of consecutive columns of its weight row: 16-byte loads straight from the row-major
// codes, no repacked copy of the weights.
#include "block_ops.h"
#include "common.cuh"
#include "elements.cuh"
#include "tcgen05.cuh"

#include <cuda_fp8.h>

namespace mmfree_cuda {

namespace {

constexpr int kWarps = 8;       // of a CTA: they share its weight rows and split the columns
constexpr int kTileK = 256;     // columns of a warp's turn (128 bytes of a weight row)
constexpr int kPitch = 36;      // words of a partial-sum row of 32 outputs: keeps its writers on different banks

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

// Eight elements of a row from column k, `left` of them inside it (the others are 0).
template <int kType, bool kVec>
__device__ __forceinline__ void load_x(const char* row, int k, int left, uint32_t (&w)[RowType<kType>::kWords]) {
  constexpr int kBytes = RowType<kType>::kBytes, kWords = RowType<kType>::kWords;
  if (kVec && left >= 8) {
    const char* p = row + static_cast<int64_t>(k) * kBytes;
    if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= left) break;
    if constexpr (kBytes == 4) w[i] = reinterpret_cast<const uint32_t*>(row)[k + i];
    else if constexpr (kBytes == 2) w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k + i]) << (16 * (i & 1));
    else w[i / 4] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(row)[k + i]) << (8 * (i & 3));
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
  } else if constexpr (kType == MMFREE_T_S8) {
    const uint32_t lo = w[0] ^ 0x80808080u, hi = w[1] ^ 0x80808080u;  // x + 128 in 0..255
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // 0x64nn is 1024 + nn in fp16
      const uint32_t v = (__byte_perm(lo, hi, i | ((4 + i) << 8)) & 0x00FF00FFu) | 0x64006400u;
      b[0][i] = h2_sub(v, 0x64806480u);
    }
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

// kRun consecutive columns of a weight row from column k.
template <int kRun, bool kVec>
__device__ __forceinline__ void load_codes(const uint8_t* row, int k, int K, uint32_t (&w)[kRun / 8]) {
  const uint8_t* p = row + k / 2;
  if (kVec && k + kRun <= K) {
    if constexpr (kRun == 32) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kRun == 16) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return;
  }
  const int bytes = (K - k + 1) / 2;  // left in the row
#pragma unroll
  for (int i = 0; i < kRun / 8; ++i) {
    w[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * i + j < bytes) w[i] |= static_cast<uint32_t>(p[4 * i + j]) << (8 * j);
  }
}

// A CTA: kBlocks blocks of 16 weight rows and 8 * kTiles activation rows at a time; its warps (and those of the other
// CTAs of its cluster) split the columns into turns of kTileK. kRun: consecutive columns of a lane, so that the 4
// lanes of a row cover 4 * kRun columns of ONE group: 32 (16-byte loads) where the group is a multiple of 128
// columns, 16 for 64, else 8. The row blocks are walked by a fixed grid, the next turn's weights loaded while this
// one's are multiplied.
template <int kType, int kTiles, int kRun, bool kVec>
__global__ void __launch_bounds__(32 * kWarps, kTiles == 4 ? 1 : 2) int4_kernel(Int4Args a, int splits, int m0) {
  using X = RowType<kType>;
  constexpr int kBlocks = 2, kRows = 16 * kBlocks, kCols = 8 * kTiles, kRuns = kTileK / (4 * kRun), kWordsRun = kRun / 8;
  constexpr int kBuffers = kTiles == 4 ? 1 : 2;  // two save a barrier a block where they fit
  __shared__ float s_part[kBuffers][kWarps][kCols][kPitch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % splits;
  const int K = a.K, turns = (K + kTileK - 1) / kTileK, blocks = (a.N + kRows - 1) / kRows;
  const int stride = kWarps * splits, first = rank * kWarps + warp;
  const int live = min(kCols, a.M - m0);
  // the activation row of this lane's operand in each tile (rows behind the last are not read)
  const char* xrow[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) xrow[i] = static_cast<const char*>(a.x) + (m0 + 8 * i + g) * a.ldx * X::kBytes;

  uint32_t w[kBlocks][2][kRuns][kWordsRun];
  const auto fetch = [&](int block, int turn) {
    if (block >= blocks || turn >= turns) return;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = min(block * kRows + 16 * b + 8 * h + g, a.N - 1);
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
          const int k = turn * kTileK + r * 4 * kRun + t * kRun;
          if (k < K) {
            load_codes<kRun, kVec>(a.codes + n * a.ldw, k, K, w[b][h][r]);
          } else {
#pragma unroll
            for (int i = 0; i < kWordsRun; ++i) w[b][h][r][i] = 0;
          }
        }
      }
  };
  const int step = gridDim.x / splits;
  int buf = 0;
  fetch(blockIdx.x / splits, first);
  for (int block = blockIdx.x / splits; block < blocks; block += step, buf = (buf + 1) % kBuffers) {
    float total[kBlocks][kTiles][4] = {};
    for (int turn = first; turn < turns; turn += stride) {
      uint32_t u[kBlocks][2][kRuns][kWordsRun];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < kRuns; ++r)
#pragma unroll
            for (int i = 0; i < kWordsRun; ++i) u[b][h][r][i] = w[b][h][r][i];
      if (turn + stride < turns) fetch(block, turn + stride);
      else fetch(block + step, first);
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const int k0 = turn * kTileK + r * 4 * kRun, k = k0 + t * kRun;
        if (k0 >= K) break;
        const int group = k0 / a.group;
        float part[kBlocks][kTiles][4] = {};
        uint32_t zero[kBlocks][2], zero16[kBlocks][2];
        float scale[kBlocks][2];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t at = static_cast<int64_t>(min(block * kRows + 16 * b + 8 * h + g, a.N - 1)) * a.parts + group;
            scale[b][h] = scale_value(a.scales, a.scale_type, at);
            const uint32_t z = a.zeros ? a.zeros[at] & 255u : 8u;
            if constexpr (X::kBf16) {
              // 128 + z, rounded where z is above 127 (a zero point is meant to be 0..15)
              const uint32_t v = __bfloat16_as_ushort(__float2bfloat16_rn(128.0f + static_cast<float>(z)));
              zero[b][h] = v | v << 16;
              zero16[b][h] = 0;
            } else {
              const uint32_t v = __half_as_ushort(__float2half_rn(1024.0f + static_cast<float>(z)));
              const uint32_t v16 = __half_as_ushort(__float2half_rn(-64.0f - static_cast<float>(z)));
              zero[b][h] = v | v << 16;
              zero16[b][h] = v16 | v16 << 16;
            }
          }
#pragma unroll
        for (int i = 0; i < kWordsRun; ++i) {
          uint32_t xb[kTiles][X::kParts][4];
#pragma unroll
          for (int c = 0; c < kTiles; ++c) {
            uint32_t xw[X::kWords];
            const int left = 8 * c + g < live ? K - (k + 8 * i) : 0;
            load_x<kType, kVec>(xrow[c], k + 8 * i, left, xw);
            split_x<kType>(xw, xb[c]);
          }
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            uint32_t p0[4], p1[4];
            split_codes<X::kBf16>(u[b][0][r][i], zero[b][0], zero16[b][0], p0);
            split_codes<X::kBf16>(u[b][1][r][i], zero[b][1], zero16[b][1], p1);
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
              for (int q = 0; q < X::kParts; ++q) {
                mma<X::kBf16>(part[b][c], p0[0], p1[0], p0[1], p1[1], xb[c][q][0], xb[c][q][1]);
                mma<X::kBf16>(part[b][c], p0[2], p1[2], p0[3], p1[3], xb[c][q][2], xb[c][q][3]);
              }
          }
        }
        // the group's sums, scaled: rows g and g + 8, columns (activation rows) 2 t and 2 t + 1
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
          float xs[2] = {1.0f, 1.0f};
          if (a.x_grouped)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int m = 8 * c + 2 * t + j;
              xs[j] = m < live ? a.x_scales[static_cast<int64_t>(m0 + m) * a.parts + group] : 0.0f;
            }
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) total[b][c][j] = fmaf(scale[b][j >> 1] * xs[j & 1], part[b][c][j], total[b][c][j]);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_part[buf][warp][8 * c + 2 * t + (j & 1)][16 * b + 8 * (j >> 1) + g] = total[b][c][j];
    __syncthreads();
    // the warps' sums, always in the same order; in a cluster, into the first warp's place for the other CTAs
    const auto put = [&](int m, float v) {
      const int n = block * kRows + lane;
      if (m >= live || n >= a.N) return;
      if (a.x_scales && !a.x_grouped) v *= a.x_scales[m0 + m];
      put_out(a.out, a.out_type, static_cast<int64_t>(m0 + m) * a.N + n, v);
    };
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int m = warp + kWarps * i;
      float v = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) v += s_part[buf][q][m][lane];
      if (splits == 1) put(m, v);
      else s_part[buf][0][m][lane] = v;  // read by this warp alone before
    }
    if (splits > 1) {
      cluster_sync();
      for (int m = rank * kWarps + warp; m < kCols; m += splits * kWarps) {
        const uint32_t at = smem_u32(&s_part[buf][0][m][lane]);
        float v = 0.0f;
        for (int q = 0; q < splits; ++q) {
          float o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(cluster_map(at, q)) : "memory");
          v += o;
        }
        put(m, v);
      }
      cluster_sync();  // before a peer's buffer is written again, or its CTA ends
    } else if (kBuffers == 1) {
      __syncthreads();
    }
  }
}

template <int kType, int kTiles, int kRun, bool kVec>
cudaError_t int4_launch(const Int4Args& a, int sms, int m0, cudaStream_t s) {
  const int blocks = static_cast<int>(ceil_div(a.N, 32)), turns = static_cast<int>(ceil_div(a.K, kTileK));
  // Columns split over a cluster's CTAs as long as that leaves every warp a turn and the CTAs fit the SMs; by the
  // weights' shape alone, so that a row's sums do not depend on how many rows there are.
  int splits = 1;
  while (splits < 8 && blocks * splits * 2 <= 2 * sms && turns > kWarps * splits) splits *= 2;
  const int wide = 2 * sms / splits;
  const int ctas = (blocks < wide ? blocks : wide) * splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(splits);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, int4_kernel<kType, kTiles, kRun, kVec>, a, splits, m0);
}

template <int kType, int kRun, bool kVec>
cudaError_t int4_rows(const Int4Args& a, int sms, cudaStream_t s) {
  for (int m0 = 0; m0 < a.M; m0 += 32) {
    const int left = a.M - m0;
    const cudaError_t e = left <= 8    ? int4_launch<kType, 1, kRun, kVec>(a, sms, m0, s)
                          : left <= 16 ? int4_launch<kType, 2, kRun, kVec>(a, sms, m0, s)
                                       : int4_launch<kType, 4, kRun, kVec>(a, sms, m0, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int kType>
cudaError_t int4_type(const Int4Args& a, int sms, cudaStream_t s) {
  const int run = a.group % 128 == 0 ? 32 : a.group % 64 == 0 ? 16 : 8;
  const int xb = RowType<kType>::kBytes, chunk = xb == 1 ? 8 : 16;  // bytes of an access to x
  const bool vec = reinterpret_cast<uintptr_t>(a.codes) % (run / 2) == 0 && (a.ldw % (run / 2) == 0 || a.N == 1) &&
                   reinterpret_cast<uintptr_t>(a.x) % chunk == 0 && (a.ldx * xb % chunk == 0 || a.M == 1);
  if (run == 32) return vec ? int4_rows<kType, 32, true>(a, sms, s) : int4_rows<kType, 32, false>(a, sms, s);
  if (run == 16) return vec ? int4_rows<kType, 16, true>(a, sms, s) : int4_rows<kType, 16, false>(a, sms, s);
  return vec ? int4_rows<kType, 8, true>(a, sms, s) : int4_rows<kType, 8, false>(a, sms, s);
}

}  // namespace

cudaError_t launch_int4_matvec(const Int4Args& a, int sm_count, cudaStream_t s) {
  switch (a.x_type) {
    case MMFREE_T_F32: return int4_type<MMFREE_T_F32>(a, sm_count, s);
    case MMFREE_T_BF16: return int4_type<MMFREE_T_BF16>(a, sm_count, s);
    case MMFREE_T_F16: return int4_type<MMFREE_T_F16>(a, sm_count, s);
    case MMFREE_T_S8: return int4_type<MMFREE_T_S8>(a, sm_count, s);
    default: return int4_type<MMFREE_T_E4M3>(a, sm_count, s);
  }
}

}  // namespace mmfree_cuda
