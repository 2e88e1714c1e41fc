// Kernels of the logits head with 4-bit weights (include/et_logit_head.h).
//
//   y[m, v] = sum_g s[v, g] * (sum_{k in g} x[m, k] (n[v, k] - 8)) + z[v, g] * (sum_{k in g} x[m, k])
//
// The inner sums run on the matrix cores with the nibbles as operands, exactly: the bit pattern of 16 + n in
// bf16 or fp16 is a constant with n in the top four mantissa bits, so a shift and an and-or make two weights
// from a register of packed ones.  sum x (16 + n) - 24 sum x = sum x (n - 8): the second term, the same for
// every vocabulary row, is one more matrix product with a constant operand, and the accumulators start from
// it.  Scales and zeros are applied to the fp32 sums of a group.  fp32 hidden states are split into three
// bf16 parts that add up to them exactly.
//
// Weight layout: blocks of 16 vocabulary rows x 128 columns, 1 KiB, the 16 bytes of a lane next to each
// other: lane (q, n) = 16 q + n holds row n of the block, its dword t the columns 32 t + 8 q + 0..7 (operand
// B of the t-th 16x16x32 product), the column 8 q + 2 i + h at bits 16 h + 4 i.  A wave reads a block with
// one 16-byte load per lane.
#pragma once

#include "ets_device.h"

namespace ets {

constexpr int kHeadBlock = 256;  // lanes of a workgroup
constexpr int kTileRows = 16;    // vocabulary rows of a block
constexpr int kChunkCols = 128;  // columns of a block

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct HeadParams {
  const u32x4* blocks;  // [tiles, chunks, 64]
  const void* scales;   // [tiles, chunks, 16, groups per chunk], or [tiles, groups, 16] for groups of 128 columns and more
  const void* zeros;    // the same, or null
  int32_t scale_is_bf16;  // of 16-bit scales: bf16, else fp16
  int32_t tiles, chunks, chunks_per_group, groups;  // (the last two for groups of 128 columns and more)
  int32_t vocab, hidden, rows;
  const void* x;
  int64_t x_stride;
  void* out;
  int64_t out_stride;
  int32_t out_dtype;
};

// ---- operands -----------------------------------------------------------------------------------
template <int XT>
struct Matrix {  // bf16, and fp32 as three bf16 parts
  static constexpr uint32_t kBase = 0x41804180u, kMask = 0x00780078u;  // 16 + n: n at mantissa bits 3..6
  static constexpr int kTop = 3;
  static constexpr uint32_t kOne = 0x3f803f80u, kMinus24 = 0xc1c0c1c0u;
  static __device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Matrix<kDtypeHalf> {
  static constexpr uint32_t kBase = 0x4c004c00u, kMask = 0x03c003c0u;  // n at mantissa bits 6..9
  static constexpr int kTop = 6;
  static constexpr uint32_t kOne = 0x3c003c00u, kMinus24 = 0xce00ce00u;
  static __device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// Eight packed weights as an operand: 16 + n each.
template <int XT>
__device__ __forceinline__ u32x4 unpack(uint32_t w) {
  using M = Matrix<XT>;
  u32x4 b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int shift = 4 * i - M::kTop;
    b[i] = ((shift < 0 ? w << -shift : w >> shift) & M::kMask) | M::kBase;
  }
  return b;
}

template <int XT>
struct Parts {
  static constexpr int value = XT == kDtypeFloat ? 3 : 1;
};

struct __attribute__((packed, aligned(2))) LooseHalves {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) LooseFloats {
  float f[8];
};

// Columns [k, k + 8) of a row of x as operand A (one per part); columns at `hidden` and behind, and rows that
// do not exist, read as 0.
template <int XT>
__device__ __forceinline__ void load_x(const void* row, int k, int hidden, bool exists, u32x4* part) {
  if (XT == kDtypeFloat) {
    const float* f = static_cast<const float*>(row) + k;
    float v[8];
    if (exists && k + 8 <= hidden) {
      const LooseFloats r = *reinterpret_cast<const LooseFloats*>(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r.f[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (exists && k + j < hidden) ? f[j] : 0.0f;
    }
    // x = high + middle + low, each cut off to the upper 16 bits of a float: exact, 8 bits of x at a time
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[j] = __float_as_uint(v[j]) & 0xffff0000u;
      const float rest = v[j] - __uint_as_float(h[j]);
      m[j] = __float_as_uint(rest) & 0xffff0000u;
      l[j] = __float_as_uint(rest - __uint_as_float(m[j]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      part[0][i] = (h[2 * i] >> 16) | h[2 * i + 1];
      part[Parts<XT>::value / 2][i] = (m[2 * i] >> 16) | m[2 * i + 1];
      part[Parts<XT>::value - 1][i] = (l[2 * i] >> 16) | (l[2 * i + 1] & 0xffff0000u);
    }
  } else {
    const uint16_t* u = static_cast<const uint16_t*>(row) + k;
    if (exists && k + 8 <= hidden) {
      const LooseHalves r = *reinterpret_cast<const LooseHalves*>(u);
#pragma unroll
      for (int i = 0; i < 4; ++i) part[0][i] = r.w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (exists && k + 2 * i < hidden) ? u[2 * i] : 0u;
        const uint32_t hi = (exists && k + 2 * i + 1 < hidden) ? u[2 * i + 1] : 0u;
        part[0][i] = lo | (hi << 16);
      }
    }
  }
}

// The scales (or zeros) of this lane's vocabulary row for the GPC groups of a chunk.
template <int GPC, int SB>
__device__ __forceinline__ void load_scales(const void* base, const HeadParams& p, int tile, int chunk, int n, float* s) {
  const int64_t at = GPC > 1 ? ((static_cast<int64_t>(tile) * p.chunks + chunk) * kTileRows + n) * GPC
                             : (static_cast<int64_t>(tile) * p.groups + chunk / p.chunks_per_group) * kTileRows + n;
  if (SB == 4) {
    struct alignas(4 * GPC) Raw { float f[GPC]; };
    const Raw r = *reinterpret_cast<const Raw*>(static_cast<const float*>(base) + at);
#pragma unroll
    for (int g = 0; g < GPC; ++g) s[g] = r.f[g];
  } else {
    struct alignas(2 * GPC) Raw { uint16_t u[GPC]; };
    const Raw r = *reinterpret_cast<const Raw*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int g = 0; g < GPC; ++g) s[g] = p.scale_is_bf16 ? __uint_as_float(static_cast<uint32_t>(r.u[g]) << 16) : half_bits_to_float(r.u[g]);
  }
}

// The one rounding of the result, to nearest even.
__device__ __forceinline__ void store_logit(const HeadParams& p, int m, int v, float y) {
  const int64_t at = m * p.out_stride + v;
  if (p.out_dtype == kDtypeFloat) {
    static_cast<float*>(p.out)[at] = y;
  } else if (p.out_dtype == kDtypeBFloat16) {
    static_cast<__bf16*>(p.out)[at] = static_cast<__bf16>(y);
  } else {
    static_cast<_Float16*>(p.out)[at] = static_cast<_Float16>(y);
  }
}

// ---- the product --------------------------------------------------------------------------------
// A workgroup makes 16 rows x (16 NT) vocabulary entries; its four waves take the chunks of columns in turn
// and their sums are added up in a fixed order at the end.
template <int XT, int GPC, int SB, bool ZEROS, int NT>
__global__ void __launch_bounds__(kHeadBlock)
head_stream_kernel(const HeadParams p) {
  using M = Matrix<XT>;
  constexpr int P = Parts<XT>::value, kWavesHere = kHeadBlock / 64, kSteps = 4 / GPC;  // products per group of a chunk
  __shared__ float red[kWavesHere][NT][64 * 4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * 16;
  const bool exists = m0 + n < p.rows;
  const char* x_row = static_cast<const char*>(p.x) + (exists ? m0 + n : 0) * p.x_stride * ElemSize<XT>::value;
  const u32x4 minus24 = {M::kMinus24, M::kMinus24, M::kMinus24, M::kMinus24}, one = {M::kOne, M::kOne, M::kOne, M::kOne};
  f32x4 total[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) total[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int chunk = wave; chunk < p.chunks; chunk += kWavesHere) {
    u32x4 w[NT];
    float s[NT][GPC], z[NT][GPC];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int tile = min(tile0 + i, p.tiles - 1);  // (tiles behind the last one are computed again and not stored)
      w[i] = p.blocks[(static_cast<int64_t>(tile) * p.chunks + chunk) * 64 + lane];
      load_scales<GPC, SB>(p.scales, p, tile, chunk, n, s[i]);
      if (ZEROS) load_scales<GPC, SB>(p.zeros, p, tile, chunk, n, z[i]);
    }
    u32x4 x[4][P];
#pragma unroll
    for (int t = 0; t < 4; ++t) load_x<XT>(x_row, chunk * kChunkCols + 32 * t + 8 * q, p.hidden, exists, x[t]);
#pragma unroll
    for (int g = 0; g < GPC; ++g) {
      f32x4 base = {0.0f, 0.0f, 0.0f, 0.0f}, sums = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = g * kSteps; t < (g + 1) * kSteps; ++t) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          base = M::product(x[t][k], minus24, base);
          if (ZEROS) sums = M::product(x[t][k], one, sums);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f32x4 acc = base;
#pragma unroll
        for (int t = g * kSteps; t < (g + 1) * kSteps; ++t) {
          const u32x4 b = unpack<XT>(w[i][t]);
#pragma unroll
          for (int k = 0; k < P; ++k) acc = M::product(x[t][k], b, acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          total[i][r] = fmaf(s[i][g], acc[r], total[i][r]);
          if (ZEROS) total[i][r] = fmaf(z[i][g], sums[r], total[i][r]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) *reinterpret_cast<f32x4*>(&red[wave][i][lane * 4]) = total[i];
  __syncthreads();
  // row m of the tile is element m & 3 of the lanes 16 (m >> 2) + column
  for (int e = tid; e < NT * 256; e += kHeadBlock) {
    const int col = e & (16 * NT - 1), m = e / (16 * NT);
    const int at = ((m >> 2) * 16 + (col & 15)) * 4 + (m & 3);
    float y = red[0][col >> 4][at];
#pragma unroll
    for (int k = 1; k < kWavesHere; ++k) y += red[k][col >> 4][at];
    const int v = tile0 * kTileRows + col;
    if (m0 + m < p.rows && v < p.vocab) store_logit(p, m0 + m, v, y);
  }
}

}  // namespace ets
