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
  int32_t scale_bytes;    // 4 (fp32) or 2
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

template <int XT>
struct RawX {  // eight columns of x as they are in memory
  u32x4 v[XT == kDtypeFloat ? 2 : 1];
};

// Columns [k, k + 8) of a row; columns at `hidden` and behind, and rows that do not exist, read as 0.
template <int XT>
__device__ __forceinline__ RawX<XT> load_raw_x(const void* row, int k, int hidden, bool exists) {
  RawX<XT> out = {};
  if (!exists) return out;
  if (k + 8 <= hidden) {
    if (XT == kDtypeFloat) {
      const LooseFloats r = *reinterpret_cast<const LooseFloats*>(static_cast<const float*>(row) + k);
      __builtin_memcpy(out.v, &r, 32);
    } else {
      const LooseHalves r = *reinterpret_cast<const LooseHalves*>(static_cast<const uint16_t*>(row) + k);
      __builtin_memcpy(out.v, &r, 16);
    }
    return out;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (k + j < hidden) {
      if (XT == kDtypeFloat) {
        out.v[j >> 2][j & 3] = static_cast<const uint32_t*>(row)[k + j];
      } else {
        out.v[0][j >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(row)[k + j]) << (16 * (j & 1));
      }
    }
  }
  return out;
}

// ... as operand A, one per part.
template <int XT>
__device__ __forceinline__ void split_x(const RawX<XT>& x, u32x4* part) {
  if (XT == kDtypeFloat) {
    // x = high + middle + low, each cut off to the upper 16 bits of a float: exact, 8 bits of x at a time
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = x.v[(j >> 2) * (XT == kDtypeFloat)][j & 3];
      h[j] = bits & 0xffff0000u;
      const float rest = __uint_as_float(bits) - __uint_as_float(h[j]);
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
    part[0] = x.v[0];
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

// Four entries of a row next to each other, those inside the vocabulary.
__device__ __forceinline__ void store_logits(const HeadParams& p, int m, int v, f32x4 y) {
  if (v + 4 <= p.vocab) {
    const int64_t at = m * p.out_stride + v;
    if (p.out_dtype == kDtypeFloat) {
      struct __attribute__((packed, aligned(4))) Four { f32x4 v; };
      reinterpret_cast<Four*>(static_cast<float*>(p.out) + at)->v = y;
    } else {
      typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
      typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      struct __attribute__((packed, aligned(2))) Four { u32x2 v; };
      reinterpret_cast<Four*>(static_cast<uint16_t*>(p.out) + at)->v =
          p.out_dtype == kDtypeBFloat16 ? __builtin_bit_cast(u32x2, __builtin_convertvector(y, bf16x4))
                                        : __builtin_bit_cast(u32x2, __builtin_convertvector(y, f16x4));
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (v + r < p.vocab) store_logit(p, m, v + r, y[r]);
    }
  }
}

// ---- the product, few rows --------------------------------------------------------------------------------
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
    for (int t = 0; t < 4; ++t) split_x<XT>(load_raw_x<XT>(x_row, chunk * kChunkCols + 32 * t + 8 * q, p.hidden, exists), x[t]);
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

// ---- the product, many rows ---------------------------------------------------------------------
// A workgroup makes (16 MT) rows x (16 NT WV) vocabulary entries: WV waves next to each other along the
// vocabulary, WK of them behind each other along the columns (each takes every WK-th chunk; their sums are
// added up in the end).  x goes through LDS, where all waves read it as operand A; a wave's weights go from
// memory to its registers, unpacked there once for all of its rows.  While one chunk is multiplied the next
// one's weights and hidden states are on their way; one barrier per chunk.
// In LDS the 16 bytes of row m, columns 32 t + 8 q + 0..7, lie at 16-byte unit 64 t + 16 q + (m ^ (4 t + q)) of their
// 16 rows: a wave's read of an operand and its write of four rows both touch every bank once.
// -24 times the sum of the eight columns.
template <int XT>
__device__ __forceinline__ float minus24_sum(const RawX<XT>& x) {
  float s = 0.0f;
  if (XT == kDtypeFloat) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s += __uint_as_float(x.v[j >> 2][j & 3]);
    return -24.0f * s;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = x.v[0][i];  // (a bit cast of the vector's element itself takes its first element)
    if (XT == kDtypeBFloat16) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{static_cast<__bf16>(-24.0f), static_cast<__bf16>(-24.0f)}, s, false);
    } else {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      s = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), f16x2{static_cast<_Float16>(-24.0f), static_cast<_Float16>(-24.0f)}, s, false);
    }
  }
  return s;
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xf, 0xf, false));
}

// The scales of this lane's vocabulary row for a chunk's groups, as they are in memory (4 words at most).
template <int GPC>
struct RawScales {
  uint32_t v[GPC];
};
template <int GPC>
__device__ __forceinline__ RawScales<GPC> load_raw_scales(const void* base, const HeadParams& p, int tile, int chunk, int n) {
  const int64_t at = GPC > 1 ? ((static_cast<int64_t>(tile) * p.chunks + chunk) * kTileRows + n) * GPC
                             : (static_cast<int64_t>(tile) * p.groups + chunk / p.chunks_per_group) * kTileRows + n;
  RawScales<GPC> r = {};
  if (p.scale_bytes == 4) {
    r = *reinterpret_cast<const RawScales<GPC>*>(static_cast<const uint32_t*>(base) + at);
  } else if (GPC == 1) {
    r.v[0] = static_cast<const uint16_t*>(base)[at];
  } else {
    struct alignas(GPC > 1 ? 2 * GPC : 4) Pairs { uint32_t v[GPC > 1 ? GPC / 2 : 1]; };
    const Pairs h = *reinterpret_cast<const Pairs*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int i = 0; i < GPC / 2; ++i) r.v[i] = h.v[i];
  }
  return r;
}
template <int GPC>
__device__ __forceinline__ float scale_of(const RawScales<GPC>& r, const HeadParams& p, int g) {
  if (p.scale_bytes == 4) return __uint_as_float(r.v[g]);
  const uint32_t h = GPC == 1 ? r.v[0] : (g & 1 ? r.v[g >> 1] >> 16 : r.v[g >> 1] & 0xffffu);
  return p.scale_is_bf16 ? __uint_as_float(h << 16) : half_bits_to_float(h);
}

template <int XT, int GPC, int MT, int NT, int WV, int WK>
__global__ void __launch_bounds__(64 * WV * WK, 2)
head_tile_kernel(const HeadParams p) {
  using M = Matrix<XT>;
  constexpr int P = Parts<XT>::value, kSteps = 4 / GPC, kLanes = 64 * WV * WK, kRows = 16 * MT;
  constexpr int kPieces = WK * kRows * 16 / kLanes;  // of eight columns, per lane and step
  static_assert(WK * kRows * 16 % kLanes == 0, "");
  constexpr int kUnits = WK * P * MT * 256;          // of 16 bytes, per buffer
  constexpr int kOut = WK * WV * 16 * NT * 16;       // floats of 16 rows of the result
  constexpr int kBytes = 2 * kUnits * 16 > kOut * 4 ? 2 * kUnits * 16 : kOut * 4;
  __shared__ __attribute__((aligned(16))) char lds[kBytes];
  __shared__ float base_lds[2][WK][GPC][kRows];
  u32x4* units = reinterpret_cast<u32x4*>(lds);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wv = wave % WV, wk = wave / WV;
  // Workgroups of one XCD (every eighth) take the row blocks of a vocabulary block one after the other, so that its
  // weights come from memory once.
  const int vocab_blocks = (p.tiles + WV * NT - 1) / (WV * NT), row_blocks = (p.rows + kRows - 1) / kRows;
  const int at = blockIdx.x >> 3, vocab_block = at / row_blocks * 8 + (blockIdx.x & 7), row_block = at % row_blocks;
  if (vocab_block >= vocab_blocks) return;
  const int m0 = row_block * kRows, tile0 = (vocab_block * WV + wv) * NT;

  RawX<XT> x_raw[kPieces];
  u32x4 w_raw[NT];
  RawScales<GPC> s_raw[NT], z_raw[NT];
  auto load_step_x = [&](int step) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * kLanes + tid, slot = piece & 15, row = (piece >> 4) % kRows, chunk = step * WK + piece / (16 * kRows);
      const int m = m0 + row;
      const char* x_row = static_cast<const char*>(p.x) + (m < p.rows ? m : 0) * p.x_stride * ElemSize<XT>::value;
      x_raw[i] = load_raw_x<XT>(x_row, chunk * kChunkCols + 8 * slot, p.hidden, m < p.rows);
    }
  };
  auto load_step_w = [&](int step) {
    const int chunk = min(step * WK + wk, p.chunks - 1);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int tile = min(tile0 + i, p.tiles - 1);
      w_raw[i] = p.blocks[(static_cast<int64_t>(tile) * p.chunks + chunk) * 64 + lane];
      s_raw[i] = load_raw_scales<GPC>(p.scales, p, tile, chunk, n);
      if (p.zeros) z_raw[i] = load_raw_scales<GPC>(p.zeros, p, tile, chunk, n);
    }
  };
  auto store_step_x = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * kLanes + tid, slot = piece & 15, row = (piece >> 4) % kRows, k = piece / (16 * kRows);
      u32x4 part[P];
      split_x<XT>(x_raw[i], part);
#pragma unroll
      for (int c = 0; c < P; ++c)
        units[buffer * kUnits + ((k * P + c) * MT + (row >> 4)) * 256 + slot * 16 + ((row & 15) ^ slot)] = part[c];
      // the sums of a group: 16 lanes hold a row's chunk
      float s = minus24_sum<XT>(x_raw[i]);
      s = dpp_add<0xb1>(s);
      s = dpp_add<0x4e>(s);
      if (GPC <= 2) s = dpp_add<0x141>(s);
      if (GPC == 1) s = dpp_add<0x140>(s);
      if (slot % (16 / GPC) == 0) base_lds[buffer][k][slot / (16 / GPC)][row] = s;
    }
  };

  f32x4 total[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int i = 0; i < NT; ++i) total[a][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int steps = (p.chunks + WK - 1) / WK;
  load_step_x(0);
  load_step_w(0);
  store_step_x(0);
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    const int buffer = step & 1;
    const bool more = step + 1 < steps, there = step * WK + wk < p.chunks;
    u32x4 w[NT];
    RawScales<GPC> s[NT], z[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) w[i] = w_raw[i], s[i] = s_raw[i], z[i] = z_raw[i];
    if (more) {
      load_step_x(step + 1);
      load_step_w(step + 1);
    }
    if (there) {
#pragma unroll
      for (int g = 0; g < GPC; ++g) {
        u32x4 b[NT][kSteps];
        float sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          sc[i] = scale_of<GPC>(s[i], p, g);
#pragma unroll
          for (int t = 0; t < kSteps; ++t) b[i][t] = unpack<XT>(w[i][g * kSteps + t]);
        }
#pragma unroll
        for (int a = 0; a < MT; ++a) {
          const f32x4 base = *reinterpret_cast<const f32x4*>(&base_lds[buffer][wk][g][16 * a + 4 * q]);
          f32x4 acc[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i] = base;
#pragma unroll
          for (int t = 0; t < kSteps; ++t) {
            const int slot = 4 * (g * kSteps + t) + q;
#pragma unroll
            for (int c = 0; c < P; ++c) {
              const u32x4 x = units[buffer * kUnits + ((wk * P + c) * MT + a) * 256 + slot * 16 + (n ^ slot)];
#pragma unroll
              for (int i = 0; i < NT; ++i) acc[i] = M::product(x, b[i][t], acc[i]);
            }
          }
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) total[a][i][r] = fmaf(sc[i], acc[i][r], total[a][i][r]);
          if (p.zeros) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const float zero = scale_of<GPC>(z[i], p, g) * (-1.0f / 24.0f);
#pragma unroll
              for (int r = 0; r < 4; ++r) total[a][i][r] = fmaf(zero, base[r], total[a][i][r]);
            }
          }
        }
      }
    }
    if (more) store_step_x(buffer ^ 1);
    __syncthreads();
  }

  // 16 rows at a time through LDS: a lane then has 16 / (4 / NT) .. consecutive entries of a row to store
  float* result = reinterpret_cast<float*>(lds);
  constexpr int kWide = NT * 16 * WV;  // vocabulary entries of the workgroup
#pragma unroll
  for (int a = 0; a < MT; ++a) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) result[(wk * 16 + 4 * q + r) * kWide + (wv * NT + i) * 16 + n] = total[a][i][r];
    __syncthreads();
    for (int e = tid * 4; e < 16 * kWide; e += kLanes * 4) {
      const int row = e / kWide, col = e % kWide, m = m0 + 16 * a + row, v = vocab_block * kWide + col;
      if (m < p.rows) {
        f32x4 y = *reinterpret_cast<const f32x4*>(&result[row * kWide + col]);
#pragma unroll
        for (int k = 1; k < WK; ++k) y += *reinterpret_cast<const f32x4*>(&result[(k * 16 + row) * kWide + col]);
        store_logits(p, m, v, y);
      }
    }
    __syncthreads();
  }
}

}  // namespace ets
