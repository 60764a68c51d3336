// Microscaled 4-bit rows (the OCP Microscaling format MXFP4): number format and packed layout shared
// by mxfp4.hip and mxfp4_linear.hip.
//
// A row of K elements is K / 2 code bytes (the even element in the low half) and K / 32 scale bytes.  A
// code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; an element of block b of 32 is code * 2^(s[b] - 127),
// NaN where s[b] = 255.  Every value of a scale byte up to 252 is a bf16 number (two significant bits, bf16's
// exponents), and quantisation gives no larger one; of 253 and 254 the codes whose value is 2^128 or more (4 and 6;
// 2, 3, 4 and 6) are infinities as bf16 and fp32, while products of two 4-bit operands take them as they are.
//
// Packed layout, of a weight's rows or of quantised activations.  Tile (t, u) holds sixteen rows
// of K elements 128 u .. 128 u + 127 as 64 chunks of 16 bytes: chunk l is the tile's row l % 16, block l / 16 --
// the order in which a wave's lanes hold a 16 x 128 operand of v_mfma_scale_f32_16x16x128_f8f6f4, so that a
// wave's load of a tile is 1 KB of consecutive bytes.  Row r of an activation's tile t is row 16 t + r; of a
// weight's, whose tiles come in pairs, weight_row(t, r): a lane's four outputs of one tile and four of the next are
// then eight consecutive columns.  Tiles lie u fastest, K rounded up to quads of four tiles.
// Behind all tiles follow the scales: one dword for (t, u / 4, l), its byte u % 4 the scale of chunk l of tile
// (t, u).  Blocks past the matrix are codes 0 of scale 127; so are rows past a weight's last, while
// activations' rows past the last are not written (their outputs are not stored).
#pragma once

#include "common.h"

namespace mxfp4 {

constexpr int kBlock = 32;   // elements of one scale
constexpr int kStep = 128;   // K elements of a tile
constexpr int kTile = 1024;  // bytes of a tile
constexpr int kQuad = 4 * kStep;

inline int64_t quads(int64_t K) { return (K + kQuad - 1) / kQuad; }
inline int64_t row_tiles(int64_t rows) { return (rows + 15) / 16; }
inline int64_t weight_tiles(int64_t rows) { return (rows + 31) / 32 * 2; }
inline int64_t tile_bytes(int64_t tiles, int64_t K) { return tiles * quads(K) * 4 * kTile; }
inline int64_t packed_bytes(int64_t tiles, int64_t K) { return tile_bytes(tiles, K) + tiles * quads(K) * 256; }

__host__ __device__ inline int64_t weight_row(int64_t t, int r) {
  return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// The scale byte of a block whose largest magnitude has these fp32 bits: floor(log2 a) - 2 + 127, at least
// 0 (2^-127, for zeros and subnormals too), 255 for a block that is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// A scale byte as the scale operand of the v_cvt_scalef32 instructions, which read its exponent field:
// byte 0 is 2^-127 and 255 NaN there too.
__device__ __forceinline__ float scale_operand(uint32_t byte) { return __uint_as_float(byte << 23); }

// (by value: a bit cast of a vector's element would take the vector's first)
__device__ __forceinline__ bf16x2_t pair(uint32_t v) { return __builtin_bit_cast(bf16x2_t, v); }

// The codes of eight bf16 values (four dwords of two), nearest with ties to the even code, saturated at 6
// (v_cvt_scalef32_pk_fp4_bf16).  CLEAR: a block of scale byte 255 has codes 0 (any others stand for NaN too).
template <bool CLEAR = true>
__device__ __forceinline__ uint32_t codes_of(const u32x4_t& x, uint32_t s) {
  if (CLEAR && s == 255) return 0;
  const float f = scale_operand(s);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(x[0]), f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(x[1]), f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(x[2]), f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(x[3]), f, 3);
  return r;
}

// The same of eight fp32 values.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], uint32_t s) {
  if (s == 255) return 0;
  const float f = scale_operand(s);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], f, 3);
  return r;
}

// Bits (of fp32) of the largest magnitude of 8 N bf16 values.
template <int N>
__device__ __forceinline__ uint32_t amax_bits(const u32x4_t (&x)[N]) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = x[i][e] & 0x7fff7fffu;
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v));
    }
  const uint32_t lo = m[0], hi = m[1];
  return (lo > hi ? lo : hi) << 16;
}

// Eight elements of one block as bf16 (exact, infinity from 2^128 on), from their four code bytes.
__device__ __forceinline__ u32x4_t bf16_of(uint32_t c, float scale) {
  u32x4_t o;
  o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
  o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
  o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
  o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  return o;
}

}  // namespace mxfp4
