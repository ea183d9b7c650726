// Microscaled 4-bit floating point (MXFP4): blocks of 32 consecutive k that
// share a power of two.
//
//   value = (-1)^s {0, 0.5, 1, 1.5, 2, 3, 4, 6}[code & 7] * 2^(byte - 127)
//
// Two codes a byte, the lower k in the low bits; a byte of 255 is NaN.  A block
// is quantised with 2^e, e = floor(log2(max |x|)) - 2 (the exponent of 4, the
// largest power of two among the values, then meets the largest magnitude's),
// not below 2^-127, each value to the nearest code, ties to the even one,
// beyond 6 to 6; a block that holds an infinity or NaN gets the byte 255.
//
// Laid out for the 16x16x128 scaled MFMA, whose lane l holds row l % 16 and the
// 32 k of block l / 16, one MX block in 16 bytes, and that block's byte:
//   weights  [NT][KT][64 lanes][16 bytes]: tile t of 16 rows (output columns)
//            and 128 k; row i of tile 2 p + j is column 32 p + 8 (i / 4) + 4 j +
//            i % 4, so that a lane's outputs of a pair are 8 consecutive columns
//   scales   [NT][KS][64 lanes][4]: byte b of lane (r, g) is that of block
//            16 s + 4 b + g, the lane's block of k-tile 4 s + b
// A product's quantised activations: of a linear layer in the same layout, rows 16
// t .. 16 t + 15 in tile t; of experts, which gather them, row by row, codes
// [rows][K / 2] and scales [rows][KS][4 g][4 b].
// Columns past N and k past K hold zeros, and scales of 2^-127.
#pragma once

#include "awq_device.h"

namespace sgl_awq {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kMxBlock = 32;

__host__ __device__ constexpr int64_t mx4_tiles(int64_t N) { return (N + 31) / 32 * 2; }  // NT
__host__ __device__ constexpr int64_t mx4_ktiles(int64_t K) { return (K + 127) / 128; }   // KT
__host__ __device__ constexpr int64_t mx4_ksteps(int64_t K) { return (K + 511) / 512; }   // KS
__host__ __device__ constexpr int64_t mx4_weight_bytes(int64_t N, int64_t K) {
  return mx4_tiles(N) * mx4_ktiles(K) * 1024;
}
__host__ __device__ constexpr int64_t mx4_scale_bytes(int64_t N, int64_t K) {
  return mx4_tiles(N) * mx4_ksteps(K) * 256;
}

// Where block kb of a row has its byte in the rows' order.
__host__ __device__ constexpr int mx4_row_byte(int kb) { return (kb & ~15) + 4 * (kb & 3) + ((kb >> 2) & 3); }

// 2^(byte - 127) as a float; 2^-127 for byte 0 is subnormal, and the hardware's
// conversions read the exponent field alone.
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}

// The byte of a block whose largest magnitude has these bits as fp32.
__device__ __forceinline__ uint32_t mx4_byte_of(uint32_t top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}

// Largest magnitude of 16-bit values, as their bits: magnitudes order as
// integers, infinities and NaN above all others.
__device__ __forceinline__ uint32_t max_abs16(uint32_t a, uint32_t b) {
  const u16x2 x = __builtin_bit_cast(u16x2, a & 0x7FFF7FFFu), y = __builtin_bit_cast(u16x2, b & 0x7FFF7FFFu);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}

template <typename DT>
struct Mx4From;  // 16-bit activations of one type

template <>
struct Mx4From<BF16> {
  __device__ __forceinline__ static uint32_t byte_of(uint32_t top16) { return mx4_byte_of(top16 << 16); }
  template <int SEL>
  __device__ __forceinline__ static uint32_t put(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, SEL);
  }
};
template <>
struct Mx4From<F16> {
  // Every fp16 magnitude, subnormal or not, is a normal float.
  __device__ __forceinline__ static uint32_t byte_of(uint32_t top16) {
    return mx4_byte_of(__builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)top16)));
  }
  template <int SEL>
  __device__ __forceinline__ static uint32_t put(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, SEL);
  }
};

// Eight 16-bit values to eight codes.
template <typename DT>
__device__ __forceinline__ uint32_t mx4_codes8(u32x4 v, float scale) {
  uint32_t r = 0;
  r = Mx4From<DT>::template put<0>(r, v[0], scale);
  r = Mx4From<DT>::template put<1>(r, v[1], scale);
  r = Mx4From<DT>::template put<2>(r, v[2], scale);
  return Mx4From<DT>::template put<3>(r, v[3], scale);
}

// One block held by one lane: 32 16-bit values to 16 bytes of codes and the byte.
template <typename DT>
__device__ __forceinline__ u32x4 mx4_block(const u32x4 (&v)[4], uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max_abs16(m, v[q][i]);
  byte = Mx4From<DT>::byte_of(max(m & 0xFFFFu, m >> 16));
  const float scale = mx4_scale(byte);
  u32x4 r;
#pragma unroll
  for (int q = 0; q < 4; ++q) r[q] = mx4_codes8<DT>(v[q], scale);
  return r;
}

// Largest of four neighbouring lanes' values.
__device__ __forceinline__ uint32_t max4(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));     // lanes 1 0 3 2 of four
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // 2 3 0 1
}

// One block held by four neighbouring lanes, 8 values each: the lane's codes, and the byte.
template <typename DT>
__device__ __forceinline__ uint32_t mx4_quarter(u32x4 v, uint32_t& byte) {
  const uint32_t m = max_abs16(max_abs16(v[0], v[1]), max_abs16(v[2], v[3]));
  byte = Mx4From<DT>::byte_of(max4(max(m & 0xFFFFu, m >> 16)));
  return mx4_codes8<DT>(v, mx4_scale(byte));
}

// acc + W X^T of 16 weight rows and 16 activation rows over 128 k; SW and SX say
// which bytes of sw and sx hold the scales.
template <int SW, int SX>
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 w, u32x4 x, uint32_t sw, uint32_t sx, f32x4 acc) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, SW, (int)sw, SX, (int)sx);
}

}  // namespace sgl_awq
