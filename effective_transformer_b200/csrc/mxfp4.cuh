// MXFP4 rows: 32 consecutive values of a row share a power-of-two scale (one byte, e8m0), each value is a 4-bit
// float (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//
// Layout.  The tensor core reads such an operand from shared memory as rows of 128 bytes (256 values) under the
// 128-byte swizzle, and its scales from tensor memory, where they come from 512-byte pieces that hold four
// scales for each of 128 rows.  Rows are kept in exactly that form, so that one untiled bulk copy moves an operand
// tile and its scales and no tensor map is needed: tiles of 128 rows x 256 values, 17408 bytes each, all k-tiles of
// a row block side by side.
//   value k of row r in a tile:  byte p * 128 + (((k / 32) ^ (p & 7)) * 16) + (k % 32) / 2, even k in the low nibble
//   scale of block b = k / 32:   byte 16384 + (b / 4) * 512 + (p % 32) * 16 + (p / 32) * 4 + b % 4
// with p = r but for its bits 1-2 and 3-4, which change places.  In the accumulator a tensor's rows are lanes (A) or
// columns (W), and with columns in this order a thread that reads four 8-column groups of a row in the layout of
// tcgen05.ld 16x256b, two columns of each, has eight neighbouring columns of the result: they go to memory from
// registers in whole 32-byte sectors, without a turn through shared memory, whose bandwidth the product is short of.
// A 16-byte piece of a row is one scale block.  Rows past the row count and, in a valid row, blocks past the width
// rounded up to 64 hold anything; the one block between an odd width / 32 and that multiple of 64 is zero.
#pragma once

#include <cuda_fp16.h>
#include <stddef.h>
#include <stdint.h>

#include "packed_f32.cuh"

namespace etb {

constexpr int kMxBlock = 32;
constexpr int kMxTileRows = 128;
constexpr int kMxTileK = 256;
constexpr int kMxCodeBytes = kMxTileRows * kMxTileK / 2;
constexpr int kMxScaleBytes = kMxTileRows * kMxTileK / kMxBlock;
constexpr int kMxTileBytes = kMxCodeBytes + kMxScaleBytes;

__host__ __device__ inline int mx_k_tiles(int k) { return (k + kMxTileK - 1) / kMxTileK; }
inline size_t mx_bytes(long long rows, int k) {
  return static_cast<size_t>((rows + kMxTileRows - 1) / kMxTileRows) * mx_k_tiles(k) * kMxTileBytes;
}
// Byte offset of tile (row block of `row`, k-tile kt).
__device__ __forceinline__ size_t mx_tile_offset(int row, int kt, int k_tiles) {
  return (static_cast<size_t>(row >> 7) * k_tiles + kt) * kMxTileBytes;
}
// Where row r stands in its group of 32 (and which row stands at r: the exchange is its own inverse).
__host__ __device__ constexpr int mx_row(int r) { return (r & ~0x1e) | ((r & 0x18) >> 2) | ((r & 0x06) << 2); }
// Within a tile: the 16-byte piece of block b (0..7) of row r (0..127), and its scale byte.
__device__ __forceinline__ int mx_code_offset(int r, int b) {
  const int p = mx_row(r);
  return p * 128 + ((b ^ (p & 7)) << 4);
}
__device__ __forceinline__ int mx_scale_offset(int r, int b) {
  const int p = mx_row(r);
  return kMxCodeBytes + (b >> 2) * 512 + (p & 31) * 16 + (p >> 5) * 4 + (b & 3);
}

// Scale of a block from the bits of its largest magnitude (fp32): 2^(floor(log2 amax) - 2), since the largest code
// carries 2^2; `byte` is that exponent + 127, `inverse` the reciprocal, a power of two too, so that x * inverse is
// exact.  Exponents end at -127 (a block of zeros, or of values below 2^-125).  A block with an infinity or a NaN
// gets the scale NaN (255): all its values read as NaN.
struct MxScale {
  uint32_t byte;
  float inverse;
};
__device__ __forceinline__ MxScale mx_scale(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23);
  const int b = e > 2 ? e - 2 : 0;
  MxScale s;
  s.byte = e == 255 ? 255u : static_cast<uint32_t>(b);
  s.inverse = e == 255 ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - b) << 23);
  return s;
}
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fffffffu : byte << 23);
}
// Eight values as codes, the first in the lowest nibble; round to nearest, ties to the even code, saturating at 6.
__device__ __forceinline__ uint32_t mx_codes8(const Pair* x, const MxScale& s) {
  const Pair inv = pack2(s.inverse, s.inverse);
  Pair f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = mul2(x[i], inv);
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(f[0].x), "f"(f[0].y), "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y));
  return s.byte == 255u ? 0u : w;
}
__device__ __forceinline__ uint32_t mx_codes8(const float* x, const MxScale& s) {
  const Pair p[4] = {pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7])};
  return mx_codes8(p, s);
}
// |x| as fp32 bits: the integer maximum of these is the largest magnitude, with NaN above infinity above the rest.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace etb
