// Values in E4M3 with a scale for each block of 128: the scale is a power of
// two in one byte (E8M0: 2^(byte - 127), 255 for NaN), which the matrix
// instruction multiplies in by itself.
//
//   a = max |x| over the block, scale = 2^k with k the smallest integer >= -126
//   for which a <= 448 2^k (k = 0 where a = 0), q = round_to_even(x / 2^k)
//
// A quotient by a power of two is exact, so q is rounded once and every byte is
// determined by the input. A block that holds a NaN or an infinity has scale
// NaN and bytes 0.
#pragma once

#include "common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = MM_FP8_BLOCK;
constexpr uint32_t kScaleNan = 255;

struct BlockScale {
  uint32_t byte;
  float inv;  // 1 / scale; 0 with `bad`
  bool bad;
  // bits: the block's largest |x| as a bit pattern, where NaN lies above infinity
  __device__ __forceinline__ explicit BlockScale(uint32_t bits) : bad(bits >= 0x7f800000u) {
    // 448 = 1.75 * 2^8
    int b = static_cast<int>(bits >> 23) - 8 + ((bits & 0x007fffffu) > 0x00600000u ? 1 : 0);
    b = bits == 0 ? 127 : max(b, 1);
    byte = bad ? kScaleNan : static_cast<uint32_t>(b);
    inv = bad ? 0.0f : __uint_as_float(static_cast<uint32_t>(254 - b) << 23);
  }
  // four values to bytes; 0 * NaN would leave NaN, hence the select
  __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) const {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
    return bad ? 0u : static_cast<uint32_t>(w);
  }
};

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == kScaleNan ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// The larger of a value over 16 neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m)));
  return v;
}

}  // namespace
