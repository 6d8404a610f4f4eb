// The 8-bit KV cache (gfx950): layout, block scales and conversions shared by its kernels.
//
// One layer's cache is codes [2][num_pages][Hkv][16][D] in e4m3 (K = 0, V = 1) and scales
// [2][num_pages][Hkv] in fp32.  A block -- 16 tokens of one kv head, of K or of V -- is D x 16 contiguous
// bytes and has one scale; a value is code x scale.  Head-major pages (the fp16 pool is token-major) keep a
// block together: a wave that attends one kv head reads 2 KiB runs (D = 128) and one scale with each.
//
// Scales are powers of two.  e4m3 is a floating format, so a scale only places its range and a finer one
// would gain nothing; powers of two make every step exact but the rounding to e4m3 itself.  A block that
// holds fp16 rows decodes to fp16 numbers exactly: a row's value x is a multiple of 2^-24, and it is stored
// as the nearest multiple of the code spacing at x, which is either below 2^-24 -- then x is stored as it
// is -- or itself a multiple of 2^-24; and the largest, 448 x scale, is below 2^16 because the scale is the
// smallest one that takes the block's largest magnitude.  So the attention kernels convert codes to fp16
// with the scale applied (v_cvt_scalef32_pk_f16_fp8, one instruction for two values), and attend exactly as
// over an fp16 pool of those values.
#pragma once

#include "ifn_common.hpp"

namespace ifn {

constexpr int kF8Page = 16;        // tokens per page, and per block
constexpr int kF8MinExp = -32;     // exponent of an empty block's scale: 448 x 2^-32 > 2^-24, the least fp16 number

typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

// Exponent of the smallest power of two s with amax <= 448 s, at least kF8MinExp (amax finite, >= 0).
// 448 = 1.75 x 2^8: exponent(amax) - 8, one more when the mantissa is above 1.75.
__device__ __forceinline__ int f8_need_exp(float amax) {
  const uint32_t b = __builtin_bit_cast(uint32_t, amax);
  const int e = int(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kF8MinExp);
}
__device__ __forceinline__ float f8_pow2(int e) { return __builtin_bit_cast(float, uint32_t(e + 127) << 23); }

#if defined(__HIP_DEVICE_COMPILE__)
// Two e4m3 codes (the low or high half of a word) as fp16, times a power-of-two scale.
template <bool kHigh>
__device__ __forceinline__ f16x2 f8_to_f16(uint32_t w, float scale) {
  return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHigh));
}
// Four fp32 values, no larger than 448, as codes (to nearest, ties to even).
__device__ __forceinline__ uint32_t f8_pack(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
// Four codes times ratio (a power of two, at most one), as codes again.  In fp32: code x ratio is exact.
__device__ __forceinline__ uint32_t f8_rescale(uint32_t w, float ratio) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  return f8_pack(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}
#else  // (device builtins: the host pass only needs the declarations)
template <bool kHigh>
__device__ __forceinline__ f16x2 f8_to_f16(uint32_t, float) { return f16x2{0, 0}; }
__device__ __forceinline__ uint32_t f8_pack(float, float, float, float) { return 0; }
__device__ __forceinline__ uint32_t f8_rescale(uint32_t, float) { return 0; }
#endif

// Eight fp16 values times inv (a power of two) as codes.
__device__ __forceinline__ u32x2 f8_quant8(f16x8 x, float inv) {
  return u32x2{f8_pack(float(x[0]) * inv, float(x[1]) * inv, float(x[2]) * inv, float(x[3]) * inv),
               f8_pack(float(x[4]) * inv, float(x[5]) * inv, float(x[6]) * inv, float(x[7]) * inv)};
}
__device__ __forceinline__ float f8_amax8(f16x8 x) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(float(x[j])));
  return m;
}

// Byte offset of block (page, head) in the K or V half.
template <int D>
__device__ __forceinline__ int64_t f8_block(int64_t page, int hkv, int h) {
  return (page * hkv + h) * (kF8Page * D);
}

}  // namespace ifn
