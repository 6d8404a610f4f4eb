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

__device__ __forceinline__ float swap_max16(float x) {  // over lanes l, l ^ 16
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
#else
  return x;
#endif
}
__device__ __forceinline__ float swap_sum(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
#else
  return x;
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x4 a, f16x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}
#else
__device__ __forceinline__ f32x4 mfma16(f16x8, f16x8, f32x4 c) { return c; }
__device__ __forceinline__ f32x4 mfma16(f16x4, f16x4, f32x4 c) { return c; }
#endif

// One page of one head in a wave's registers, lane (n = lane % 16, g = lane / 16): K chunk i = dims 64 i + 16 g .. + 15
// of token n, V row t = dims n D / 16 .. of token 4 g + t.  As a 16-row fragment (f8_frag) chunk i's halves are K's
// dims in the order (i, half, g, 8 dims); a transposed V word (f8_transpose) is one dim of the lane's four tokens.
template <int D>
struct F8Page {
  static constexpr int kKL = D / 64, kVW = D / 64;  // 16-byte chunks of K; words per V row
  u32x4 k[kKL];
  uint32_t v[4][kVW];
};

template <int D, bool kStream>
__device__ __forceinline__ void f8_load_page(const uint8_t* k, const uint8_t* v, F8Page<D>& r) {  // the lane's addresses
  constexpr int kVW = F8Page<D>::kVW;
#pragma unroll
  for (int i = 0; i < F8Page<D>::kKL; ++i) r.k[i] = kStream ? ld16_stream(k + 64 * i) : ld16(k + 64 * i);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (kVW == 1) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(v + t * D);
      r.v[t][0] = kStream ? __builtin_nontemporal_load(p) : *p;
    } else if constexpr (kVW == 2) {
      const u32x2* p = reinterpret_cast<const u32x2*>(v + t * D);
      const u32x2 x = kStream ? __builtin_nontemporal_load(p) : *p;
      r.v[t][0] = x[0];
      r.v[t][1] = x[1];
    } else {
      const u32x4 x = kStream ? ld16_stream(v + t * D) : ld16(v + t * D);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[t][j % kVW] = x[j];
    }
  }
}
// Word j of tr: dim 4 c + j of the lane's V rows, one byte for each of its four tokens.
__device__ __forceinline__ void f8_transpose4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&tr)[4]) {
  const uint32_t ab = __builtin_amdgcn_perm(r1, r0, 0x05010400u), ab2 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
  const uint32_t cd = __builtin_amdgcn_perm(r3, r2, 0x05010400u), cd2 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
  tr[0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
  tr[1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
  tr[2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
  tr[3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}
template <int D>
__device__ __forceinline__ void f8_transpose(const F8Page<D>& r, int c, uint32_t (&tr)[4]) {
  f8_transpose4(r.v[0][c], r.v[1][c], r.v[2][c], r.v[3][c], tr);
}
// Eight codes (two words, a scale each) as a fragment of eight fp16.
__device__ __forceinline__ f16x8 f8_frag(uint32_t w0, uint32_t w1, float s0, float s1) {
  const f16x2 a = f8_to_f16<false>(w0, s0), b = f8_to_f16<true>(w0, s0), c = f8_to_f16<false>(w1, s1),
              d = f8_to_f16<true>(w1, s1);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A score, or -inf where it is not kept: by its bits, since the score of a row that nobody stored may be NaN, which
// the prefill files' float operations are compiled not to expect.
__device__ __forceinline__ float f8_masked(bool keep, float s) {
  return __builtin_bit_cast(float, keep ? __builtin_bit_cast(uint32_t, s) : 0xff800000u);
}

// No instruction: the values must have arrived at this point.
template <class A, class B>
__device__ __forceinline__ void settle(A& a, B& b) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(a));
  asm volatile("" : "+v"(b));
#endif
}

// Byte offset of block (page, head) in the K or V half.
template <int D>
__device__ __forceinline__ int64_t f8_block(int64_t page, int hkv, int h) {
  return (page * hkv + h) * (kF8Page * D);
}

// Prefill in workgroups of 128 columns (paged_prefill_fp8_block.hip), on one or two key groups.
int prefill_fp8_block_launch(f16* out, const f16* q, const uint8_t* codes, const float* scales, int64_t num_pages,
                             const int32_t* table, int32_t query_start, int32_t T, int32_t hq, int32_t hkv, int32_t d,
                             float scale_log2, int groups, hipStream_t stream);

}  // namespace ifn
