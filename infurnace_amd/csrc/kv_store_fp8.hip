// KV append into the 8-bit cache (store_kv_fp8): fp16 rows to e4m3 blocks with one power-of-two scale each.
//
// The 8-bit form of the reference's documented store_kv (docs/architecture.md:245, 249-253; placeholder
// src/infurnace/kernels/kv_store.py).  For the rows x_t of a call that fall into one block, at offsets o_t:
//
//   need = 2^max(-32, ceil(log2(max |x| / 448)))
//   an o_t is 0: the block starts -- s' = need, and its rows that are not stored become zero
//   otherwise:   s' = max(s, need), and its other codes become e4m3(c s / s')  (unchanged where s' = s)
//   c'[o_t] = e4m3(x_t / s')
//
// A block is changed as a whole, so one wave owns it: the wave of the call's first token in that page (a
// token has none of its page among the 63 before it), which finds the page's other tokens among the 63 that
// follow.  A call keeps a page's tokens that near to each other (any order; of two with one slot the later
// is stored).  Lane (row = lane / 4, part = lane % 4) holds 8 dims of every 32 of one of the block's 16 rows.
#include "kv_fp8.hpp"

namespace ifn {

constexpr int kStoreF8Threads = 256;
constexpr int kStoreF8Waves = kStoreF8Threads / kWave;

// per: consecutive tokens a wave looks at for first ones.
template <int D>
__global__ __launch_bounds__(kStoreF8Threads) void store_kv_fp8_kernel(
    uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t num_pages, const int32_t* __restrict__ slots,
    const uint8_t* __restrict__ active, const f16* __restrict__ new_k, const f16* __restrict__ new_v,
    int32_t num_tokens, int32_t hkv, int32_t per) {
  constexpr int kC = D / 32;  // 8-dim pieces of a row per lane
  const int lane = threadIdx.x % kWave;
  const int64_t w = int64_t(blockIdx.x) * kStoreF8Waves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int which = int(w % (2 * hkv));  // K heads, then V heads
  const int64_t t0 = w / (2 * hkv) * per;
  if (t0 >= num_tokens) return;
  const bool is_v = which >= hkv;
  const int h = is_v ? which - hkv : which;
  const int64_t num_slots = num_pages * kF8Page;
  // slots of the 64 tokens before t0, from t0 on, and after those; -1 where nothing is stored
  auto slot_at = [&](int64_t t) -> int {
    if (t < 0 || t >= num_tokens) return -1;
    const int s = slots[t];
    const bool on = active == nullptr || active[t] != 0;
    return on && s >= 0 && s < num_slots ? s : -1;
  };
  const int s0 = slot_at(t0 - kWave + lane), s1 = slot_at(t0 + lane);
  const int s2 = per > 1 ? slot_at(t0 + kWave + lane) : -1;
  const f16* src = (is_v ? new_v : new_k) + int64_t(h) * D;
  const int row = lane / 4, part = lane % 4;

  for (int i = 0; i < per; ++i) {
    const int slot = __builtin_amdgcn_readlane(s1, i);
    if (slot < 0) continue;
    const int page = slot / kF8Page;
    const bool m0 = s0 >= 0 && s0 / kF8Page == page && lane > i;  // the 63 tokens before token t0 + i
    const bool m1 = s1 >= 0 && s1 / kF8Page == page;
    const bool m2 = s2 >= 0 && s2 / kF8Page == page && lane < i;  // ... and up to the 63 behind it
    if (__builtin_amdgcn_ballot_w64(m0 || (m1 && lane < i)) != 0) continue;
    // the block's rows in this call: the latest token of each offset
    int from = -1;
#pragma unroll
    for (int o = 0; o < kF8Page; ++o) {
      const uint64_t b1 = __builtin_amdgcn_ballot_w64(m1 && s1 % kF8Page == o);
      const uint64_t b2 = __builtin_amdgcn_ballot_w64(m2 && s2 % kF8Page == o);
      const int f = b2 != 0 ? 127 - __builtin_clzll(b2) : b1 != 0 ? 63 - __builtin_clzll(b1) : -1;
      if (row == o) from = f;
    }
    const bool mine = from >= 0;
    const bool begins = __builtin_amdgcn_readlane(from, 0) >= 0;
    f16x8 x[kC];
    float amax = 0.f;
    if (mine) {
      const f16* p = src + (t0 + from) * hkv * D + 8 * part;
#pragma unroll
      for (int c = 0; c < kC; ++c) x[c] = as_h8(ld16_stream(p + 32 * c));
    }
    const int64_t sc = ((is_v ? num_pages : 0) + page) * hkv + h;
    const float old = scales[sc];
    if (mine) {
#pragma unroll
      for (int c = 0; c < kC; ++c) amax = fmaxf(amax, f8_amax8(x[c]));
    }
    amax = wave_max(amax);
    const float need = f8_pow2(f8_need_exp(amax));
    const float now = begins ? need : fmaxf(old, need);
    uint8_t* blk = codes + (is_v ? num_pages * hkv * (kF8Page * D) : 0) + f8_block<D>(page, hkv, h) + row * D + 8 * part;
    if (mine) {
      const float inv = 1.f / now;  // (exact: a power of two)
#pragma unroll
      for (int c = 0; c < kC; ++c) *reinterpret_cast<u32x2*>(blk + 32 * c) = f8_quant8(x[c], inv);
    } else if (begins) {
#pragma unroll
      for (int c = 0; c < kC; ++c) *reinterpret_cast<u32x2*>(blk + 32 * c) = u32x2{0u, 0u};
    } else if (now != old) {
      const float ratio = old / now;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(blk + 32 * c);
        *reinterpret_cast<u32x2*>(blk + 32 * c) = u32x2{f8_rescale(v[0], ratio), f8_rescale(v[1], ratio)};
      }
    }
    if (lane == 0 && (begins || now != old)) scales[sc] = now;
  }
}

}  // namespace ifn

extern "C" int ifn_store_kv_fp8(void* codes_layer, float* scales_layer, int64_t num_pages,
                                const int32_t* slot_mapping, const uint8_t* active_mask, const void* new_k,
                                const void* new_v, int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                int32_t block_size, void* stream) {
  using namespace ifn;
  if (codes_layer == nullptr || scales_layer == nullptr || slot_mapping == nullptr || new_k == nullptr ||
      new_v == nullptr)
    return IFN_ERR_INVALID_ARGUMENT;
  if (num_pages < 1 || num_tokens < 0 || num_kv_heads < 1 || head_dim < 1 || block_size < 1)
    return IFN_ERR_INVALID_ARGUMENT;
  if (block_size != kF8Page || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return IFN_ERR_UNSUPPORTED;
  if (num_pages > (int64_t(1) << 31) / kF8Page) return IFN_ERR_UNSUPPORTED;  // (slots are int32)
  IFN_CHECK_ALIGN16(codes_layer);
  IFN_CHECK_ALIGN16(new_k);
  IFN_CHECK_ALIGN16(new_v);
  if (num_tokens == 0) return IFN_OK;
  const int32_t per = num_tokens >= 1024 ? kF8Page : 1;
  const int64_t waves = ceil_div(num_tokens, per) * 2 * num_kv_heads;
  const int64_t blocks = ceil_div(waves, kStoreF8Waves);
  if (blocks >= int64_t(1) << 31) return IFN_ERR_UNSUPPORTED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto k = head_dim == 64 ? store_kv_fp8_kernel<64> : head_dim == 128 ? store_kv_fp8_kernel<128> : store_kv_fp8_kernel<256>;
  k<<<dim3(unsigned(blocks)), dim3(kStoreF8Threads), 0, s>>>(
      static_cast<uint8_t*>(codes_layer), scales_layer, num_pages, slot_mapping, active_mask,
      static_cast<const f16*>(new_k), static_cast<const f16*>(new_v), num_tokens, num_kv_heads, per);
  return ifn_launch_status();
}
