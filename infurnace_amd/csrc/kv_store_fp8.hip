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
// A block is changed as a whole, so one wave owns a page's two blocks of a head: the wave of the call's first token in
// that page.  It looks at the 63 tokens before its own and after it.  That is enough where the page's tokens are
// a run in order that starts at offset 0 or with the call and ends at offset 15 or with it (a chunk's are; slots are
// distinct), or where the call has no more tokens; otherwise it goes through all slots of the call.  Of two tokens
// with one slot the later is stored.  D / 8 lanes take a row, 8 dims each: a load instruction reads whole rows of a
// head, a store writes whole lines of a block.
//
// What bounds it: small calls by their round trips (slots, rows and scales, stores), 4.1 us; large ones by memory (8192
// tokens of 8 x 128: 11.9 us, 4.2 TB/s; 30000: 34.6 us, 5.3 TB/s, where a large copy reaches 4.7).
#include "kv_fp8.hpp"

namespace ifn {

constexpr int kStoreF8Threads = 256;
constexpr int kStoreF8Waves = kStoreF8Threads / kWave;

// Maximum over the 64 lanes.
__device__ __forceinline__ float wave_max_fast(float x) {
  x = fmaxf(x, dpp<kDppXor1>(x));
  x = fmaxf(x, dpp<kDppXor2>(x));
  x = fmaxf(x, dpp<kDppHalfMirror>(x));
  x = fmaxf(x, dpp<kDppMirror>(x));
  return max_lane32(swap_max16(x));
}

// per: consecutive tokens a wave looks at for first ones.
template <int D>
__global__ __launch_bounds__(kStoreF8Threads) void store_kv_fp8_kernel(
    const int32_t* __restrict__ slots, const uint8_t* __restrict__ active, int64_t num_pages, int32_t num_tokens,
    int32_t hkv, int32_t per,  // (up to here in registers at dispatch: build.py)
    uint8_t* __restrict__ codes, float* __restrict__ scales, const f16* __restrict__ new_k,
    const f16* __restrict__ new_v) {
  constexpr int kLanes = D / 8;           // lanes per row
  constexpr int kRows = kWave / kLanes;   // rows per instruction
  constexpr int kC = kF8Page / kRows;     // instructions per block: instruction c, rows kRows c + lane / kLanes
  const int lane = threadIdx.x % kWave;
  const uint32_t w = blockIdx.x * kStoreF8Waves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int h = int(w % uint32_t(hkv));
  const int64_t t0 = int64_t(w / uint32_t(hkv)) * per;
  if (t0 >= num_tokens) return;
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
  const int p0 = s0 >> 4, p1 = s1 >> 4, p2 = s2 >> 4;  // pages (-1: none)
  // first tokens are among those whose page is not the one before's
  int before = __shfl_up(p1, 1);
  const int last0 = __builtin_amdgcn_readlane(p0, kWave - 1);
  if (lane == 0) before = last0;
  uint64_t todo = __builtin_amdgcn_ballot_w64(p1 >= 0 && p1 != before && lane < per);
  const int row0 = lane / kLanes, piece = 8 * (lane % kLanes);

  while (todo != 0) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int slot = __builtin_amdgcn_readlane(s1, i), page = slot >> 4;
    const bool m1 = p1 == page;
    const bool m2 = p2 == page && lane < i;  // (up to the 63 behind the token)
    if (__builtin_amdgcn_ballot_w64((p0 == page && lane > i) || (m1 && lane < i)) != 0) continue;
    // the block's rows in this call, as tokens from t0: a run of the page's tokens in order, or the latest of each offset
    int from[kC];
    const uint64_t b1 = __builtin_amdgcn_ballot_w64(m1), b2 = __builtin_amdgcn_ballot_w64(m2);
    const uint64_t r1 = b1 >> i;
    const bool run = b2 == 0 && (r1 & (r1 + 1)) == 0 && __builtin_amdgcn_ballot_w64(m1 && s1 - slot != lane - i) == 0;
    const int off = slot & 15, end = off + __builtin_popcountll(b1);
    const bool whole = run && (off == 0 || t0 + i == 0) && (end == kF8Page || t0 + i + end - off == num_tokens);
    if (!whole && (t0 + i >= kWave || t0 + i + kWave < num_tokens)) {
#pragma unroll
      for (int c = 0; c < kC; ++c) from[c] = -1;
      bool first = true;
      for (int64_t at = 0; at < num_tokens && first; at += 4 * kWave) {
        int s[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) s[x] = slot_at(at + kWave * x + lane);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          for (uint64_t of = __builtin_amdgcn_ballot_w64((s[x] >> 4) == page); of != 0; of &= of - 1) {
            const int j = __builtin_ctzll(of), o = __builtin_amdgcn_readlane(s[x], j) & 15;
            const int f = int(at + kWave * x + j - t0);
            first = first && f >= i;
#pragma unroll
            for (int c = 0; c < kC; ++c)
              if (kRows * c + row0 == o) from[c] = f;
          }
        }
      }
      if (!first) continue;
    } else if (run) {
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const int row = kRows * c + row0;
        from[c] = row >= off && row < end ? i + row - off : -1;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kC; ++c) from[c] = -1;
#pragma unroll
      for (int o = 0; o < kF8Page; ++o) {
        const uint64_t o1 = __builtin_amdgcn_ballot_w64(m1 && (s1 & 15) == o);
        const uint64_t o2 = __builtin_amdgcn_ballot_w64(m2 && (s2 & 15) == o);
        const int f = o2 != 0 ? 127 - __builtin_clzll(o2) : o1 != 0 ? 63 - __builtin_clzll(o1) : -1;
        if (row0 == o % kRows) from[o / kRows] = f;
      }
    }
    const bool begins = __builtin_amdgcn_readlane(from[0], 0) >= 0;
    f16x8 x[2][kC];
    float old[2], amax[2] = {0.f, 0.f};
    const int64_t src = t0 * hkv * D + int64_t(h) * D + piece;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const f16* rows = kv == 0 ? new_k : new_v;
#pragma unroll
      for (int c = 0; c < kC; ++c)  // (rows that are not in the call: zeros)
        x[kv][c] = as_h8(from[c] >= 0 ? ld16_stream(rows + src + int64_t(from[c]) * hkv * D) : u32x4{0u, 0u, 0u, 0u});
      old[kv] = scales[(kv * num_pages + page) * hkv + h];
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int c = 0; c < kC; ++c) amax[kv] = fmaxf(amax[kv], f8_amax8(x[kv][c]));
      const float need = f8_pow2(f8_need_exp(wave_max_fast(amax[kv])));
      const float now = begins ? need : fmaxf(old[kv], need), inv = 1.f / now;  // (exact: powers of two)
      uint8_t* blk = codes + kv * num_pages * hkv * (kF8Page * D) + f8_block<D>(page, hkv, h) + row0 * D + piece;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        u32x2* dst = reinterpret_cast<u32x2*>(blk + kRows * c * D);
        if (begins || from[c] >= 0) {  // (a block that starts: its other rows are zero)
          *dst = f8_quant8(x[kv][c], inv);
        } else if (now != old[kv]) {
          const u32x2 v = *dst;
          *dst = u32x2{f8_rescale(v[0], old[kv] / now), f8_rescale(v[1], old[kv] / now)};
        }
      }
      if (lane == 0 && (begins || now != old[kv])) scales[(kv * num_pages + page) * hkv + h] = now;
    }
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
  // A wave for every token is best for the tokens of a step, each in a page of its own (8 heads, 256 of them: 5.8 us,
  // 12.9 with four a wave, 43 with 16), a wave for every 16 for a chunk (2000 tokens: 22.2, 10.5, 5.5).  By what the
  // call most likely is: steps have few tokens.  (512 tokens: a chunk 7.2, 5.2, 4.9, a step 8.1, 15.7, 55.)
  const int64_t most = int64_t(num_tokens) * num_kv_heads;
  const int32_t per = most <= 2048 ? 1 : most <= 8192 ? 4 : kF8Page;
  const int64_t waves = ceil_div(num_tokens, per) * num_kv_heads;
  const int64_t blocks = ceil_div(waves, kStoreF8Waves);
  if (waves >= int64_t(1) << 31) return IFN_ERR_UNSUPPORTED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto k = head_dim == 64 ? store_kv_fp8_kernel<64> : head_dim == 128 ? store_kv_fp8_kernel<128> : store_kv_fp8_kernel<256>;
  k<<<dim3(unsigned(blocks)), dim3(kStoreF8Threads), 0, s>>>(
      slot_mapping, active_mask, num_pages, num_tokens, num_kv_heads, per, static_cast<uint8_t*>(codes_layer),
      scales_layer, static_cast<const f16*>(new_k), static_cast<const f16*>(new_v));
  return ifn_launch_status();
}
