// Causal chunked-prefill paged attention over the 8-bit KV cache (gfx950 MFMA fp16).
//
// The 8-bit form of the reference's documented paged_attention with a multi-token query
// (docs/architecture.md:246; contiguous semantics src/infurnace/executor/tinygrad/model.py:116-132): query row
// i sits at query_start + i and sees keys [0, query_start + i].  Blocks and scales: kv_fp8.hpp.
//
// The (query, head) pairs of one kv head are the columns of the products, column c = query c / G, head c % G
// of the group, so any group size fills the matrix instructions.  A workgroup serves 32 columns; its waves are
// key groups that take 32-key tiles in turn and merge through LDS at the end.  S^T = K Q^T and O^T += V^T P^T
// with v_mfma_f32_32x32x16_f16: lane (c = lane % 32, half = lane / 32) has the scores of column c and keys
// 8 a + 4 half + i of the tile, which are the second product's B operand as they are (its k order is
// free: k = 8 half + j is key 8 (j / 4) + 4 half + j % 4 of a page).  Codes go from memory to the matrix cores
// in registers: K as loaded, V after a byte transpose of four keys (v_perm).
#include <algorithm>

#include "kv_fp8.hpp"

namespace ifn {

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
#else
__device__ __forceinline__ f32x16 mfma32(f16x8, f16x8, f32x16 c) { return c; }
#endif

__device__ __forceinline__ f16x8 f8_frag(uint32_t w0, uint32_t w1, float s0, float s1) {
  const f16x2 a = f8_to_f16<false>(w0, s0), b = f8_to_f16<true>(w0, s0), c = f8_to_f16<false>(w1, s1),
              d = f8_to_f16<true>(w1, s1);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int D, int KW>  // KW: waves (key groups) of a workgroup
__global__ __launch_bounds__(KW * kWave) void prefill_fp8_kernel(
    f16* __restrict__ out, const f16* __restrict__ q, const uint8_t* __restrict__ codes,
    const float* __restrict__ scales, int64_t num_pages, const int32_t* __restrict__ table, int32_t query_start,
    int32_t T, int32_t hkv, int32_t G, int32_t n_blocks, float scale_log2) {
  constexpr int kKC = D / 32;  // 16-byte K chunks a lane holds of its key's row
  constexpr int kDT = D / 32;  // output tiles: tile t's row m is dim m D / 32 + t
  __shared__ float s_o[KW][16 * kDT][kWave];
  __shared__ float s_ml[2][KW][32];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane % 32, half = lane / 32;
  const int h = int(blockIdx.x) % hkv, blk = n_blocks - 1 - int(blockIdx.x) / hkv;  // (longest key ranges first)
  const int hq = hkv * G;
  const int64_t c0 = int64_t(blk) * 32, cols = int64_t(T) * G;
  const int64_t c = min(c0 + col, cols - 1);
  const int my_q = int(c / G), my_h = h * G + int(c % G);
  const int my_pos = query_start + my_q;
  const int last_q = int((min(c0 + 31, cols - 1)) / G);
  const int keys = query_start + last_q + 1;              // keys some column sees
  const int first_pos = query_start + int(c0 / G);        // every column sees keys up to this one
  const int pages = (keys + kF8Page - 1) / kF8Page, tiles = (pages + 1) / 2;

  f16x8 qf[2 * kKC];
  {
    const f16* qp = q + (int64_t(my_q) * hq + my_h) * D + 16 * half;
#pragma unroll
    for (int i = 0; i < kKC; ++i) {
      qf[2 * i] = as_h8(ld16(qp + 32 * i));
      qf[2 * i + 1] = as_h8(ld16(qp + 32 * i + 8));
    }
  }
  float m = kNegBig, l = 0.f;
  f32x16 acc[kDT];
#pragma unroll
  for (int t = 0; t < kDT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[t][j] = 0.f;
  const int64_t v_codes = num_pages * hkv * (kF8Page * D), v_scales = num_pages * hkv;

  for (int tile = wave; tile < tiles; tile += KW) {
    const int p0 = 2 * tile;
    int id[2];
    float ks[2], vs[2];
    bool live[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int raw = table[min(p0 + x, pages - 1)];
      live[x] = p0 + x < pages && raw >= 0 && int64_t(raw) < num_pages;
      id[x] = __builtin_amdgcn_readfirstlane(live[x] ? raw : 0);
      ks[x] = scales[int64_t(id[x]) * hkv + h];
      vs[x] = scales[v_scales + int64_t(id[x]) * hkv + h];
    }
    const uint8_t* kp = codes + f8_block<D>(col < 16 ? id[0] : id[1], hkv, h) + (col % 16) * D + 16 * half;
    u32x4 kr[kKC];
#pragma unroll
    for (int i = 0; i < kKC; ++i) kr[i] = ld16(kp + 32 * i);
    uint32_t vr[2][8];  // page x: keys 4 half + i, 8 + 4 half + i; dims col D / 32 ..
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint8_t* vp = codes + v_codes + f8_block<D>(id[x], hkv, h) + 4 * half * D + col * (D / 32);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint8_t* p = vp + (8 * (j / 4) + j % 4) * D;
        if constexpr (kDT == 4) vr[x][j] = *reinterpret_cast<const uint32_t*>(p);
        else vr[x][j] = *reinterpret_cast<const uint16_t*>(p);
      }
    }
    const float my_ks = col < 16 ? ks[0] : ks[1];
    f32x16 s;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
    for (int i = 0; i < kKC; ++i) {
      s = mfma32(f8_frag(kr[i][0], kr[i][1], my_ks, my_ks), qf[2 * i], s);
      s = mfma32(f8_frag(kr[i][2], kr[i][3], my_ks, my_ks), qf[2 * i + 1], s);
    }
    float sv[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) sv[j] = s[j] * scale_log2;
    if (p0 * kF8Page + 31 > first_pos || !live[0] || !live[1]) {  // (uniform)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = p0 * kF8Page + 8 * (j / 4) + 4 * half + j % 4;
        sv[j] = live[j / 8] && key <= my_pos ? sv[j] : -INFINITY;
        const int vk = (p0 + j / 8) * kF8Page + 8 * ((j % 8) / 4) + 4 * half + j % 4;
        if (!(live[j / 8] && vk < keys)) vr[j / 8][j % 8] = 0u;  // (rows nobody stored may hold NaN, and 0 x NaN is NaN)
      }
    }
    float mx = sv[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) mx = fmaxf(mx, sv[j]);
    mx = max_lane32(mx);
    if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
      const float mn = fmaxf(m, mx);
      const float al = exp2_fast(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < kDT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[t][j] *= al;
    }
    f16x8 pf[2];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float p = exp2_fast(sv[j] - m);
      l += p;
      pf[j / 8][j % 8] = f16(p);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t tr[2][4];  // word t: dim t of four keys
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t ab = __builtin_amdgcn_perm(vr[x][4 * y + 1], vr[x][4 * y], 0x05010400u);
        const uint32_t cd = __builtin_amdgcn_perm(vr[x][4 * y + 3], vr[x][4 * y + 2], 0x05010400u);
        tr[y][0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
        tr[y][1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
        if constexpr (kDT == 4) {
          const uint32_t ab2 = __builtin_amdgcn_perm(vr[x][4 * y + 1], vr[x][4 * y], 0x07030602u);
          const uint32_t cd2 = __builtin_amdgcn_perm(vr[x][4 * y + 3], vr[x][4 * y + 2], 0x07030602u);
          tr[y][2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
          tr[y][3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
        }
      }
#pragma unroll
      for (int t = 0; t < kDT; ++t) acc[t] = mfma32(f8_frag(tr[0][t], tr[1][t], vs[x], vs[x]), pf[x], acc[t]);
    }
  }

  // The waves' states of each column: maxima and sums first, then the outputs in a common scale, each wave
  // adding up its share of the rows.
  l += __shfl_xor(l, 32);
  if (half == 0) {
    s_ml[0][wave][col] = m;
    s_ml[1][wave][col] = l;
  }
  __syncthreads();
  float M = kNegBig, L = 0.f;
#pragma unroll
  for (int w = 0; w < KW; ++w) M = fmaxf(M, s_ml[0][w][col]);
#pragma unroll
  for (int w = 0; w < KW; ++w) L += s_ml[1][w][col] * exp2_fast(s_ml[0][w][col] - M);
  const float al = exp2_fast(m - M);
#pragma unroll
  for (int t = 0; t < kDT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) s_o[wave][j * kDT + t][lane] = acc[t][j] * al;
  __syncthreads();
  const float inv = L > 0.f ? 1.f / L : 0.f;
  if (c0 + col >= cols) return;
  f16* op = out + (int64_t(my_q) * hq + my_h) * D;
  for (int j = wave; j < 16; j += KW) {
    float o[kDT];
#pragma unroll
    for (int t = 0; t < kDT; ++t) {
      o[t] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) o[t] += s_o[w][j * kDT + t][lane];
    }
    const int row = 8 * (j / 4) + 4 * half + j % 4;
    if constexpr (kDT == 4)
      *reinterpret_cast<f16x4*>(op + row * 4) = f16x4{f16(o[0] * inv), f16(o[1] * inv), f16(o[2] * inv), f16(o[3] * inv)};
    else
      *reinterpret_cast<f16x2*>(op + row * 2) = f16x2{f16(o[0] * inv), f16(o[1] * inv)};
  }
}

}  // namespace ifn

extern "C" int ifn_paged_prefill_fp8(void* out, const void* query, const void* codes_layer,
                                     const float* scales_layer, int64_t num_pages, const int32_t* block_table,
                                     int32_t max_pages, int32_t query_start, int32_t num_q_tokens,
                                     int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, float scale, void* stream) {
  using namespace ifn;
  if (out == nullptr || query == nullptr || codes_layer == nullptr || scales_layer == nullptr || block_table == nullptr)
    return IFN_ERR_INVALID_ARGUMENT;
  if (num_pages < 1 || max_pages < 1 || query_start < 0 || num_q_tokens < 0 || num_q_heads < 1 || num_kv_heads < 1 ||
      num_q_heads % num_kv_heads != 0 || head_dim < 1 || block_size < 1)
    return IFN_ERR_INVALID_ARGUMENT;
  if (block_size != kF8Page || (head_dim != 64 && head_dim != 128)) return IFN_ERR_UNSUPPORTED;
  if (int64_t(query_start) + num_q_tokens > int64_t(max_pages) * kF8Page) return IFN_ERR_INVALID_ARGUMENT;
  if (int64_t(query_start) + num_q_tokens > (int64_t(1) << 31) - 64 || num_pages > (int64_t(1) << 31) / kF8Page)
    return IFN_ERR_UNSUPPORTED;
  IFN_CHECK_ALIGN16(out);
  IFN_CHECK_ALIGN16(query);
  IFN_CHECK_ALIGN16(codes_layer);
  if (num_q_tokens == 0) return IFN_OK;
  const int32_t G = num_q_heads / num_kv_heads;
  const int64_t n_blocks = ceil_div(int64_t(num_q_tokens) * G, 32);
  if (n_blocks * num_kv_heads >= (int64_t(1) << 31)) return IFN_ERR_UNSUPPORTED;
  const float sl = (scale > 0.f ? scale : 1.f / sqrtf(float(head_dim))) * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto k = head_dim == 64 ? prefill_fp8_kernel<64, 4> : prefill_fp8_kernel<128, 4>;
  k<<<dim3(unsigned(n_blocks * num_kv_heads)), dim3(4 * kWave), 0, s>>>(
      static_cast<f16*>(out), static_cast<const f16*>(query), static_cast<const uint8_t*>(codes_layer), scales_layer,
      num_pages, block_table, query_start, num_q_tokens, num_kv_heads, G, int32_t(n_blocks), sl);
  return ifn_launch_status();
}
