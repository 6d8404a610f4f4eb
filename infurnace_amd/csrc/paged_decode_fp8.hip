// Paged GQA decode over the 8-bit KV cache (gfx950 MFMA), with the step's append and the pages' attention
// weights fused in.
//
// The 8-bit form of the reference's documented paged_attention for decode (docs/architecture.md:246;
// contiguous semantics src/infurnace/executor/tinygrad/model.py:196-200): out = softmax(scale q K^T) V over the
// row's first L tokens, query head h reading kv head h / G.  Blocks and scales: kv_fp8.hpp.
//
//  * A wave attends one kv head.  The pages of all rows, row after row, form one list per head; the grid's
//    waves are Hkv x (streams), and stream r takes pages [T r / nr, T (r+1) / nr) of the list for its head, so
//    ragged batches cost every wave the same bytes.  Waves share nothing but the rows' offsets in the list
//    (LDS); Hkv and the group size G (up to 16) are run-time numbers.  A row that starts inside a range costs
//    it kRowStart pages more (its query, its first loads).
//  * Two pages (32 tokens) are one step: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_f16, the
//    group's queries in the 16 columns.  Lane (n = lane % 16, g = lane / 16) loads K of token n, dims
//    64 i + 16 g .. + 15 (the fragments' k order is theirs to choose, as long as Q's is the same), gets the
//    scores of query n and tokens 4 g .. 4 g + 3 of each page, and needs V of the same tokens for the second
//    product: it loads 4 token rows x D / 16 dims of V and transposes the bytes (v_perm).  So codes go from
//    memory to the matrix cores without LDS and without an exchange between lanes; only the running maximum
//    is reduced over the four g (v_permlane swaps).  The running sum stays a lane's own until the end.
//  * Codes become fp16 exactly (kv_fp8.hpp).  Probabilities are rounded to fp16 for the second product (2^-12
//    relative, averaged over the keys); scores, maxima, sums and outputs are fp32.
//  * A row held by several streams: their states (m, l, O in fp32) go to the workspace and the wave that
//    arrives last, by a ticket per (row, head), merges them in range order.
//  * Fused append (kAppend): the wave that holds a row's last page adds the row's new token to the block in
//    its registers (new scale, rescaled codes), stores what changed and attends over the result.
//  * Page weights (kWeights): each page's log2-sum-exp per query head goes to the workspace; the wave that
//    finishes a (row, head) turns them into sum_g exp2(lse - total) and adds them to page_weights.
#include <algorithm>
#include <type_traits>

#include "kv_fp8.hpp"

namespace ifn {

constexpr int kF8DecThreads = 512;
constexpr int kF8DecWaves = kF8DecThreads / kWave;
constexpr int kF8MaxBatch = 4096;  // rows per call (LDS offsets)
constexpr int kF8MaxGroup = 16;    // query heads per kv head (MFMA columns)
constexpr int kRowStart = 1;       // pages a row's start counts for in the split
constexpr int kMinPages = 2;       // fewest list positions per range

struct F8Cache {
  uint8_t* codes;
  float* scales;
  int64_t num_pages;
};
struct F8Append {
  const f16* new_k;  // [batch][Hkv][D]
  const f16* new_v;
};
// Workspace: [tickets][ml: slots x Hkv x G x 2][o: slots x Hkv x G x D][lse: batch x Hkv x max_pages x G], fp32;
// slot = row + range.
struct F8Workspace {
  uint32_t* count;
  float* ml;
  float* o;
  float* lse;
};

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
#else
__device__ __forceinline__ f32x4 mfma16(f16x8, f16x8, f32x4 c) { return c; }
#endif

// One page of one head as loaded: K chunk i = 16 dims of token n, V row t = D / 16 dims of token 4 g + t.
template <int D>
struct F8Page {
  static constexpr int kKL = D / 64, kVW = D / 64;  // 16-byte chunks of K; words per V row
  u32x4 k[kKL];
  uint32_t v[4][kVW];
};

// Pages of row b in the list: its own, and kRowStart more in front when it has any.
__device__ __forceinline__ int f8_offsets(int* s_cum, int* s_wsum, const int32_t* seq_lens, const uint8_t* active,
                                          int batch, int cap) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int running = 0;
  for (int base = 0; base < batch; base += kF8DecThreads) {
    const int i = base + tid;
    int n = 0;
    if (i < batch) {
      const int sl = seq_lens[i];
      const int act = active != nullptr ? int(active[i]) : 1;
      const int len = act != 0 ? max(0, min(sl, cap)) : 0;
      n = (len + kF8Page - 1) / kF8Page;
      if (n > 0) n += kRowStart;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (lane == kWave - 1) s_wsum[wave] = x;
    __syncthreads();
    int pre = 0, tot = 0;
    for (int w = 0; w < kF8DecWaves; ++w) {
      const int v = s_wsum[w];
      pre += w < wave ? v : 0;
      tot += v;
    }
    if (i < batch) s_cum[i] = running + pre + x - n;
    running += tot;
    __syncthreads();
  }
  if (tid == 0) s_cum[batch] = running;
  __syncthreads();
  return running;
}

template <int D, bool kAppend, bool kWeights>
__global__ __launch_bounds__(kF8DecThreads) void decode_fp8_kernel(
    f16* __restrict__ out, const f16* __restrict__ q, F8Cache cache, const int32_t* __restrict__ block_tables,
    int32_t max_pages, const int32_t* __restrict__ seq_lens, const uint8_t* __restrict__ active, int32_t batch,
    int32_t hkv, int32_t G, int32_t max_len, float scale_log2, F8Workspace ws, F8Append ap,
    float* __restrict__ page_weights, int32_t streams) {
  constexpr int kKL = F8Page<D>::kKL, kVW = F8Page<D>::kVW;
  constexpr int kT = D / 16;   // output tiles (dims m D / 16 + tile)
  constexpr int kU = D / 16;   // 4-dim units of a lane's outputs: unit r (D / 64) + q = dims of row 4 g + r, 4 q ..
  __shared__ int s_cum[kF8MaxBatch + 1];
  __shared__ int s_wsum[kF8DecWaves];
  const int lane = threadIdx.x % kWave;
  const int n = lane % 16, g = lane / 16;
  const int cap = min(max_pages * kF8Page, max_len);
  const int T = f8_offsets(s_cum, s_wsum, seq_lens, active, batch, cap);

  const int64_t wave = int64_t(blockIdx.x) * kF8DecWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int stream = int(wave / hkv), h = int(wave % hkv);
  const int hq = hkv * G;

  // Active rows without keys get zeros: row b by wave b, b + waves, ... of the grid.
  for (int64_t b = wave; b < batch; b += int64_t(gridDim.x) * kF8DecWaves) {
    if (s_cum[b + 1] == s_cum[b] && (active == nullptr || active[b] != 0)) {
      for (int i = lane; i < hq * D / 8; i += kWave) st16(out + b * hq * D + i * 8, u32x4{0u, 0u, 0u, 0u});
    }
  }
  const int nr = min(streams, (T + kMinPages - 1) / kMinPages);
  if (stream >= nr) return;
  const int t0 = int(int64_t(T) * stream / nr), t1 = int(int64_t(T) * (stream + 1) / nr);
  auto range_of = [&](int t) -> int { return int((int64_t(t + 1) * nr - 1) / T); };

  const int64_t v_codes = cache.num_pages * hkv * (kF8Page * D), v_scales = cache.num_pages * hkv;
  const uint32_t k_lane = n * D + 16 * g, v_lane = 4 * g * D + n * (D / 16);

  int lo = 0, hi = batch - 1;  // the last row that starts at or before t0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_cum[mid] <= t0) lo = mid; else hi = mid - 1;
  }
  int npend = 0, pend_b[2] = {0, 0}, pend_f[2] = {0, 0}, pend_np[2] = {0, 0};

  // sum_g exp2(lse - total) of every page of (b, h), added to page_weights.  lse_n: lane n's (n < G) total.
  auto add_weights = [&](int b, float lse_n, int npages) {
    const int64_t seg = int64_t(b) * hkv + h;
    const float* pl = ws.lse + seg * max_pages * G;
    float* dst = page_weights + seg * max_pages;
    for (int j0 = 0; j0 < npages; j0 += kWave) {
      const int j = j0 + lane;
      float w = 0.f;
      for (int x = 0; x < G; ++x) {
        const float tot = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lse_n), x));
        if (j < npages) w += exp2_fast(ld_dev(pl + int64_t(j) * G + x) - tot);
      }
      if (j < npages) dst[j] += w;
    }
  };

  for (int b = lo; b < batch; ++b) {  // pieces of the range
    const int cb = __builtin_amdgcn_readfirstlane(s_cum[b]) + kRowStart;
    const int npages = __builtin_amdgcn_readfirstlane(s_cum[b + 1]) - cb;
    if (npages <= 0) continue;
    if (cb >= t1) break;
    const int a = max(t0, cb) - cb, e = min(t1, cb + npages) - cb;
    if (a >= e) continue;
    const int first = range_of(cb), nranges = range_of(cb + npages - 1) - first + 1;
    const int row_len = seq_lens[b], len = min(row_len, cap);
    const int32_t* bt = block_tables + int64_t(b) * max_pages;

    // queries: column n holds head h G + n (columns from G on: zeros), in K's order of dims
    f16x8 qf[2 * kKL];
    {
      const f16* qp = q + (int64_t(b) * hq + h * G + min(n, G - 1)) * D + 16 * g;
#pragma unroll
      for (int i = 0; i < kKL; ++i) {
        const u32x4 z = u32x4{0u, 0u, 0u, 0u};
        const u32x4 x0 = ld16(qp + 64 * i), x1 = ld16(qp + 64 * i + 8);
        qf[2 * i] = as_h8(n < G ? x0 : z);
        qf[2 * i + 1] = as_h8(n < G ? x1 : z);
      }
    }
    // page ids and scales, 64 per window, one per lane
    int ids = 0, win = a;
    float ksc = 0.f, vsc = 0.f;
    auto load_window = [&](int w0) {
      win = w0;
      const int id = bt[min(w0 + lane, e - 1)];
      const bool ok = id >= 0 && int64_t(id) < cache.num_pages;
      ids = ok ? id : -1;
      const int64_t at = int64_t(ok ? id : 0) * hkv + h;
      ksc = cache.scales[at];
      vsc = cache.scales[v_scales + at];
    };
    load_window(a);

    auto issue_page = [&](int p, F8Page<D>& r) __attribute__((always_inline)) {
      const int id = max(__builtin_amdgcn_readlane(ids, p - win), 0);
      const uint8_t* kb = cache.codes + f8_block<D>(id, hkv, h);
      const uint8_t* vb = kb + v_codes;
#pragma unroll
      for (int i = 0; i < kKL; ++i) r.k[i] = ld16_stream(kb + k_lane + 64 * i);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint8_t* p4 = vb + v_lane + t * D;
        if constexpr (kVW == 1) {
          r.v[t][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p4));
        } else if constexpr (kVW == 2) {
          const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p4));
          r.v[t][0] = x[0];
          r.v[t][1] = x[1];
        } else {
          const u32x4 x = ld16_stream(p4);
#pragma unroll
          for (int j = 0; j < 4; ++j) r.v[t][j % kVW] = x[j];
        }
      }
    };

    float m = kNegBig, l = 0.f;
    f32x4 acc[kT];
#pragma unroll
    for (int i = 0; i < kT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The step's token into the row's last page, in registers: new scales, codes, and the stores.
    auto append = [&](F8Page<D>& r, float& ks, float& vs, int id) {
      const int off = (len - 1) % kF8Page;
      const f16* nk = ap.new_k + (int64_t(b) * hkv + h) * D;
      const f16* nv = ap.new_v + (int64_t(b) * hkv + h) * D;
      f16x8 xk[2 * kKL];
      float ka = 0.f, va = 0.f;
#pragma unroll
      for (int i = 0; i < kKL; ++i) {
        xk[2 * i] = as_h8(ld16(nk + 64 * i + 16 * g));
        xk[2 * i + 1] = as_h8(ld16(nk + 64 * i + 16 * g + 8));
      }
      f16 xv[4 * kVW];
#pragma unroll
      for (int j = 0; j < 4 * kVW; j += 4) {
        const f16x4 x = *reinterpret_cast<const f16x4*>(nv + n * (D / 16) + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          xv[j + c] = x[c];
          va = fmaxf(va, fabsf(float(x[c])));
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * kKL; ++i) ka = fmaxf(ka, f8_amax8(xk[i]));
      ka = max_lane32(swap_max16(ka));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) va = fmaxf(va, __shfl_xor(va, o));
      const float nks = f8_pow2(f8_need_exp(ka)), nvs = f8_pow2(f8_need_exp(va));
      const float ks1 = off == 0 ? nks : fmaxf(ks, nks), vs1 = off == 0 ? nvs : fmaxf(vs, nvs);
      const bool k_all = off == 0 || ks1 != ks, v_all = off == 0 || vs1 != vs;  // (uniform)
      if (k_all) {
#pragma unroll
        for (int i = 0; i < kKL; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) r.k[i][j] = off == 0 ? 0u : f8_rescale(r.k[i][j], ks / ks1);
      }
      if (v_all) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < kVW; ++j) r.v[t][j] = off == 0 ? 0u : f8_rescale(r.v[t][j], vs / vs1);
      }
      const float ki = 1.f / ks1, vi = 1.f / vs1;
#pragma unroll
      for (int i = 0; i < kKL; ++i) {
        const u32x2 c0 = f8_quant8(xk[2 * i], ki), c1 = f8_quant8(xk[2 * i + 1], ki);
        if (n == off) r.k[i] = u32x4{c0[0], c0[1], c1[0], c1[1]};
      }
#pragma unroll
      for (int j = 0; j < kVW; ++j) {
        const uint32_t c = f8_pack(float(xv[4 * j]) * vi, float(xv[4 * j + 1]) * vi, float(xv[4 * j + 2]) * vi,
                                   float(xv[4 * j + 3]) * vi);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (4 * g + t == off) r.v[t][j] = c;
      }
      uint8_t* kb = cache.codes + f8_block<D>(id, hkv, h);
      uint8_t* vb = kb + v_codes;
      if (k_all || n == off) {
#pragma unroll
        for (int i = 0; i < kKL; ++i) st16(kb + k_lane + 64 * i, r.k[i]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (v_all || 4 * g + t == off) {
#pragma unroll
          for (int j = 0; j < kVW; ++j) *reinterpret_cast<uint32_t*>(vb + v_lane + t * D + 4 * j) = r.v[t][j];
        }
      }
      if (lane == 0) {
        const int64_t at = int64_t(id) * hkv + h;
        if (k_all) cache.scales[at] = ks1;
        if (v_all) cache.scales[v_scales + at] = vs1;
      }
      ks = ks1;
      vs = vs1;
    };

    // Pages p and p + 1 (two: whether the second is in the piece).
    auto consume = [&](int p, bool two, F8Page<D>& r0, F8Page<D>& r1) __attribute__((always_inline)) {
      f32x4 s[2];
      float vs[2];
      bool live[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        F8Page<D>& r = x == 0 ? r0 : r1;
        const int at = x == 0 || two ? p + x - win : p - win;
        const int id = __builtin_amdgcn_readlane(ids, at);
        live[x] = id >= 0 && (x == 0 || two);
        float ks = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ksc), at));
        vs[x] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vsc), at));
        if constexpr (kAppend) {
          if (live[x] && p + x == npages - 1 && row_len <= cap) append(r, ks, vs[x], id);
        }
        s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKL; ++i) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t w0 = r.k[i][2 * half], w1 = r.k[i][2 * half + 1];
            const f16x2 h0 = f8_to_f16<false>(w0, ks), h1 = f8_to_f16<true>(w0, ks), h2 = f8_to_f16<false>(w1, ks),
                        h3 = f8_to_f16<true>(w1, ks);
            s[x] = mfma16(f16x8{h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]}, qf[2 * i + half], s[x]);
          }
        }
      }
      // scores in base 2; tokens past the row's end, and of pages outside the pool, have none
      float sv[8];
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int left = live[x] ? len - (p + x) * kF8Page : 0;
        if (left < kF8Page) {  // (uniform)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool in = 4 * g + j < left;
            sv[4 * x + j] = in ? s[x][j] * scale_log2 : -INFINITY;
#pragma unroll
            for (int c = 0; c < kVW; ++c) {  // (their codes may be anything, and 0 x NaN is NaN)
              uint32_t& w = (x == 0 ? r0 : r1).v[j][c];
              w = in ? w : 0u;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) sv[4 * x + j] = s[x][j] * scale_log2;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, sv[j]);
      mx = max_lane32(swap_max16(mx));
      if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
        const float mn = fmaxf(m, mx);
        const float al = exp2_fast(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int i = 0; i < kT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] *= al;
      }
      float pr[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) pr[j] = exp2_fast(sv[j] - m);
      const float l0 = (pr[0] + pr[1]) + (pr[2] + pr[3]), l1 = (pr[4] + pr[5]) + (pr[6] + pr[7]);
      l += l0 + l1;
      if constexpr (kWeights) {
        const float w0 = swap_sum(l0), w1 = swap_sum(l1);
        if (g == 0 && n < G) {
          float* dst = ws.lse + ((int64_t(b) * hkv + h) * max_pages + p) * G + n;
          st_dev(dst, __builtin_amdgcn_logf(w0) + m);
          if (two) st_dev(dst + G, __builtin_amdgcn_logf(w1) + m);
        }
      }
      const f16x8 pf = f16x8{f16(pr[0]), f16(pr[1]), f16(pr[2]), f16(pr[3]), f16(pr[4]), f16(pr[5]), f16(pr[6]), f16(pr[7])};
#pragma unroll
      for (int c = 0; c < kVW; ++c) {
        uint32_t tr[2][4];  // byte transposes: word i = dim 4 c + i of tokens 4 g .. 4 g + 3
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const F8Page<D>& r = x == 0 ? r0 : r1;
          const uint32_t ab = __builtin_amdgcn_perm(r.v[1][c], r.v[0][c], 0x05010400u);
          const uint32_t ab2 = __builtin_amdgcn_perm(r.v[1][c], r.v[0][c], 0x07030602u);
          const uint32_t cd = __builtin_amdgcn_perm(r.v[3][c], r.v[2][c], 0x05010400u);
          const uint32_t cd2 = __builtin_amdgcn_perm(r.v[3][c], r.v[2][c], 0x07030602u);
          tr[x][0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
          tr[x][1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
          tr[x][2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
          tr[x][3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x2 h0 = f8_to_f16<false>(tr[0][i], vs[0]), h1 = f8_to_f16<true>(tr[0][i], vs[0]),
                      h2 = f8_to_f16<false>(tr[1][i], vs[1]), h3 = f8_to_f16<true>(tr[1][i], vs[1]);
          acc[4 * c + i] = mfma16(f16x8{h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]}, pf, acc[4 * c + i]);
        }
      }
    };

    F8Page<D> a0, a1, b0, b1;
    for (int w0 = a; w0 < e; w0 += kWave) {  // windows of 64 pages
      const int we = min(w0 + kWave, e);
      if (w0 != a) load_window(w0);
      const int steps = (we - w0 + 1) / 2;
      auto issue = [&](int i, F8Page<D>& r0, F8Page<D>& r1) __attribute__((always_inline)) {
        const int p = w0 + 2 * i;
        issue_page(p, r0);
        issue_page(min(p + 1, we - 1), r1);
      };
      auto step = [&](int i, F8Page<D>& r0, F8Page<D>& r1) __attribute__((always_inline)) {
        consume(w0 + 2 * i, w0 + 2 * i + 1 < we, r0, r1);
      };
      issue(0, a0, a1);
      int i = 0;
      for (; i + 2 < steps; i += 2) {
        issue(i + 1, b0, b1);
        __builtin_amdgcn_sched_barrier(0);
        step(i, a0, a1);
        issue(i + 2, a0, a1);
        __builtin_amdgcn_sched_barrier(0);
        step(i + 1, b0, b1);
      }
      if (i + 1 < steps) {
        issue(i + 1, b0, b1);
        __builtin_amdgcn_sched_barrier(0);
        step(i, a0, a1);
        step(i + 1, b0, b1);
      } else {
        step(i, a0, a1);
      }
    }

    l = swap_sum(l);
    if (nranges == 1) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (n < G) {
        f16* op = out + (int64_t(b) * hq + h * G + n) * D + 4 * g * (D / 16);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < kVW; ++c)
            *reinterpret_cast<f16x4*>(op + r * (D / 16) + 4 * c) =
                f16x4{f16(acc[4 * c][r] * inv), f16(acc[4 * c + 1][r] * inv), f16(acc[4 * c + 2][r] * inv),
                      f16(acc[4 * c + 3][r] * inv)};
      }
      if constexpr (kWeights) {
        wait_all_mem();  // (this wave's own lse stores)
        add_weights(b, l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY, npages);
      }
    } else {
      const int64_t slot = (int64_t(b) + stream) * hkv + h;
      if (n < G) {
        if (g == 0) st_dev8(ws.ml + (slot * G + n) * 2, f32x2{m, l});
        float* so = ws.o + slot * G * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < kVW; ++c) {
            float* dst = so + ((r * kVW + c) * 4 * G + g * G + n) * 4;
            st_dev8(dst, f32x2{acc[4 * c][r], acc[4 * c + 1][r]});
            st_dev8(dst + 2, f32x2{acc[4 * c + 2][r], acc[4 * c + 3][r]});
          }
      }
      pend_b[npend & 1] = b;  // (only the first and the last piece of a range can be split)
      pend_f[npend & 1] = first;
      pend_np[npend & 1] = nranges;
      ++npend;
    }
  }

  for (int x = 0; x < npend; ++x) {
    const int b = x == 0 ? pend_b[0] : pend_b[1], np = x == 0 ? pend_np[0] : pend_np[1];
    const int first = x == 0 ? pend_f[0] : pend_f[1];
    uint32_t* ticket = ws.count + int64_t(b) * hkv + h;
    if (!wave_arrive_last(ticket, uint32_t(np - 1), lane)) continue;
    const int64_t slot0 = (int64_t(b) + first) * hkv + h;  // state j: slot0 + j hkv
    // totals of query n % G
    float M = kNegBig, L = 0.f;
    const int nn = min(n, G - 1);
    for (int j = 0; j < np; ++j) {
      const f32x2 ml = ld_dev8(ws.ml + ((slot0 + int64_t(j) * hkv) * G + nn) * 2);
      const float mn = fmaxf(M, ml[0]);
      L = L * exp2_fast(M - mn) + ml[1] * exp2_fast(ml[0] - mn);
      M = mn;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    for (int u0 = 0; u0 < kU * 4 * G; u0 += kWave) {  // 4-dim units: (r kVW + c) 4 G + g G + n
      const int u = u0 + lane;
      const bool on = u < kU * 4 * G;
      const int cl = u % (4 * G), un = cl % G, ug = cl / G, i4 = u / (4 * G);
      const float Mu = __shfl(M, un), iu = __shfl(inv, un);
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
      if (on) {
        for (int j = 0; j < np; ++j) {
          const int64_t sl = slot0 + int64_t(j) * hkv;
          const float w = exp2_fast(ld_dev(ws.ml + (sl * G + un) * 2) - Mu);
          const float* src = ws.o + sl * G * D + u * 4;
          const f32x2 x0 = ld_dev8(src), x1 = ld_dev8(src + 2);
          o = f32x4{fmaf(w, x0[0], o[0]), fmaf(w, x0[1], o[1]), fmaf(w, x1[0], o[2]), fmaf(w, x1[1], o[3])};
        }
        *reinterpret_cast<f16x4*>(out + (int64_t(b) * hq + h * G + un) * D + (4 * ug + i4 / kVW) * (D / 16) + 4 * (i4 % kVW)) =
            f16x4{f16(o[0] * iu), f16(o[1] * iu), f16(o[2] * iu), f16(o[3] * iu)};
      }
    }
    if constexpr (kWeights) {
      const int npages = s_cum[b + 1] - s_cum[b] - kRowStart;
      add_weights(b, L > 0.f ? M + __builtin_amdgcn_logf(L) : INFINITY, __builtin_amdgcn_readfirstlane(npages));
    }
    if (lane == 0) reset_ticket(ticket);
  }
}

// Streams of a call: at most one wave per kv head and stream, kF8WavesPerCu waves a CU, and no more than the
// longest call of these sizes has ranges.
constexpr int kF8WavesPerCu = 8;
static int64_t f8_streams(int64_t batch, int32_t hkv, int32_t max_len, int cus) {
  const int64_t most = ceil_div(batch * (ceil_div(max_len, kF8Page) + kRowStart), kMinPages);
  const int64_t waves = int64_t(cus) * kF8WavesPerCu;
  return std::max<int64_t>(1, std::min(most, std::max<int64_t>(1, waves / hkv)));
}
static size_t f8_ws_layout(int64_t batch, int64_t streams, int32_t hkv, int32_t G, int32_t d, int32_t max_pages,
                           bool weights, size_t* off_ml, size_t* off_o, size_t* off_lse) {
  const size_t slots = size_t(batch + streams) * hkv * G;
  size_t off = kTicketBytes;
  *off_ml = off;
  off = align256(off + slots * 2 * sizeof(float));
  *off_o = off;
  off = align256(off + slots * d * sizeof(float));
  *off_lse = off;
  if (weights) off = align256(off + size_t(batch) * hkv * max_pages * G * sizeof(float));
  return off;
}

static int f8_decode(void* out, const void* query, void* codes, float* scales, int64_t num_pages,
                     const int32_t* block_tables, int32_t max_pages, const int32_t* seq_lens,
                     const uint8_t* active, const void* new_k, const void* new_v, bool append, float* page_weights,
                     int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t block_size, int32_t max_len,
                     float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (out == nullptr || query == nullptr || codes == nullptr || scales == nullptr || block_tables == nullptr ||
      seq_lens == nullptr || (append && (new_k == nullptr || new_v == nullptr)))
    return IFN_ERR_INVALID_ARGUMENT;
  if (batch < 0 || hq < 1 || hkv < 1 || hq % hkv != 0 || d < 1 || block_size < 1 || num_pages < 1 || max_pages < 1 ||
      max_len < 0)
    return IFN_ERR_INVALID_ARGUMENT;
  const int32_t G = hq / hkv;
  if (block_size != kF8Page || (d != 64 && d != 128 && d != 256) || G > kF8MaxGroup || batch > kF8MaxBatch ||
      int64_t(batch) * hkv > kMaxTickets || max_pages > (1 << 27) / kF8Page ||
      int64_t(batch) * (max_pages + kRowStart) > (int64_t(1) << 30) || num_pages > (int64_t(1) << 31) / kF8Page)
    return IFN_ERR_UNSUPPORTED;
  IFN_CHECK_ALIGN16(out);
  IFN_CHECK_ALIGN16(query);
  IFN_CHECK_ALIGN16(codes);
  if (append) {
    IFN_CHECK_ALIGN16(new_k);
    IFN_CHECK_ALIGN16(new_v);
  }
  if (batch == 0) return IFN_OK;
  const int32_t cap = int32_t(std::min<int64_t>(int64_t(max_pages) * kF8Page, max_len));
  const int cus = device_cu_count();
  if (workspace == nullptr) return IFN_ERR_WORKSPACE;
  IFN_CHECK_ALIGN16(workspace);
  const int64_t streams = f8_streams(batch, hkv, cap, std::max(1, cus));
  size_t off_ml, off_o, off_lse;
  if (workspace_bytes < f8_ws_layout(batch, streams, hkv, G, d, max_pages, page_weights != nullptr, &off_ml, &off_o,
                                     &off_lse))
    return IFN_ERR_WORKSPACE;
  if (cus < 1) return IFN_ERR_HIP;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const F8Workspace ws{reinterpret_cast<uint32_t*>(w), reinterpret_cast<float*>(w + off_ml),
                       reinterpret_cast<float*>(w + off_o), reinterpret_cast<float*>(w + off_lse)};
  const F8Cache cache{static_cast<uint8_t*>(codes), scales, num_pages};
  const F8Append ap{static_cast<const f16*>(new_k), static_cast<const f16*>(new_v)};
  const float sl = (scale > 0.f ? scale : 1.f / sqrtf(float(d))) * kLog2e;
  const int64_t blocks = ceil_div(streams * hkv, kF8DecWaves);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto k) {
    k<<<dim3(unsigned(blocks)), dim3(kF8DecThreads), 0, s>>>(
        static_cast<f16*>(out), static_cast<const f16*>(query), cache, block_tables, max_pages, seq_lens, active, batch,
        hkv, G, cap, sl, ws, ap, page_weights, int32_t(streams));
  };
  auto pick = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    const bool wt = page_weights != nullptr;
    if (append) wt ? launch(decode_fp8_kernel<D, true, true>) : launch(decode_fp8_kernel<D, true, false>);
    else wt ? launch(decode_fp8_kernel<D, false, true>) : launch(decode_fp8_kernel<D, false, false>);
  };
  if (d == 64) pick(std::integral_constant<int, 64>{});
  else if (d == 128) pick(std::integral_constant<int, 128>{});
  else pick(std::integral_constant<int, 256>{});
  return ifn_launch_status();
}

}  // namespace ifn

extern "C" size_t ifn_paged_decode_fp8_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                       int32_t head_dim, int32_t block_size,
                                                       int32_t max_pages_per_seq, int32_t max_seq_len,
                                                       int32_t page_weights) {
  using namespace ifn;
  if (batch < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads != 0 || head_dim < 1 ||
      block_size < 1 || max_pages_per_seq < 1 || max_seq_len < 0)
    return 0;
  const int64_t cap = std::min<int64_t>(int64_t(max_pages_per_seq) * kF8Page, max_seq_len);
  const int64_t streams = f8_streams(batch, num_kv_heads, int32_t(cap), std::max(1, device_cu_count()));
  size_t a, b, c;
  return f8_ws_layout(batch, streams, num_kv_heads, num_q_heads / num_kv_heads, head_dim, max_pages_per_seq,
                      page_weights != 0, &a, &b, &c);
}

extern "C" int ifn_paged_decode_fp8(void* out, const void* query, const void* codes_layer,
                                    const float* scales_layer, int64_t num_pages, const int32_t* block_tables,
                                    int32_t max_pages_per_seq, const int32_t* seq_lens, const uint8_t* active_mask,
                                    float* page_weights, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                    int32_t head_dim, int32_t block_size, int32_t max_seq_len, float scale,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  return ifn::f8_decode(out, query, const_cast<void*>(codes_layer), const_cast<float*>(scales_layer), num_pages,
                        block_tables, max_pages_per_seq, seq_lens, active_mask, nullptr, nullptr, false, page_weights,
                        batch, num_q_heads, num_kv_heads, head_dim, block_size, max_seq_len, scale, workspace,
                        workspace_bytes, stream);
}

extern "C" int ifn_paged_decode_append_fp8(void* out, const void* query, void* codes_layer, float* scales_layer,
                                           int64_t num_pages, const int32_t* block_tables,
                                           int32_t max_pages_per_seq, const int32_t* seq_lens,
                                           const uint8_t* active_mask, const void* new_k, const void* new_v,
                                           float* page_weights, int32_t batch, int32_t num_q_heads,
                                           int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                           int32_t max_seq_len, float scale, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  return ifn::f8_decode(out, query, codes_layer, scales_layer, num_pages, block_tables, max_pages_per_seq, seq_lens,
                        active_mask, new_k, new_v, true, page_weights, batch, num_q_heads, num_kv_heads, head_dim,
                        block_size, max_seq_len, scale, workspace, workspace_bytes, stream);
}
