// Paged GQA decode over the 8-bit KV cache (gfx950 MFMA), with the step's append and the pages' attention
// weights fused in.
//
// The 8-bit form of the reference's documented paged_attention for decode (docs/architecture.md:246;
// contiguous semantics src/infurnace/executor/tinygrad/model.py:196-200): out = softmax(scale q K^T) V over the
// row's first L tokens, query head h reading kv head h / G.  Blocks and scales: kv_fp8.hpp.
//
//  * A wave attends one kv head.  The pages of all rows, row after row, form one list per head, which the grid's
//    waves cut into ranges: stream r takes pages [T r / nr, T (r+1) / nr), so ragged batches cost every wave the
//    same bytes.  Hkv and the group size G (up to 16) are run-time numbers.
//  * S^T = K Q^T with v_mfma_f32_16x16x32_f16 and O^T += V^T P^T with v_mfma_f32_16x16x16_f16, the group's queries in
//    the 16 columns, a page's tokens in the 16 rows.  Lane (n = lane % 16, g = lane / 16) loads K of token n, dims
//    64 i + 16 g .. + 15 (the fragments' k order is theirs to choose, as long as Q's is the same), gets the scores of
//    query n and tokens 4 g .. 4 g + 3, and needs V of the same tokens for the second product: it loads 4 token rows
//    x D / 16 dims of V and transposes the bytes (v_perm).  So codes go from memory to the matrix cores without LDS
//    and without an exchange between lanes; only the running maximum is reduced over the four g (v_permlane swaps).
//    The running sum stays a lane's own until the end.
//  * Codes become fp16 exactly (kv_fp8.hpp).  Probabilities are rounded to fp16 for the second product (2^-12
//    relative, averaged over the keys); scores, maxima, sums and outputs are fp32.
//  * A row held by several ranges: the four waves of a workgroup have consecutive ranges of one head and merge their
//    states (m, l, O in fp32) in LDS; what other workgroups hold too goes to the workspace, and the workgroup that
//    arrives last, by a ticket per (row, head), merges it in range order.
//  * Fused append (kAppend): the wave that holds a row's last page adds the row's new token to the block in
//    its registers (new scale, rescaled codes), stores what changed and attends over the result.
//  * Page weights (kWeights): each page's log2-sum-exp per query head goes to the workspace; whoever finishes a
//    (row, head) turns them into sum_g exp2(lse - total) and adds them to page_weights.
//
// What bounds it: memory, above about 100 MB.  128 rows of 1023-8190 keys, 32 / 8 heads x 128 (1.21 GB): 203-213 us on
// different cards, 5.7-6.0 TB/s; 32 rows of 128-4096, 16 / 8 heads (143 MB): 33 us, of which about 4 before a wave's
// first page (lengths, ids, scales), 20 streaming, 3 of uneven waves and 6 after (states written through to memory,
// ticket, merge).  One row of 512 keys: 8.6 us, all of it those steps.
#include <algorithm>
#include <type_traits>

#include "kv_fp8.hpp"

namespace ifn {

// Threads of a workgroup.  Small ones: a workgroup's waves wait for each other before they merge (one row of 512
// keys 8.7 us with 256, 10.3 with 512; 48 rows of 100-4000, 2 kv heads, 22.5 and 24.2).
constexpr int kDecThreads = 256;
constexpr int kDecWaves = kDecThreads / kWave;
constexpr int kDecPerSimd = 2;     // waves a SIMD is to hold (registers)
constexpr int f8_per_simd(int d) { return d == 256 ? 1 : kDecPerSimd; }
// Pages in a wave's ring.  The memory is as busy with 2 as with 4 (128 rows of 1023-8190 keys: 203 and 204 us), and
// short pieces request fewer pages twice (32 rows of 128-4096: 33.6 and 35.6 us).
constexpr int kRing = 2;
constexpr int kF8MaxBatch = 4096;  // rows per call (LDS offsets)
constexpr int kF8MaxGroup = 16;    // query heads per kv head (MFMA columns)
// Pages a row's start counts for in the split: its ids, scales and query take three round trips before the first
// page, and its state is merged.  With 3, 9 and 16: 48 rows of 100-4000 keys, 2 kv heads, 22.5, 20.3 and 20.2 us; 32
// rows of 128-4096 33.5, 33.2 and 33.6; one row of 512 8.7, 8.6 and 9.2 (the start's own ranges have nothing to do).
constexpr int kRowStart = 9;
constexpr int kMinPages = 2;       // fewest list positions per range
// Most ranges per row of the call.  A row's states are merged 16 workgroups a round trip, so more than 64 waves a row
// cost another one (one row of 8000 keys, 32 / 8 heads: 16.2, 13.1, 14.2 and 18.8 us with 32, 64, 128 and 256 ranges).
constexpr int kMaxRanges = 64;

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
// slot = row + workgroup (of a head).
struct F8Workspace {
  uint32_t* count;
  float* ml;
  float* o;
  float* lse;
};

// Pages of row b in the list: its own, and kRowStart more in front when it has any.
__device__ __forceinline__ int f8_row(const int32_t* seq_lens, const uint8_t* active, int b, int cap) {
  const int sl = seq_lens[b];
  const int act = active != nullptr ? int(active[b]) : 1;
  const int n = ((act != 0 ? max(0, min(sl, cap)) : 0) + kF8Page - 1) / kF8Page;
  return n > 0 ? n + kRowStart : 0;
}
__device__ __forceinline__ int f8_wave_scan(int x) {  // inclusive
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// Offsets of the rows, s_cum[0 .. batch]; returns the total.  Up to 64 rows every wave computes (and stores) them all, so
// that no wave waits for another.
template <int kWaves>
__device__ __forceinline__ int f8_offsets(int* s_cum, int* s_wsum, const int32_t* seq_lens, const uint8_t* active,
                                          int batch, int cap) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  if (batch <= kWave) {
    const int n = lane < batch ? f8_row(seq_lens, active, lane, cap) : 0;
    const int x = f8_wave_scan(n);
    if (lane < batch) s_cum[lane] = x - n;
    const int total = __builtin_amdgcn_readlane(x, kWave - 1);
    if (lane == 0) s_cum[batch] = total;
    return total;
  }
  int running = 0;
  for (int base = 0; base < batch; base += kWaves * kWave) {
    const int i = base + tid;
    const int n = i < batch ? f8_row(seq_lens, active, i, cap) : 0;
    const int x = f8_wave_scan(n);
    if (lane == kWave - 1) s_wsum[wave] = x;
    __syncthreads();
    int pre = 0, tot = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
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

// The end of a row split over ranges: its np states, slots slot0 + j hkv, merged in range order for the 4-dim unit u
// of query un (kMergeBatch states a round trip).
constexpr int kMergeBatch = 16;
__device__ __forceinline__ void f8_merge(__amdgpu_buffer_rsrc_t r_ml, __amdgpu_buffer_rsrc_t r_o, int64_t slot0, int hkv,
                                         int np, int G, int D, int un, int u, float& M, float& L, f32x4& O) {
  M = kNegBig;
  L = 0.f;
  O = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < np; j0 += kMergeBatch) {
    const int cnt = min(kMergeBatch, np - j0);
    f32x2 ml[kMergeBatch];
    f32x4 o[kMergeBatch];
#pragma unroll
    for (int x = 0; x < kMergeBatch; ++x) {
      if (x < cnt) {
        const uint32_t sl = uint32_t(slot0 + int64_t(j0 + x) * hkv);
        ml[x] = ld_dev2(r_ml, (sl * G + un) * 8);
        o[x] = ld_dev4(r_o, (sl * G * D + u * 4) * 4);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    float gm = M;
#pragma unroll
    for (int x = 0; x < kMergeBatch; ++x)
      if (x < cnt) gm = fmaxf(gm, ml[x][0]);
    const float sc = exp2_fast(M - gm);
    M = gm;
    L *= sc;
    O = f32x4{O[0] * sc, O[1] * sc, O[2] * sc, O[3] * sc};
#pragma unroll
    for (int x = 0; x < kMergeBatch; ++x) {
      if (x < cnt) {
        const float w = exp2_fast(ml[x][0] - M);
        L = fmaf(w, ml[x][1], L);
        O = f32x4{fmaf(w, o[x][0], O[0]), fmaf(w, o[x][1], O[1]), fmaf(w, o[x][2], O[2]), fmaf(w, o[x][3], O[3])};
      }
    }
  }
}

template <int D, bool kAppend, bool kWeights>
__global__ __launch_bounds__(kDecThreads, f8_per_simd(D)) void decode_fp8_kernel(
    const int32_t* __restrict__ seq_lens, const uint8_t* __restrict__ active, int32_t batch, int32_t max_pages,
    int32_t max_len, int32_t hkv, int32_t G, int32_t streams, const int32_t* __restrict__ block_tables,
    const f16* __restrict__ q,  // (up to here in registers at dispatch: build.py)
    F8Cache cache, f16* __restrict__ out, float scale_log2, F8Workspace ws, F8Append ap,
    float* __restrict__ page_weights) {
  constexpr int kKL = F8Page<D>::kKL, kVW = F8Page<D>::kVW;
  constexpr int kT = D / 16;   // output tiles (dims m D / 16 + tile)
  constexpr int kU = D / 16;   // 4-dim units of a lane's outputs: unit r (D / 64) + q = dims of row 4 g + r, 4 q ..
  constexpr int kWaves = kDecWaves;
  constexpr int S = kRing;
  static_assert(kWave % S == 0, "windows are whole turns of the ring");
  constexpr int kEnt = 2 * kWaves;  // states a workgroup has at its end: at most two a wave
  __shared__ int s_wsum[kWaves];
  __shared__ int s_row[kEnt], s_span[kEnt];  // a state's row (-1: none), and the workgroups that hold it: first << 16 | last
  __shared__ float s_m[kEnt][kF8MaxGroup], s_l[kEnt][kF8MaxGroup], s_tot[kF8MaxGroup];
  __shared__ uint32_t s_ticket[2];
  extern __shared__ __attribute__((aligned(16))) f32x4 s_o[];  // [kEnt][G D / 4], then the rows' offsets [batch + 1]
  int* const s_cum = reinterpret_cast<int*>(s_o + kEnt * G * (D / 4));
  const int lane = threadIdx.x % kWave;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // kWeights, behind them: a wave's page sums of one window, [kWaves][64][G]
  float* const my_lse = reinterpret_cast<float*>(s_cum + batch + 1) + wv * kWave * G;
  const int n = lane % 16, g = lane / 16;
  const int cap = min(max_pages * kF8Page, max_len);
  const int T = f8_offsets<kWaves>(s_cum, s_wsum, seq_lens, active, batch, cap);

  const int h = int(blockIdx.x) % hkv, wg = int(blockIdx.x) / hkv;
  const int stream = wg * kWaves + wv;
  const int hq = hkv * G;

  // Active rows without keys get zeros: row b by wave b, b + waves, ... of the grid.
  for (int64_t b = int64_t(blockIdx.x) * kWaves + wv; b < batch; b += int64_t(gridDim.x) * kWaves) {
    if (s_cum[b + 1] == s_cum[b] && (active == nullptr || active[b] != 0)) {
      for (int i = lane; i < hq * D / 8; i += kWave) st16(out + b * hq * D + i * 8, u32x4{0u, 0u, 0u, 0u});
    }
  }
  const int nr = min(min(streams, kMaxRanges * batch), (T + kMinPages - 1) / kMinPages);
  if (wg * kWaves >= nr) return;
  const bool works = stream < nr;  // (the workgroup's last waves may have no range)
  // the first `rem` ranges have base + 1 pages, the others base
  const uint32_t base = uint32_t(T) / uint32_t(nr), rem = uint32_t(T) - base * nr, bend = rem * (base + 1);
  const int t0 = works ? int(stream * base + min(uint32_t(stream), rem)) : T;
  const int t1 = works ? t0 + int(base) + (uint32_t(stream) < rem ? 1 : 0) : T;
  auto range_of = [&](int t) -> int {
    const uint32_t u = uint32_t(t);
    return int(u < bend ? u / (base + 1) : rem + (u - bend) / base);
  };

  const int64_t v_codes = cache.num_pages * hkv * (kF8Page * D), v_scales = cache.num_pages * hkv;
  const uint32_t k_lane = n * D + 16 * g, v_lane = 4 * g * D + n * (D / 16);
  const int units = kU * 4 * G;  // 4-dim units of a state: (x kVW + c) 4 G + g G + n
  const uint32_t n_states = uint32_t(batch + streams / kWaves) * hkv * G;
  const __amdgpu_buffer_rsrc_t r_ml = make_rsrc(ws.ml, n_states * 8u), r_o = make_rsrc(ws.o, n_states * D * 4u);

  int lo = 0, hi = batch - 1;  // the last row that starts at or before t0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_cum[mid] <= t0) lo = mid; else hi = mid - 1;
  }
  int npend = 0;  // this wave's states of rows that other ranges hold too: the range's first and last piece, at most
  if (lane < 2) s_row[2 * wv + lane] = -1;

  // sum_g exp2(lse - total) of every page of (b, h), added to page_weights by `threads` threads, the id-th of them here.
  auto add_weights = [&](int b, auto total, int npages, int id, int threads) __attribute__((always_inline)) {
    const int64_t seg = int64_t(b) * hkv + h;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(ws.lse + seg * max_pages * G, uint32_t(npages) * G * 4u);
    float* dst = page_weights + seg * max_pages;
    constexpr int kB = 4;  // pages a thread has in flight
    for (int j0 = 0; j0 < npages; j0 += kB * threads) {
      float w[kB];
#pragma unroll
      for (int c = 0; c < kB; ++c) {
        const int j = j0 + c * threads + id;
        w[c] = j < npages ? dst[j] : 0.f;
      }
      for (int x = 0; x < G; x += 4) {  // (the words past a page's group are not used)
        f32x4 v[kB];
#pragma unroll
        for (int c = 0; c < kB; ++c) v[c] = ld_dev4(r, uint32_t((j0 + c * threads + id) * G + x) * 4u);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float tot = total(min(x + y, G - 1));
          if (x + y < G) {
#pragma unroll
            for (int c = 0; c < kB; ++c) w[c] += exp2_fast(v[c][y] - tot);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kB; ++c) {
        const int j = j0 + c * threads + id;
        if (j < npages) dst[j] = w[c];
      }
    }
  };

  for (int b = lo; b < batch && works; ++b) {  // pieces of the range
    const int cb = __builtin_amdgcn_readfirstlane(s_cum[b]) + kRowStart;
    const int npages = __builtin_amdgcn_readfirstlane(s_cum[b + 1]) - cb;
    if (npages <= 0) continue;
    if (cb >= t1) break;
    const int a = max(t0, cb) - cb, e = min(t1, cb + npages) - cb;
    if (a >= e) continue;
    const int32_t* bt = block_tables + int64_t(b) * max_pages + a;
    const int np = e - a;  // the piece's pages, counted from 0 below

    // page ids and scales, one per lane: the window of 64 pages that is being attended and the next one
    auto load_ids = [&](int w) {
      const int id = bt[min(w * kWave + lane, np - 1)];
      return id;
    };
    auto in_pool = [&](int id) { return id >= 0 && int64_t(id) < cache.num_pages; };
    auto load_scale = [&](int id, int64_t half) { return cache.scales[half + int64_t(in_pool(id) ? id : 0) * hkv + h]; };
    int win = 0;
    int ids0 = load_ids(0), ids1 = load_ids(1);
    const int row_len = seq_lens[b], len = min(row_len, cap);

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
    // the step's token, when its page is in this piece: K dims as a lane's of K, V dims as of V
    const bool appends = kAppend && e == npages && row_len <= cap;
    f16x8 xk[kAppend ? 2 * kKL : 1];
    f16x4 xv[kAppend ? kVW : 1];
    if constexpr (kAppend) {
      if (appends) {
        const f16* nk = ap.new_k + (int64_t(b) * hkv + h) * D + 16 * g;
        const f16* nv = ap.new_v + (int64_t(b) * hkv + h) * D + n * (D / 16);
#pragma unroll
        for (int i = 0; i < kKL; ++i) {
          xk[2 * i] = as_h8(ld16(nk + 64 * i));
          xk[2 * i + 1] = as_h8(ld16(nk + 64 * i + 8));
        }
#pragma unroll
        for (int j = 0; j < kVW; ++j) xv[j] = *reinterpret_cast<const f16x4*>(nv + 4 * j);
      }
    }

    float m = kNegBig, l = 0.f;
    f32x4 acc[kT];
#pragma unroll
    for (int i = 0; i < kT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // id of page p of this window or the next one
    auto page_id = [&](int p) { return __builtin_amdgcn_readlane((p >> 6) == win ? ids0 : ids1, p & 63); };
    auto page_scale = [&](float x, int p) {  // (of this window)
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), p & 63));
    };
    auto issue_page = [&](int p, F8Page<D>& r) __attribute__((always_inline)) {
      const int raw = page_id(p), id = in_pool(raw) ? raw : 0;
      const uint8_t* kb = cache.codes + f8_block<D>(id, hkv, h);
      const uint8_t* vb = kb + v_codes;
      f8_load_page<D, true>(kb + k_lane, vb + v_lane, r);
    };
    const int last = np - 1;

    // The step's token into the row's last page, in registers: new scales, codes, and the stores.
    auto append = [&](F8Page<D>& r, float& ks, float& vs, int id) __attribute__((always_inline)) {
      const int off = (len - 1) % kF8Page;
      float ka = 0.f, va = 0.f;
#pragma unroll
      for (int j = 0; j < kVW; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) va = fmaxf(va, fabsf(float(xv[j][c])));
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
        const uint32_t c = f8_pack(float(xv[j][0]) * vi, float(xv[j][1]) * vi, float(xv[j][2]) * vi, float(xv[j][3]) * vi);
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

    float ksc = 0.f, vsc = 0.f;
    // Page p of the piece.  tail: its last page, which may end inside, and where the step's token may belong.
    auto consume = [&](int p, F8Page<D>& r, auto tail_t) __attribute__((always_inline)) {
      constexpr bool tail = decltype(tail_t)::value;
      const int id = __builtin_amdgcn_readlane(ids0, p & 63);
      const int left = !in_pool(id) ? 0 : tail ? len - (a + p) * kF8Page : kF8Page;  // tokens of the page that are attended
      float ks = page_scale(ksc, p), vs = page_scale(vsc, p);
      if constexpr (kAppend && tail) {
        if (appends && in_pool(id)) append(r, ks, vs, id);
      }
      f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kKL; ++c) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          s = mfma16(f8_frag(r.k[c][2 * half], r.k[c][2 * half + 1], ks, ks), qf[2 * c + half], s);
        }
      }
      // scores in base 2; tokens past the row's end, and of pages outside the pool, have none
      float sv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) sv[j] = s[j] * scale_log2;
      if (left < kF8Page) {  // (uniform)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = 4 * g + j < left;
          sv[j] = in ? sv[j] : -INFINITY;
#pragma unroll
          for (int c = 0; c < kVW; ++c) r.v[j][c] = in ? r.v[j][c] : 0u;  // (their codes may be anything, and 0 x NaN is NaN)
        }
      }
      const float mx = max_lane32(swap_max16(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]))));
      if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
        const float mn = fmaxf(m, mx);
        const float al = exp2_fast(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[t][j] *= al;
      }
      float pr[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) pr[j] = exp2_fast(sv[j] - m);
      const float l0 = (pr[0] + pr[1]) + (pr[2] + pr[3]);
      l += l0;
      if constexpr (kWeights) {
        const float lw = __builtin_amdgcn_logf(swap_sum(l0)) + m;
        if (g == 0 && n < G) my_lse[(p & 63) * G + n] = lw;
      }
      const f16x4 pf = f16x4{f16(pr[0]), f16(pr[1]), f16(pr[2]), f16(pr[3])};
#pragma unroll
      for (int c = 0; c < kVW; ++c) {
        uint32_t tr[4];
        f8_transpose(r, c, tr);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f16x2 h0 = f8_to_f16<false>(tr[j], vs), h1 = f8_to_f16<true>(tr[j], vs);
          acc[4 * c + j] = mfma16(f16x4{h0[0], h0[1], h1[0], h1[1]}, pf, acc[4 * c + j]);
        }
      }
    };
    // The page sums of a window go out together: whole lines, where a page's own are 4 G bytes (128 rows of 1023-8190
    // keys, 32 / 8 heads: 249 us with a store for every four pages, 223 so, 213 without weights).
    auto flush_lse = [&](int p0, int count) __attribute__((always_inline)) {
      float* dst = ws.lse + ((int64_t(b) * hkv + h) * max_pages + a + p0) * G;
      for (int x = lane; x < count * G; x += kWave) st_dev(dst + x, my_lse[x]);
    };

    // Ring of S pages: page p + S - 1 is requested while page p is attended.  Past the piece's end the last page is
    // requested again, so that the loads in flight are a fixed number and no wait is for more than one page.
    F8Page<D> r[S], rt;
    const std::integral_constant<bool, false> mid{};
    const std::integral_constant<bool, true> end{};
    settle(ids0, ids1);
    ksc = load_scale(ids0, 0);
    vsc = load_scale(ids0, v_scales);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < S - 1; ++x) issue_page(min(x, last), r[x]);
    __builtin_amdgcn_sched_barrier(0);
    settle(ksc, vsc);
    int p = 0;
    for (;; ++win) {  // one window of pages; the next one's scales and the one after's ids are on their way meanwhile
      float k_next = 0.f, v_next = 0.f;
      int id_next = 0;
      const bool more = (win + 1) * kWave <= last;
      if (more) {
        k_next = load_scale(ids1, 0);
        v_next = load_scale(ids1, v_scales);
        id_next = load_ids(win + 2);
      }
      const int stop = min(last, (win + 1) * kWave);
      for (; p + S <= stop; p += S) {
#pragma unroll
        for (int x = 0; x < S; ++x) {
          issue_page(min(p + x + S - 1, last), r[(x + S - 1) % S]);
          __builtin_amdgcn_sched_barrier(0);
          consume(p + x, r[x], mid);
        }
      }
      if (!more) break;
      if constexpr (kWeights) flush_lse(win * kWave, kWave);
      ids0 = ids1;
      ids1 = id_next;
      ksc = k_next;
      vsc = v_next;
      settle(ids0, ids1);
      settle(ksc, vsc);
    }
#pragma unroll
    for (int x = 0; x < S; ++x) {
      if (p + x < last) {
        if (p + x + S - 1 <= last) issue_page(p + x + S - 1, r[(x + S - 1) % S]);
        __builtin_amdgcn_sched_barrier(0);
        consume(p + x, r[x], mid);
      } else if (p + x == last) {
        rt = r[x];
      }
    }
    consume(last, rt, end);
    if constexpr (kWeights) flush_lse(win * kWave, np - win * kWave);

    const int first = range_of(cb), nranges = range_of(cb + npages - 1) - first + 1;
    l = swap_sum(l);
    if (nranges == 1) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (n < G) {
        f16* op = out + (int64_t(b) * hq + h * G + n) * D + 4 * g * (D / 16);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int c = 0; c < kVW; ++c)
            *reinterpret_cast<f16x4*>(op + x * (D / 16) + 4 * c) =
                f16x4{f16(acc[4 * c][x] * inv), f16(acc[4 * c + 1][x] * inv), f16(acc[4 * c + 2][x] * inv),
                      f16(acc[4 * c + 3][x] * inv)};
      }
      if constexpr (kWeights) {
        wait_all_mem();  // (this wave's own lse stores)
        const float tot = l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
        add_weights(b, [&](int x) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, tot), x)); },
                    npages, lane, kWave);
      }
    } else {
      const int en = 2 * wv + npend;
      if (n < G) {
        if (g == 0) {
          s_m[en][n] = m;
          s_l[en][n] = l;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int c = 0; c < kVW; ++c)
            s_o[en * units + (x * kVW + c) * 4 * G + g * G + n] = f32x4{acc[4 * c][x], acc[4 * c + 1][x], acc[4 * c + 2][x], acc[4 * c + 3][x]};
      }
      if (lane == 0) {
        s_row[en] = b;
        s_span[en] = (first / kWaves) << 16 | (first + nranges - 1) / kWaves;
      }
      ++npend;
    }
  }

  // The workgroup's states, in range order: those of one row are merged; a row that only this workgroup holds is
  // done, the others' states (the first and the last row's, at most) are published.
  if constexpr (kWeights) wait_all_mem();
  __syncthreads();
  const int tid = threadIdx.x;
  auto write_unit = [&](int b, int u, f32x4 o, float inv) {
    const int cl = u % (4 * G), un = cl % G, ug = cl / G, i4 = u / (4 * G);
    *reinterpret_cast<f16x4*>(out + (int64_t(b) * hq + h * G + un) * D + (4 * ug + i4 / kVW) * (D / 16) + 4 * (i4 % kVW)) =
        f16x4{f16(o[0] * inv), f16(o[1] * inv), f16(o[2] * inv), f16(o[3] * inv)};
  };
  auto row_weights = [&](int b) {  // s_tot holds the row's totals
    __syncthreads();
    add_weights(b, [&](int x) { return s_tot[x]; }, s_cum[b + 1] - s_cum[b] - kRowStart, tid, kWaves * kWave);
    __syncthreads();
  };
  int open = 0, open_b[2] = {0, 0}, open_wg[2] = {0, 0}, open_np[2] = {0, 0};
  const int e_row = s_row[lane % kEnt], e_span = s_span[lane % kEnt];  // lane e: state e's
  uint32_t todo = uint32_t(__builtin_amdgcn_ballot_w64(lane < kEnt && e_row >= 0));
  while (todo != 0) {
    const int e0 = __builtin_ctz(todo);
    const int b = __builtin_amdgcn_readlane(e_row, e0), span = __builtin_amdgcn_readlane(e_span, e0);
    const uint32_t of_row = uint32_t(__builtin_amdgcn_ballot_w64(lane < kEnt && e_row == b));
    todo &= ~of_row;
    const int wg0 = span >> 16, wg1 = span & 0xffff;
    const bool whole = wg0 == wg1;
    for (int u = tid; u < units; u += kWaves * kWave) {
      const int un = u % (4 * G) % G;
      float em[kEnt], el[kEnt], M = kNegBig, L = 0.f;
      f32x4 eo[kEnt], o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kEnt; ++x) {
        if ((of_row >> x) & 1u) {
          em[x] = s_m[x][un];
          el[x] = s_l[x][un];
          eo[x] = s_o[x * units + u];
        }
      }
#pragma unroll
      for (int x = 0; x < kEnt; ++x)
        if ((of_row >> x) & 1u) M = fmaxf(M, em[x]);
#pragma unroll
      for (int x = 0; x < kEnt; ++x) {
        if ((of_row >> x) & 1u) {
          const float w = exp2_fast(em[x] - M);
          L = fmaf(w, el[x], L);
          o = f32x4{fmaf(w, eo[x][0], o[0]), fmaf(w, eo[x][1], o[1]), fmaf(w, eo[x][2], o[2]), fmaf(w, eo[x][3], o[3])};
        }
      }
      if (whole) {
        write_unit(b, u, o, L > 0.f ? 1.f / L : 0.f);
        if (kWeights && u < G) s_tot[u] = L > 0.f ? M + __builtin_amdgcn_logf(L) : INFINITY;
      } else {
        const uint32_t slot = uint32_t((int64_t(b) + wg) * hkv + h);
        st_dev4(r_o, (slot * G * D + u * 4) * 4, o);
        if (u < G) st_dev2(r_ml, (slot * G + u) * 8, f32x2{M, L});
      }
    }
    if (whole) {
      if constexpr (kWeights) row_weights(b);
    } else {
      open_b[open & 1] = b;
      open_wg[open & 1] = wg0;
      open_np[open & 1] = wg1 - wg0 + 1;
      ++open;
    }
  }
  if (open == 0) return;
  wait_all_mem();
  __syncthreads();
  if (tid < open)
    s_ticket[tid] = __hip_atomic_fetch_add(ws.count + int64_t(tid == 0 ? open_b[0] : open_b[1]) * hkv + h, 1u,
                                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  compiler_fence();  // the merge loads below stay behind the tickets
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x >= open || s_ticket[x] != uint32_t(open_np[x] - 1)) continue;
    const int b = open_b[x];
    const int64_t slot0 = (int64_t(b) + open_wg[x]) * hkv + h;  // state j: slot0 + j hkv
    for (int u = tid; u < units; u += kWaves * kWave) {
      float M, L;
      f32x4 o;
      f8_merge(r_ml, r_o, slot0, hkv, open_np[x], G, D, u % (4 * G) % G, u, M, L, o);
      write_unit(b, u, o, L > 0.f ? 1.f / L : 0.f);
      if (kWeights && u < G) s_tot[u] = L > 0.f ? M + __builtin_amdgcn_logf(L) : INFINITY;
    }
    if constexpr (kWeights) row_weights(b);
    if (tid == 0) reset_ticket(ws.count + int64_t(b) * hkv + h);
  }
}

// Streams of a call, whole workgroups of them: as many waves as the card holds at once, over all kv heads (64 rows of
// 500-4000 keys x 256 dims, 2 kv heads: 37.8 us, 51.6 with twice as many), and no more than the longest call of these
// sizes has ranges.
constexpr int kSimdsPerCu = 4;
static int64_t f8_streams(int64_t batch, int32_t hkv, int32_t d, int32_t max_len, int cus) {
  const int64_t most = ceil_div(ceil_div(batch * (ceil_div(max_len, kF8Page) + kRowStart), kMinPages), kDecWaves);
  const int64_t wgs = int64_t(cus) * kSimdsPerCu * f8_per_simd(d) / kDecWaves / hkv;
  return kDecWaves * std::max<int64_t>(1, std::min(most, wgs));
}
static size_t f8_ws_layout(int64_t batch, int64_t wgs, int32_t hkv, int32_t G, int32_t d, int32_t max_pages,
                           bool weights, size_t* off_ml, size_t* off_o, size_t* off_lse) {
  const size_t slots = size_t(batch + wgs) * hkv * G;
  size_t off = kTicketBytes;
  *off_ml = off;
  off = align256(off + slots * 2 * sizeof(float));
  *off_o = off;
  off = align256(off + slots * d * sizeof(float));
  *off_lse = off;
  if (weights) off = align256(off + size_t(batch) * hkv * max_pages * G * sizeof(float));
  return off;
}

// LDS of a workgroup beside the kernel's own variables (under 2 KB): its states, the rows' offsets, its page sums.
static size_t f8_lds(int64_t batch, int32_t G, int32_t d, bool weights) {
  return size_t(2 * kDecWaves) * G * d * sizeof(float) + size_t(batch + 1) * sizeof(int) +
         (weights ? size_t(kDecWaves) * kWave * G * sizeof(float) : 0);
}
constexpr size_t kF8MaxLds = (160 - 2) << 10;

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
      int64_t(batch) * (max_pages + kRowStart) > (int64_t(1) << 30) || num_pages > (int64_t(1) << 31) / kF8Page ||
      f8_lds(batch, G, d, page_weights != nullptr) > kF8MaxLds)
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
  const int64_t streams = f8_streams(batch, hkv, d, cap, std::max(1, cus));
  size_t off_ml, off_o, off_lse;
  if (workspace_bytes < f8_ws_layout(batch, streams / kDecWaves, hkv, G, d, max_pages, page_weights != nullptr, &off_ml, &off_o,
                                     &off_lse))
    return IFN_ERR_WORKSPACE;
  if (cus < 1) return IFN_ERR_HIP;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const F8Workspace ws{reinterpret_cast<uint32_t*>(w), reinterpret_cast<float*>(w + off_ml),
                       reinterpret_cast<float*>(w + off_o), reinterpret_cast<float*>(w + off_lse)};
  const F8Cache cache{static_cast<uint8_t*>(codes), scales, num_pages};
  const F8Append ap{static_cast<const f16*>(new_k), static_cast<const f16*>(new_v)};
  const float sl = (scale > 0.f ? scale : 1.f / sqrtf(float(d))) * kLog2e;
  const int64_t blocks = streams / kDecWaves * hkv;
  const size_t lds = f8_lds(batch, G, d, page_weights != nullptr);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto k) {
    k<<<dim3(unsigned(blocks)), dim3(kDecThreads), lds, s>>>(
        seq_lens, active, batch, max_pages, cap, hkv, G, int32_t(streams), block_tables,
        static_cast<const f16*>(query), cache, static_cast<f16*>(out), sl, ws, ap, page_weights);
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
  const int64_t wgs = f8_streams(batch, num_kv_heads, head_dim, int32_t(cap), std::max(1, device_cu_count())) / kDecWaves;
  size_t a, b, c;
  return f8_ws_layout(batch, wgs, num_kv_heads, num_q_heads / num_kv_heads, head_dim, max_pages_per_seq,
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
