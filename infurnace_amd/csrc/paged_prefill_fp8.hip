// Causal chunked-prefill paged attention over the 8-bit KV cache (gfx950 MFMA fp16).
//
// The 8-bit form of the reference's documented paged_attention with a multi-token query
// (docs/architecture.md:246; contiguous semantics src/infurnace/executor/tinygrad/model.py:116-132): query row
// i sits at query_start + i and sees keys [0, query_start + i].  Blocks and scales: kv_fp8.hpp.
//
// The (query, head) pairs of one kv head are the columns of the products, column c = query c / G, head c % G
// of the group, so any group size fills the matrix instructions.  A workgroup serves 32 columns (two tiles of 16); its
// four waves are key groups that take 32-key tiles (two pages) in turn and merge through LDS at the end.  Calls with
// few columns split the keys over workgroups too.  S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_f16: lane
// (n = lane % 16, g = lane / 16) has the scores of column n and tokens 4 g .. 4 g + 3 of both pages, which are the
// second product's B operand as they are (its k order is free).  Codes go from memory to the matrix cores in
// registers, as in paged_decode_fp8.hip: K as loaded, V after a byte transpose.  Every 32 columns read and convert a
// tile again, so calls that fill the chip in workgroups of 128 columns go to paged_prefill_fp8_block.hip.
//
// What bounds it: vector work (42% of the waves' time) and waits for loads (33%; 8 KB a tile of 32 x 32, the data path
// of the L1 76% busy), about 0.9 us a tile and SIMD whether it has one wave or two.  512 queries at 1024, 16 / 8 heads
// x 128 (5.4 GFLOP): 15.9 us, of which 3 before the first tile and 2 to merge; 16 queries at 4096: 13.3 us.
#include <algorithm>

#include "kv_fp8.hpp"

namespace ifn {

constexpr int kPfTiles = 2;             // column tiles of a workgroup
constexpr int kPfWaves = 4;             // waves (key groups) of a workgroup
constexpr int kPfThreads = kPfWaves * kWave;
constexpr int kPfMaxSplit = 8;
constexpr int kPfCols = 16 * kPfTiles;

template <int D>
__global__ __launch_bounds__(kPfThreads, 2) void prefill_fp8_kernel(
    const int32_t* __restrict__ table, const f16* __restrict__ q, int64_t num_pages, int32_t query_start, int32_t T,
    int32_t hkv, int32_t G, int32_t n_blocks, int32_t nsplit,  // (up to here in registers at dispatch: build.py)
    const float* __restrict__ scales, const uint8_t* __restrict__ codes, f16* __restrict__ out, float scale_log2,
    PrefillWorkspace ws) {
  constexpr int kKL = F8Page<D>::kKL, kVW = F8Page<D>::kVW;
  constexpr int kT = D / 16, NC = kPfTiles, KW = kPfWaves;
  __shared__ f32x4 s_o[KW][NC * kT][kWave];
  __shared__ float s_ml[2][KW][kPfCols];
  __shared__ uint32_t s_ticket;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = lane % 16, g = lane / 16;
  // kv head, then key split, then column block, the longest key ranges first
  const int h = int(blockIdx.x) % hkv, rest = int(blockIdx.x) / hkv;
  const int split = rest % nsplit, blk = n_blocks - 1 - rest / nsplit;
  const int hq = hkv * G;
  const uint32_t c0 = uint32_t(blk) * kPfCols, cols = uint32_t(T) * G;  // (the host: rows below 2^31)
  const int keys = query_start + int(min(c0 + kPfCols - 1, cols - 1) / uint32_t(G)) + 1;  // keys some column sees
  const int first_pos = query_start + int(c0 / uint32_t(G));        // every column sees keys up to this one
  const int pages = (keys + kF8Page - 1) / kF8Page, tiles = (pages + 1) / 2;
  const int stride = KW * nsplit, lead = KW * split + wave;
  const int mine = (tiles - lead + stride - 1) / stride, last = mine - 1;  // this wave's tiles: lead + stride i

  // Page ids and scales of the wave's tiles, 32 tiles per window, one page per lane.
  const int64_t v_codes = num_pages * hkv * (kF8Page * D), v_scales = num_pages * hkv;
  auto load_ids = [&](int w) {
    const int pg = 2 * (lead + stride * (32 * w + lane / 2)) + lane % 2;
    const int id = table[min(pg, pages - 1)];
    return pg < pages && id >= 0 && int64_t(id) < num_pages ? id : -1;
  };
  auto load_scale = [&](int id, int64_t kv) { return scales[kv + int64_t(max(id, 0)) * hkv + h]; };
  int win = 0, ids = load_ids(0), ids1 = load_ids(1);

  int my_pos[NC];
  uint32_t my_row[NC];  // (query, head) row of the lane's column of each tile
  f16x8 qf[NC][2 * kKL];
#pragma unroll
  for (int x = 0; x < NC; ++x) {
    const uint32_t c = min(c0 + 16 * x + n, cols - 1), t = c / uint32_t(G);
    my_pos[x] = query_start + int(t);
    my_row[x] = t * hq + h * G + (c - t * G);
    const f16* qp = q + int64_t(my_row[x]) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < kKL; ++i) {
      qf[x][2 * i] = as_h8(ld16(qp + 64 * i));
      qf[x][2 * i + 1] = as_h8(ld16(qp + 64 * i + 8));
    }
  }
  float m[NC], l[NC], ksc = 0.f, vsc = 0.f;
  f32x4 acc[NC][kT];
#pragma unroll
  for (int x = 0; x < NC; ++x) {
    m[x] = kNegBig;
    l[x] = 0.f;
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint32_t k_lane = n * D + 16 * g, v_lane = 4 * g * D + n * (D / 16);
  auto issue = [&](int i, F8Page<D> (&r)[2]) __attribute__((always_inline)) {  // tile i of the wave's, of this window or the next
    const int src = (i >> 5) == win ? ids : ids1;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint8_t* b = codes + f8_block<D>(max(__builtin_amdgcn_readlane(src, ((2 * i) & 63) + y), 0), hkv, h);
      f8_load_page<D, false>(b + k_lane, b + v_codes + v_lane, r[y]);
    }
  };
  auto consume = [&](int i, F8Page<D> (&r)[2]) __attribute__((always_inline)) {
    const int at = (2 * i) & 63;
    const int key0 = 32 * (lead + stride * i);
    auto get = [&](float v, int y) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at + y)); };
    const bool live[2] = {__builtin_amdgcn_readlane(ids, at) >= 0, __builtin_amdgcn_readlane(ids, at + 1) >= 0};
    const float vs0 = get(vsc, 0), vs1 = get(vsc, 1);
    f32x4 s[NC][2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const float ks = get(ksc, y);
#pragma unroll
      for (int x = 0; x < NC; ++x) s[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kKL; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f16x8 kf = f8_frag(r[y].k[c][2 * half], r[y].k[c][2 * half + 1], ks, ks);
#pragma unroll
          for (int x = 0; x < NC; ++x) s[x][y] = mfma16(kf, qf[x][2 * c + half], s[x][y]);
        }
    }
    if (key0 + 31 > first_pos || !live[0] || !live[1]) {  // (uniform)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int x = 0; x < NC; ++x) {
          const int lim = live[y] ? my_pos[x] - key0 - 16 * y - 4 * g : -1;
#pragma unroll
          for (int j = 0; j < 4; ++j) s[x][y][j] = f8_masked(j <= lim, s[x][y][j]);
        }
        const int end = live[y] ? keys - key0 - 16 * y - 4 * g : 0;  // (rows nobody stored may hold NaN, and 0 x NaN is NaN)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < kVW; ++c) r[y].v[j][c] = j < end ? r[y].v[j][c] : 0u;
      }
    }
    f16x8 pf[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      float mx = fmaxf(fmaxf(fmaxf(s[x][0][0], s[x][0][1]), fmaxf(s[x][0][2], s[x][0][3])),
                       fmaxf(fmaxf(s[x][1][0], s[x][1][1]), fmaxf(s[x][1][2], s[x][1][3])));
      mx = max_lane32(swap_max16(mx)) * scale_log2;
      // (the reference maximum moves only when a score exceeds it by more than 8 in log2 units, so P < 2^8)
      if (__builtin_amdgcn_ballot_w64(mx > m[x] + 8.f) != 0) {
        const float mn = fmaxf(m[x], mx);
        const float al = exp2_fast(m[x] - mn);
        m[x] = mn;
        l[x] *= al;
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[x][t][j] *= al;
      }
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = exp2_fast(fmaf(s[x][j / 4][j % 4], scale_log2, -m[x]));
        sum += p;
        pf[x][j] = f16(p);
      }
      l[x] += sum;
    }
#pragma unroll
    for (int c = 0; c < kVW; ++c) {
      uint32_t tr0[4], tr1[4];
      f8_transpose(r[0], c, tr0);
      f8_transpose(r[1], c, tr1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f16x8 vf = f8_frag(tr0[j], tr1[j], vs0, vs1);
#pragma unroll
        for (int x = 0; x < NC; ++x) acc[x][4 * c + j] = mfma16(vf, pf[x], acc[x][4 * c + j]);
      }
    }
  };

  // Two tiles in registers: tile i + 1 is requested while tile i is attended (past the last one it again, so that no
  // wait is for more than one tile).
  if (mine > 0) {
    F8Page<D> r0[2], r1[2];
    settle(ids, ids1);
    ksc = load_scale(ids, 0);
    vsc = load_scale(ids, v_scales);
    __builtin_amdgcn_sched_barrier(0);
    issue(0, r0);
    __builtin_amdgcn_sched_barrier(0);
    settle(ksc, vsc);
    int i = 0;
    for (;; ++win) {
      const bool more = 32 * (win + 1) <= last;
      float k_next = 0.f, v_next = 0.f;
      int id_next = 0;
      if (more) {
        k_next = load_scale(ids1, 0);
        v_next = load_scale(ids1, v_scales);
        id_next = load_ids(win + 2);
      }
      const int stop = min(last, 32 * (win + 1));
      for (; i + 2 <= stop; i += 2) {
        issue(i + 1, r1);
        __builtin_amdgcn_sched_barrier(0);
        consume(i, r0);
        issue(min(i + 2, last), r0);
        __builtin_amdgcn_sched_barrier(0);
        consume(i + 1, r1);
      }
      if (!more) break;
      ids = ids1;
      ids1 = id_next;
      ksc = k_next;
      vsc = v_next;
      settle(ids, ids1);
      settle(ksc, vsc);
    }
    if (i < last) {
      issue(last, r1);
      __builtin_amdgcn_sched_barrier(0);
      consume(i, r0);
      consume(last, r1);
    } else {
      consume(last, r0);
    }
  }

  // The waves' states of each column: maxima and sums first, then the outputs in a common scale through LDS, each wave
  // adding up its share of the 4-dim units (unit x kT + r kVW + c of a lane: column 16 x + n, dims (4 g + r) D / 16 +
  // 4 c ..).  With the keys split over workgroups too, these states go to the workspace, and the workgroup that
  // arrives last merges them in split order.
  float al[NC], Ms[NC], Ls[NC];
#pragma unroll
  for (int x = 0; x < NC; ++x) {
    l[x] = swap_sum(l[x]);
    if (g == 0) {
      s_ml[0][wave][16 * x + n] = m[x];
      s_ml[1][wave][16 * x + n] = l[x];
    }
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NC; ++x) {
    Ms[x] = kNegBig;
    Ls[x] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) Ms[x] = fmaxf(Ms[x], s_ml[0][w][16 * x + n]);
#pragma unroll
    for (int w = 0; w < KW; ++w) Ls[x] += s_ml[1][w][16 * x + n] * exp2_fast(s_ml[0][w][16 * x + n] - Ms[x]);
    al[x] = exp2_fast(m[x] - Ms[x]);
  }
#pragma unroll
  for (int x = 0; x < NC; ++x)
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int r = t / kVW, c = t % kVW;
      s_o[wave][x * kT + t][lane] = f32x4{acc[x][4 * c][r] * al[x], acc[x][4 * c + 1][r] * al[x],
                                          acc[x][4 * c + 2][r] * al[x], acc[x][4 * c + 3][r] * al[x]};
    }
  __syncthreads();
  auto write = [&](int u, f32x4 o, float L) {
    const int x = u / kT, r = u % kT / kVW, c = u % kVW;
    const float k = L > 0.f ? 1.f / L : 0.f;
    const int64_t row = x == 0 ? my_row[0] : my_row[1];
    if (c0 + 16 * x + n < cols)
      *reinterpret_cast<f16x4*>(out + row * D + (4 * g + r) * (D / 16) + 4 * c) =
          f16x4{f16(o[0] * k), f16(o[1] * k), f16(o[2] * k), f16(o[3] * k)};
  };
  constexpr int kUnits = NC * kT;  // of a lane
  const int64_t seg = int64_t(blk) * hkv + h;
  // (a split call has at most 2 workgroups a CU, so its offsets fit 32 bits)
  const __amdgpu_buffer_rsrc_t r_ml = make_rsrc(ws.ml, uint32_t(n_blocks) * hkv * nsplit * kPfCols * 8u);
  const __amdgpu_buffer_rsrc_t r_o = make_rsrc(ws.o, uint32_t(n_blocks) * hkv * nsplit * kUnits * kWave * 16u);
  const uint32_t state0 = uint32_t(seg) * nsplit;
#pragma unroll
  for (int v = 0; v < kUnits / KW; ++v) {
    const int u = wave + KW * v;
    f32x4 o = s_o[0][u][lane];
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      const f32x4 y = s_o[w][u][lane];
      o = f32x4{o[0] + y[0], o[1] + y[1], o[2] + y[2], o[3] + y[3]};
    }
    if (nsplit == 1) write(u, o, u / kT == 0 ? Ls[0] : Ls[1]);
    else st_dev4(r_o, (((state0 + split) * kUnits + u) * kWave + lane) * 16, o);
  }
  if (nsplit == 1) return;
  if (wave == 0 && g == 0) {
#pragma unroll
    for (int x = 0; x < NC; ++x) st_dev2(r_ml, ((state0 + split) * kPfCols + 16 * x + n) * 8, f32x2{Ms[x], Ls[x]});
  }
  if (!arrive_last(ws.count + seg, uint32_t(nsplit - 1), &s_ticket)) return;
  float L[NC];
  f32x4 o[kUnits / KW];
#pragma unroll
  for (int x = 0; x < NC; ++x) {
    Ms[x] = kNegBig;
    L[x] = 0.f;
  }
#pragma unroll
  for (int v = 0; v < kUnits / KW; ++v) o[v] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kB = 4;  // states a round trip
  for (int s0 = 0; s0 < nsplit; s0 += kB) {
    f32x2 ml[kB][NC];
    f32x4 y[kB][kUnits / KW];
#pragma unroll
    for (int s = 0; s < kB; ++s) {
      const uint32_t st = state0 + min(s0 + s, nsplit - 1);
#pragma unroll
      for (int x = 0; x < NC; ++x) ml[s][x] = ld_dev2(r_ml, (st * kPfCols + 16 * x + n) * 8);
#pragma unroll
      for (int v = 0; v < kUnits / KW; ++v) y[s][v] = ld_dev4(r_o, ((st * kUnits + wave + KW * v) * kWave + lane) * 16);
    }
    __builtin_amdgcn_sched_barrier(0);
    float w[kB][NC], keep[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      float mn = Ms[x];
#pragma unroll
      for (int s = 0; s < kB; ++s)
        if (s0 + s < nsplit) mn = fmaxf(mn, ml[s][x][0]);
      keep[x] = exp2_fast(Ms[x] - mn);
      Ms[x] = mn;
      L[x] *= keep[x];
#pragma unroll
      for (int s = 0; s < kB; ++s) {
        w[s][x] = s0 + s < nsplit ? exp2_fast(ml[s][x][0] - mn) : 0.f;
        L[x] = fmaf(w[s][x], ml[s][x][1], L[x]);
      }
    }
#pragma unroll
    for (int v = 0; v < kUnits / KW; ++v) {
      const int x = (KW * v) / kT;  // (a wave's units u = wave + KW v: the same column tile for every wave)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[v][j] *= keep[x];
#pragma unroll
        for (int s = 0; s < kB; ++s) o[v][j] = fmaf(w[s][x], y[s][v][j], o[v][j]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < kUnits / KW; ++v) write(wave + KW * v, o[v], L[(KW * v) / kT]);
  if (threadIdx.x == 0) reset_ticket(ws.count + seg);
}

// How a call is made.  groups: 128-column workgroups (paged_prefill_fp8_block.hip) on one or two key groups; 0: this
// file's, the keys of a block split over nsplit workgroups.
struct PfPlan {
  int groups, nsplit;
};
// By n, the 128-column workgroups, and the keys a column sees on average (us: 32 columns / one / two key groups of 128
// columns; 8 kv heads, 256 CUs):
//  * n > CUs, 128 dims: one group, two workgroups a CU (32 q heads, 1536 queries at 1024, n = 384: 75.7 / 65.4 / 73.4;
//    2048 at 4096, n = 512: 244 / 177 / 194), or two where the chip is not full twice and a chunk's own keys make the
//    blocks uneven and long (16 q heads, 3000 at 0, n = 376: 67.1 / 69.0 / 59.9; but 32, 1536 at 0: 42.3 / 40.3 / 44.7).
//  * CUs / 2 < n <= CUs, 128 dims: two groups once there is enough to do (32 q heads, 1024 at 1024, n = 256: 48.3 /
//    46.0 / 43.8, at 0: 26.4 / 26.8 / 28.1; 768 at 4096, n = 192: 89.2 / 95.5 / 81.0, at 1024: 36.4 / 39.7 / 37.9).
//  * less: 32 columns (512 at 4096, n = 128: 62.3 / 90.2 / 75.9).
//  * 64 dims: one group for large calls (32 q heads, 2048 at 1024, n = 512: 66.4 / 58.3 / 66.3, at 0: 39.0 / 40.4 /
//    44.3), else 32 columns.
//  * 32 columns, fewer workgroups than CUs: the keys split over up to eight more of them, as long as a workgroup has
//    about 12 tiles (16 queries at 4096, 16 q heads: 32.9 us with one, 21.6, 15.5, 13.3 with 2, 4, 8, 13.5 with 16; at
//    1500 10.7 with 4, 10.8 with 6; at 512 10.1 with one, 10.5 with two).  Two workgroups a CU gain nothing (64
//    queries, 32 q heads, at 4096: 17.0 with 4, 21.2 with 6).
static PfPlan pf_plan(int64_t T, int64_t start, int32_t hq, int32_t hkv, int32_t d, int64_t cus) {
  const int64_t cols = T * (hq / hkv), n = ceil_div(cols, 128) * hkv;
  const int64_t load = n * (start + T / 2);  // workgroups x average keys
  if (d == 128) {
    if (n > cus) return {n >= 2 * cus || start >= T / 2 || start + T < 2048 ? 1 : 2, 1};
    if (2 * n > cus && load >= 1500 * cus) return {2, 1};
  } else if (n > cus && load >= 4000 * cus) {
    return {1, 1};
  }
  const int64_t wgs = ceil_div(cols, kPfCols) * hkv, tiles = ceil_div(start + T, 2 * kF8Page);
  const int64_t most = std::min<int64_t>({cus / wgs, (tiles + 1) / 12, kPfMaxSplit});
  return {0, int(std::max<int64_t>(1, most))};
}
static size_t pf_ws_layout(int64_t wgs, int nsplit, int32_t d, size_t* off_ml, size_t* off_o) {
  size_t off = kTicketBytes;
  *off_ml = off;
  if (nsplit > 1) off = align256(off + size_t(wgs) * nsplit * kPfCols * 8);
  *off_o = off;
  if (nsplit > 1) off = align256(off + size_t(wgs) * nsplit * kPfCols * d * 4);
  return off;
}

}  // namespace ifn

extern "C" size_t ifn_paged_prefill_fp8_workspace_bytes(int32_t num_q_tokens, int32_t query_start,
                                                        int32_t num_q_heads, int32_t num_kv_heads,
                                                        int32_t head_dim, int32_t block_size) {
  using namespace ifn;
  if (num_q_tokens < 0 || query_start < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads != 0 ||
      head_dim < 1 || block_size < 1)
    return 0;
  if (num_q_tokens == 0) return kTicketBytes;
  const PfPlan p = pf_plan(num_q_tokens, query_start, num_q_heads, num_kv_heads, head_dim, std::max(1, device_cu_count()));
  size_t a, b;
  return pf_ws_layout(ceil_div(int64_t(num_q_tokens) * (num_q_heads / num_kv_heads), kPfCols) * num_kv_heads, p.nsplit,
                      head_dim, &a, &b);
}

extern "C" int ifn_paged_prefill_fp8(void* out, const void* query, const void* codes_layer,
                                     const float* scales_layer, int64_t num_pages, const int32_t* block_table,
                                     int32_t max_pages, int32_t query_start, int32_t num_q_tokens,
                                     int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, float scale, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  using namespace ifn;
  if (out == nullptr || query == nullptr || codes_layer == nullptr || scales_layer == nullptr || block_table == nullptr)
    return IFN_ERR_INVALID_ARGUMENT;
  if (num_pages < 1 || max_pages < 1 || query_start < 0 || num_q_tokens < 0 || num_q_heads < 1 || num_kv_heads < 1 ||
      num_q_heads % num_kv_heads != 0 || head_dim < 1 || block_size < 1)
    return IFN_ERR_INVALID_ARGUMENT;
  if (block_size != kF8Page || (head_dim != 64 && head_dim != 128)) return IFN_ERR_UNSUPPORTED;
  if (int64_t(query_start) + num_q_tokens > int64_t(max_pages) * kF8Page) return IFN_ERR_INVALID_ARGUMENT;
  if (int64_t(query_start) + num_q_tokens > (int64_t(1) << 31) - 64 || num_pages > (int64_t(1) << 31) / kF8Page ||
      int64_t(num_q_tokens) * num_q_heads > (int64_t(1) << 31) - 256)
    return IFN_ERR_UNSUPPORTED;
  IFN_CHECK_ALIGN16(out);
  IFN_CHECK_ALIGN16(query);
  IFN_CHECK_ALIGN16(codes_layer);
  if (num_q_tokens == 0) return IFN_OK;
  if (workspace == nullptr) return IFN_ERR_WORKSPACE;
  IFN_CHECK_ALIGN16(workspace);
  const int32_t G = num_q_heads / num_kv_heads;
  const int64_t n_blocks = ceil_div(int64_t(num_q_tokens) * G, kPfCols);
  const int cus = device_cu_count();
  const PfPlan plan = pf_plan(num_q_tokens, query_start, num_q_heads, num_kv_heads, head_dim, std::max(1, cus));
  size_t off_ml, off_o;
  if (workspace_bytes < pf_ws_layout(n_blocks * num_kv_heads, plan.nsplit, head_dim, &off_ml, &off_o))
    return IFN_ERR_WORKSPACE;
  if (n_blocks * num_kv_heads * plan.nsplit >= (int64_t(1) << 31)) return IFN_ERR_UNSUPPORTED;
  if (cus < 1) return IFN_ERR_HIP;
  const float sl = (scale > 0.f ? scale : 1.f / sqrtf(float(head_dim))) * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  f16* o = static_cast<f16*>(out);
  const f16* q = static_cast<const f16*>(query);
  const uint8_t* codes = static_cast<const uint8_t*>(codes_layer);
  if (plan.groups > 0)
    return prefill_fp8_block_launch(o, q, codes, scales_layer, num_pages, block_table, query_start, num_q_tokens,
                                    num_q_heads, num_kv_heads, head_dim, sl, plan.groups, s);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const PrefillWorkspace ws{reinterpret_cast<uint32_t*>(w), reinterpret_cast<float*>(w + off_ml),
                            reinterpret_cast<float*>(w + off_o)};
  auto k = head_dim == 64 ? prefill_fp8_kernel<64> : prefill_fp8_kernel<128>;
  k<<<dim3(unsigned(n_blocks * num_kv_heads * plan.nsplit)), dim3(kPfThreads), 0, s>>>(
      block_table, q, num_pages, query_start, num_q_tokens, num_kv_heads, G, int32_t(n_blocks), plan.nsplit,
      scales_layer, codes, o, sl, ws);
  return ifn_launch_status();
}
