// Causal chunked-prefill paged attention over the 8-bit KV cache for chunks that fill the chip (gfx950 MFMA fp16).
//
// Same operation as paged_prefill_fp8.hip (docs/architecture.md:246; contiguous semantics
// src/infurnace/executor/tinygrad/model.py:116-132), for calls with enough columns -- (query, head) pairs of a kv
// head -- for workgroups of 128.
//
//  * A workgroup of 4 waves serves 128 columns of one kv head, 32 a wave; two workgroups share a CU.  With too few
//    workgroups for that, a workgroup has two such key groups of 4 waves (KS = 2), which take alternate tiles and
//    merge through LDS at the end.
//  * All waves walk the same 64-key tiles.  Wave w brings page w of the tile: codes through registers, converted to
//    fp16 with the blocks' scales (exact), and written to LDS in the order of the matrix fragments, so that a
//    fragment is one 16-byte read a lane, consecutive lanes consecutive.  The conversion is paid once per 128
//    columns, and V's transpose once, on bytes (v_perm); K runs one tile ahead of V.
//  * S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_f16: a lane owns one column, its scores are the second
//    product's B operands as they are.  Rows past the sequence's end and pages outside the pool come as zeros (the
//    buffer descriptors' bounds), their scores are masked.
//
// What bounds it: the matrix cores and the vector work beside them, at the clock the power leaves.  2048 queries at 6144,
// 32 / 8 heads x 128 (240 GFLOP): 252 us, 955 TFLOP/s; a large fp16 product on the same card: 1200.
#include <algorithm>

#include "kv_fp8.hpp"

namespace ifn {

constexpr int kP8Tile = 64;                       // keys per tile
constexpr int kP8Pages = kP8Tile / kF8Page;
constexpr int kP8Waves = 4;
constexpr int kP8Threads = kP8Waves * kWave;
constexpr int kP8Cols = 32 * kP8Waves;            // columns of a workgroup
constexpr int kP8XcdCus = 32;                     // CUs per XCD, 8 XCDs

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void pin(f16x8& a, f16x8& b) {  // no instruction: the values must exist here
  asm volatile("" : "+v"(a), "+v"(b));
}
#else
__device__ __forceinline__ f32x16 mfma32(f16x8, f16x8, f32x16 c) { return c; }
__device__ __forceinline__ void pin(f16x8&, f16x8&) {}
#endif
// Workgroup barrier for LDS traffic alone: this wave's LDS writes are done, its loads may be in flight.
__device__ __forceinline__ void p8_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
template <int D, int KS>
__global__ __launch_bounds__(KS * kP8Threads, 2) void prefill_fp8_block_kernel(
    f16* __restrict__ out, const f16* __restrict__ q, const uint8_t* __restrict__ codes,
    const float* __restrict__ scales, int64_t num_pages, const int32_t* __restrict__ table, int32_t query_start,
    int32_t T, int32_t hkv, int32_t G, int32_t n_blocks, float scale_log2) {
  constexpr int kSteps = D / 16;          // MFMA steps over the head dims
  constexpr int kDT = D / 32;             // output tiles
  constexpr int kKC = D / 64;             // 16-byte chunks of a lane's K row
  constexpr int kVW = D / 64;             // words of a lane's V rows
  constexpr int kTileB = kP8Tile * D * 2; // bytes of K, and of V, of a tile
  constexpr int kBufB = 2 * kTileB;
  constexpr int kOwn = kDT / KS;          // output tiles a wave finishes
  constexpr int kMergeB = KS > 1 ? KS * kP8Threads * (16 * kOwn + 2) * 4 : 0;
  constexpr int kLds = 2 * KS * kBufB > kMergeB ? 2 * KS * kBufB : kMergeB;
  __shared__ __attribute__((aligned(16))) unsigned char smem[kLds];
  int bid = int(blockIdx.x);
  if constexpr (KS == 1) {
    // Two workgroups per CU, 32 apart on their XCD: every other round of the chip runs in reverse, so that long key
    // ranges meet short ones.
    const int per = 8 * kP8XcdCus, r = bid % per;
    if ((bid / per) % 2 == 1 && bid - r + per <= int(gridDim.x)) bid += 8 * (kP8XcdCus - 1 - 2 * (r / 8));
  }
  const int h = bid % hkv;                       // (8 kv heads: an XCD's L2 holds one)
  const int blk = n_blocks - 1 - bid / hkv;      // longest key ranges first
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wave = wv % kP8Waves, grp = wv / kP8Waves;
  const int col = lane % 32, half = lane / 32;
  const int hq = hkv * G;
  const uint32_t cols = uint32_t(T) * G, c0 = uint32_t(blk) * kP8Cols, wc0 = c0 + 32 * wave;  // (the host: below 2^31)
  const uint32_t my_c = min(wc0 + col, cols - 1), per_q = uint32_t(G);
  const int my_q = int(my_c / per_q), my_h = h * G + int(my_c % per_q);
  const int my_pos = query_start + my_q;
  const int total = query_start + T;
  const int n_tiles = int(ceil_div(query_start + int(min(c0 + kP8Cols - 1, cols - 1) / per_q) + 1, kP8Tile));
  const int wave_first = query_start + int(min(wc0, cols - 1) / per_q);
  const int wave_tiles = int(ceil_div(query_start + int(min(wc0 + 31, cols - 1) / per_q) + 1, kP8Tile));

  // Page ids and scales, 64 pages per window (16 tiles), one per lane, a window ahead.
  const int seq_pages = int(ceil_div(total, kF8Page));
  const int64_t v_codes = num_pages * hkv * (kF8Page * D), v_scales = num_pages * hkv;
  auto load_ids = [&](int w) __attribute__((always_inline)) {
    const int pg = 64 * w + lane;
    const int id = table[min(pg, seq_pages - 1)];
    return pg < seq_pages && id >= 0 && int64_t(id) < num_pages ? id : -1;
  };
  auto load_scale = [&](int id, int64_t kv) __attribute__((always_inline)) { return scales[kv + int64_t(max(id, 0)) * hkv + h]; };
  int win = 0, ids = load_ids(0), ids_next = load_ids(1);
  float ksc = load_scale(ids, 0), vsc = load_scale(ids, v_scales);
  float ksc_next = load_scale(ids_next, 0), vsc_next = load_scale(ids_next, v_scales);

  f16x8 qf[kSteps];  // this lane's column, step s: dims 16 s + 8 half .. + 7 (columns past the chunk: its last)
  {
    const f16* qp = q + (int64_t(my_q) * hq + my_h) * D + 8 * half;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = as_h8(ld16(qp + 16 * s));
  }

  // Staging: lane (x = lane % 16, y = lane / 16) holds dims 64 i + 16 y .. + 15 of K row x, and of V rows 4 y .. + 3
  // the dims x D / 16 ..  K dims 16 s + 8 f .. are fragment step s, half f; V's dim e of the lane's is row
  // 16 (e / kDT) + x of output tile e % kDT.
  const int x16 = lane % 16, y4 = lane / 16;
  const uint32_t k_off = x16 * D + 16 * y4, v_off = 4 * y4 * D + x16 * (D / 16);
  lds_u8* const lds = (lds_u8*)(smem) + grp * 2 * kBufB;
  const uint32_t k_wr = uint32_t((((wave / 2) * kSteps + y4) * 64 + 16 * (wave % 2) + x16) * 16);
  const uint32_t v_wr = uint32_t(kTileB + ((wave * kDT) * 64 + 32 * (y4 % 2) + x16) * 16 + 8 * (y4 / 2));
  u32x4 kst[kKC];
  uint32_t vst[4][kVW];
  struct Tile {
    int kt, fl;      // first key; page flags (bit p: page p is in the pool)
    int page, rows;  // this wave's page of the tile and its keys (0: none)
    float ks, vs;
  };
  auto tile_at = [&](int i) __attribute__((always_inline)) -> Tile {
    const int t = KS * i + grp;
    if ((t >> 4) != win) {  // (uniform)
      win = t >> 4;
      ids = ids_next;
      ksc = ksc_next;
      vsc = vsc_next;
      ids_next = load_ids(win + 1);
      ksc_next = load_scale(ids_next, 0);
      vsc_next = load_scale(ids_next, v_scales);
    }
    const int fl = int(__builtin_amdgcn_ballot_w64(ids >= 0) >> (4 * (t & 15))) & 15;
    const bool ok = ((fl >> wave) & 1) != 0;
    const int at = (kP8Pages * t + wave) & 63;
    auto get = [&](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at)); };
    return Tile{kP8Tile * t, fl, __builtin_amdgcn_readfirstlane(ok ? __builtin_amdgcn_readlane(ids, at) : 0),
                __builtin_amdgcn_readfirstlane(ok ? min(max(total - kP8Tile * t - kF8Page * wave, 0), kF8Page) : 0),
                get(ksc), get(vsc)};
  };
  auto block = [&](const Tile& t, int64_t kv) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes + kv + f8_block<D>(t.page, hkv, h)), 0,
                                             t.rows * D, 0x00020000);
  };
  auto load_k = [&](const Tile& t) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = block(t, 0);
#pragma unroll
    for (int i = 0; i < kKC; ++i) kst[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k_off + 64 * i, 0, 0));
  };
  auto load_v = [&](const Tile& t) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = block(t, v_codes);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kVW == 1) {
        vst[j][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_raw_buffer_load_b32(r, v_off + j * D, 0, 0));
      } else {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, v_off + j * D, 0, 0));
        vst[j][0] = v[0];
        vst[j][1 % kVW] = v[1];
      }
    }
  };
  auto store_k = [&](const Tile& t, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kKC; ++i)
#pragma unroll
      for (int f = 0; f < 2; ++f)
        *reinterpret_cast<lds_u32x4*>(lds + buf * kBufB + k_wr + (4 * i * 64 + 32 * f) * 16) =
            __builtin_bit_cast(u32x4, f8_frag(kst[i][2 * f], kst[i][2 * f + 1], t.ks, t.ks));
  };
  auto store_v = [&](const Tile& t, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kVW; ++c) {
      uint32_t tr[4];
      f8_transpose4(vst[0][c], vst[1][c], vst[2][c], vst[3][c], tr);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * c + j;
        *reinterpret_cast<lds_u32x2*>(lds + buf * kBufB + v_wr + ((e % kDT) * 64 + 16 * (e / kDT)) * 16) =
            u32x2{__builtin_bit_cast(uint32_t, f8_to_f16<false>(tr[j], t.vs)), __builtin_bit_cast(uint32_t, f8_to_f16<true>(tr[j], t.vs))};
      }
    }
  };

  float m = kNegBig, lsum = 0.f, cand;
  f32x16 acc[kDT];
#pragma unroll
  for (int t = 0; t < kDT; ++t) acc[t] = f32x16{};
  const uint32_t frag = uint32_t(lane * 16);
  auto score = [&](f32x16 (&st)[2], const lds_u8* b) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        st[j] = mfma32(as_h8(*reinterpret_cast<const lds_u32x4*>(b + frag + (j * kSteps + s) * 1024)), qf[s],
                       s == 0 ? f32x16{} : st[j]);
  };
  // Causal limit, the sequence's end, pages outside the pool: score r of half j is key 32 j + 8 (r / 4) + 4 half + r % 4.
  auto mask = [&](f32x16 (&st)[2], const Tile& ti) __attribute__((always_inline)) {
    if (!((ti.fl == 15) & (ti.kt + kP8Tile - 1 <= wave_first))) {
      const int lim = my_pos - ti.kt;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int lp = ((ti.fl >> (2 * j + r / 8)) & 1) ? lim - 4 * half : -1;
          st[j][r] = f8_masked(32 * j + 8 * (r / 4) + r % 4 <= lp, st[j][r]);
        }
    }
  };
  auto row_max = [&](const f32x16 (&st)[2]) __attribute__((always_inline)) {
    float mx[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const f32x16& v = st[a / 4];
      const int o = 4 * (a % 4);
      mx[a] = fmaxf(fmaxf(v[o], v[o + 1]), fmaxf(v[o + 2], v[o + 3]));
    }
    cand = max_lane32(fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                            fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])))) * scale_log2;
  };
  // The reference maximum moves only when a score exceeds it by more than 8 (log2 units), so P < 2^8.
  auto rescale = [&]() __attribute__((always_inline)) {
    const bool grow = cand > m + 8.f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float mn = grow ? cand : m;
      const float alpha = exp2_fast(m - mn);
      lsum *= alpha;
#pragma unroll
      for (int t = 0; t < kDT; ++t) acc[t] *= alpha;
      m = mn;
    }
  };
  // Probabilities of keys 16 u .. 16 u + 15 in fp16 (what the second product multiplies, and lsum adds).
  auto prob = [&](const f32x16 (&st)[2], int u) __attribute__((always_inline)) -> f16x8 {
    float e[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) e[r] = exp2_fast(fmaf(st[u / 2][8 * (u % 2) + r], scale_log2, -m));
    return f16x8{f16(e[0]), f16(e[1]), f16(e[2]), f16(e[3]), f16(e[4]), f16(e[5]), f16(e[6]), f16(e[7])};
  };
  auto add_row_sum = [&](const f16x8& p) __attribute__((always_inline)) {
    const f16x2 one = f16x2{f16(1.f), f16(1.f)};
#pragma unroll
    for (int e = 0; e < 4; ++e) lsum = __builtin_amdgcn_fdot2(f16x2{p[2 * e], p[2 * e + 1]}, one, lsum, false);
  };
  auto pv = [&](const lds_u8* b, const f16x8& p, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kDT; ++t)
      acc[t] = mfma32(as_h8(*reinterpret_cast<const lds_u32x4*>(b + kTileB + frag + (u * kDT + t) * 1024)), p, acc[t]);
  };

  // Step i: tile i + 1's scores beside half of tile i's probabilities, then tile i's second product beside the other
  // half.  K of tile i + 2 and V of tile i + 1 go to the buffers that K of tile i and V of tile i - 1 left at the
  // barrier before; the loads of the next ones are issued.  (A wave whose columns end earlier only stages.)
  const int steps = int(ceil_div(n_tiles, KS));
  const int wave_steps = wave_tiles > grp ? int(ceil_div(wave_tiles - grp, KS)) : 0;
  Tile t1, t2;  // tiles i + 1 and i + 2
  auto step = [&](f32x16 (&sc)[2], f32x16 (&sn)[2], int i) __attribute__((always_inline)) {
    store_k(t2, i & 1);
    store_v(t1, (i + 1) & 1);
    const Tile t3 = tile_at(i + 3);
    load_k(t3);
    load_v(t2);
    if (i < wave_steps) {
      rescale();
      __builtin_amdgcn_sched_barrier(0);
      score(sn, lds + ((i + 1) & 1) * kBufB);
      f16x8 p[4];
      p[0] = prob(sc, 0);
      p[1] = prob(sc, 1);
      add_row_sum(p[0]);
      add_row_sum(p[1]);
      pin(p[0], p[1]);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // K fragment reads, two ahead
#pragma unroll
      for (int x = 0; x < 2 * kSteps; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // K fragment read
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // VALU
        __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);  // exp2
      }
      __builtin_amdgcn_sched_barrier(0);
      mask(sn, t1);
      const lds_u8* const vb = lds + (i & 1) * kBufB;
      pv(vb, p[0], 0);
      pv(vb, p[1], 1);
      p[2] = prob(sc, 2);
      p[3] = prob(sc, 3);
      pv(vb, p[2], 2);
      pv(vb, p[3], 3);
      add_row_sum(p[2]);
      add_row_sum(p[3]);
      row_max(sn);
    }
    t1 = t2;
    t2 = t3;
    p8_barrier();
  };
  f32x16 sa[2], sb[2];
  {
    const Tile t0 = tile_at(0);
    t1 = tile_at(1);
    t2 = tile_at(2);
    load_k(t0);
    load_v(t0);
    store_k(t0, 0);
    load_k(t1);
    store_v(t0, 0);
    load_v(t1);
    store_k(t1, 1);
    load_k(t2);
    p8_barrier();
    score(sa, lds);
    mask(sa, t0);
    row_max(sa);
    p8_barrier();  // every wave has left K of tile 0
  }
  for (int i = 0; i < steps; i += 2) {
    step(sa, sb, i);
    step(sb, sa, i + 1);
  }

  float l = lsum + __shfl_xor(lsum, 32);
  f32x16 o[kOwn];
  if constexpr (KS == 1) {
#pragma unroll
    for (int d = 0; d < kOwn; ++d) o[d] = acc[d];
  } else {
    // The two key groups of a column block merge through LDS (free: the last barrier has passed): each wave hands
    // over the output tiles its partner finishes, with (m, l).
    float* const mb = reinterpret_cast<float*>(smem);
    auto slot = [&](int g) __attribute__((always_inline)) { return mb + ((g * kP8Waves + wave) * (16 * kOwn + 2)) * kWave + lane; };
    float* const mine = slot(grp);
    mine[0] = m;
    mine[kWave] = l;
#pragma unroll
    for (int d = 0; d < kOwn; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(2 + 16 * d + r) * kWave] = grp == 0 ? acc[kOwn + d][r] : acc[d][r];
    __syncthreads();
    const float* const other = slot(1 - grp);
    const float mo = other[0], lo = other[kWave];
    const float mm = fmaxf(m, mo), a = exp2_fast(m - mm), b = exp2_fast(mo - mm);
    l = fmaf(b, lo, a * l);
#pragma unroll
    for (int d = 0; d < kOwn; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        o[d][r] = fmaf(b, other[(2 + 16 * d + r) * kWave], a * (grp == 0 ? acc[d][r] : acc[kOwn + d][r]));
  }
  if (wc0 + col >= cols) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  // Row m = 8 a + 4 half + b of tile t is dim (m % 16) D / 16 + kDT (m / 16) + t: register 4 a + b.
  f16* op = out + (int64_t(my_q) * hq + my_h) * D + kOwn * grp;
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f16* dst = op + (8 * (a % 2) + 4 * half + b) * (D / 16) + kDT * (a / 2);
      const int r = 4 * a + b;
      if constexpr (kOwn == 4)
        *reinterpret_cast<f16x4*>(dst) = f16x4{f16(o[0][r] * inv), f16(o[1][r] * inv), f16(o[2][r] * inv), f16(o[3][r] * inv)};
      else if constexpr (kOwn == 2)
        *reinterpret_cast<f16x2*>(dst) = f16x2{f16(o[0][r] * inv), f16(o[1][r] * inv)};
      else
        *dst = f16(o[0][r] * inv);
    }
}

int prefill_fp8_block_launch(f16* out, const f16* q, const uint8_t* codes, const float* scales, int64_t num_pages,
                             const int32_t* table, int32_t query_start, int32_t T, int32_t hq, int32_t hkv, int32_t d,
                             float scale_log2, int groups, hipStream_t stream) {
  const int64_t n = ceil_div(int64_t(T) * (hq / hkv), kP8Cols);
  if (n * hkv >= int64_t(1) << 31) return IFN_ERR_UNSUPPORTED;
  auto k = d == 128 ? (groups == 2 ? prefill_fp8_block_kernel<128, 2> : prefill_fp8_block_kernel<128, 1>)
                    : (groups == 2 ? prefill_fp8_block_kernel<64, 2> : prefill_fp8_block_kernel<64, 1>);
  k<<<dim3(unsigned(n * hkv)), dim3(unsigned(groups * kP8Threads)), 0, stream>>>(
      out, q, codes, scales, num_pages, table, query_start, T, hkv, hq / hkv, int32_t(n), scale_log2);
  return ifn_launch_status();
}

}  // namespace ifn
