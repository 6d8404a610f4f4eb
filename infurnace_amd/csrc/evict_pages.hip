// Eviction of cache pages by accumulated attention weight (evict_pages).
//
// No counterpart in the reference, whose cache rows never shrink; it works on the tables of its documented
// paged layout (docs/architecture.md:225-240).  A row of n = ceil(len / 16) pages with n > keep keeps its first
// `sink` and last `recent` pages and, of the others, the keep - sink - recent of largest weight: the sum over
// kv heads of weights[b][h][j], in 64 bits and rounded to fp32 (NaN counts as the lowest, ties go to the lower
// j).  The row's table and weights close up in order; the evicted ids follow the kept ones.
//
// One workgroup per row.  The sums become integers that order as the floats do; a radix select, four passes of
// eight bits over LDS, finds the smallest kept one and how many of its equals are kept; then one ordered pass
// with prefix sums writes the row.  Counts are integers, so LDS atomics leave no trace of their order.
#include "ifn_common.hpp"

namespace ifn {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kEvictMaxPages = 32768;  // table columns (LDS: one key each)

// Larger float, larger integer; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

__global__ __launch_bounds__(kEvictThreads) void evict_pages_kernel(
    int32_t* __restrict__ out_tables, int32_t* __restrict__ out_lens, float* __restrict__ out_weights,
    int32_t* __restrict__ num_evicted, const int32_t* __restrict__ tables, int32_t max_pages,
    const int32_t* __restrict__ lens, const uint8_t* __restrict__ active, const float* __restrict__ weights,
    int32_t hkv, int32_t keep, int32_t sink, int32_t recent) {
  extern __shared__ uint32_t s_key[];  // max_pages
  __shared__ int s_hist[256];
  __shared__ int s_sum[2][kEvictWaves];
  __shared__ int s_pick[2];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t b = blockIdx.x;
  const int cap = max_pages * 16;
  const int len = lens[b];
  const bool on = active == nullptr || active[b] != 0;
  const int n = (max(0, min(len, cap)) + 15) / 16;
  const bool cut = on && n > keep;
  const int gone = cut ? n - keep : 0;
  const int32_t* row = tables + b * max_pages;
  int32_t* out_row = out_tables + b * max_pages;
  const float* w = weights + b * hkv * max_pages;
  float* out_w = out_weights + b * hkv * max_pages;
  if (tid == 0) {
    out_lens[b] = len - 16 * gone;
    num_evicted[b] = gone;
  }
  if (!cut) {
    for (int j = tid; j < max_pages; j += kEvictThreads) out_row[j] = row[j];
    for (int64_t i = tid; i < int64_t(hkv) * max_pages; i += kEvictThreads)
      out_w[i] = int(i % max_pages) < n ? w[i] : 0.f;
    return;
  }
  const int lo = sink, hi = n - recent;  // candidates [lo, hi)
  for (int j = lo + tid; j < hi; j += kEvictThreads) {
    double s = 0.0;
    for (int h = 0; h < hkv; ++h) s += double(w[int64_t(h) * max_pages + j]);
    s_key[j] = order_key(float(s));
  }
  // the left-th largest key, digit by digit
  int left = keep - sink - recent;
  uint32_t prefix = 0, mask = 0;
  if (left > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kEvictThreads) {
        const uint32_t k = s_key[j];
        if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (wave == 0) {  // lane i: digits 255 - 4 i .. 252 - 4 i
        int c[4], mine = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) mine += c[x] = s_hist[255 - 4 * lane - x];
        int upto = mine;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
          const int y = __shfl_up(upto, o);
          if (lane >= o) upto += y;
        }
        int before = upto - mine;
        if (before < left && upto >= left) {
          int x = 0;
          while (before + c[x] < left) before += c[x++];
          s_pick[0] = 255 - 4 * lane - x;
          s_pick[1] = left - before;
        }
      }
      __syncthreads();
      prefix |= uint32_t(s_pick[0]) << shift;
      mask |= 255u << shift;
      left = s_pick[1];
    }
  } else {
    __syncthreads();
  }
  // kept: over the key, or one of the first `left` equal to it
  int kept = 0, equal = 0;
  for (int j0 = 0; j0 < max_pages; j0 += kEvictThreads) {
    const int j = j0 + tid;
    bool eq = false, take = j < lo || (j >= hi && j < n);
    if (j >= lo && j < hi && keep > sink + recent) {
      const uint32_t k = s_key[j];
      take = k > prefix;
      eq = k == prefix;
    }
    const uint64_t beq = __builtin_amdgcn_ballot_w64(eq);
    if (lane == 0) s_sum[0][wave] = __builtin_popcountll(beq);
    __syncthreads();
    int pre = 0, tot = 0;
#pragma unroll
    for (int x = 0; x < kEvictWaves; ++x) {
      const int v = s_sum[0][x];
      pre += x < wave ? v : 0;
      tot += v;
    }
    const uint64_t below = (uint64_t(1) << lane) - 1;
    if (eq && equal + pre + __builtin_popcountll(beq & below) < left) take = true;
    equal += tot;
    const uint64_t bt = __builtin_amdgcn_ballot_w64(take);
    if (lane == 0) s_sum[1][wave] = __builtin_popcountll(bt);
    __syncthreads();
    pre = tot = 0;
#pragma unroll
    for (int x = 0; x < kEvictWaves; ++x) {
      const int v = s_sum[1][x];
      pre += x < wave ? v : 0;
      tot += v;
    }
    const int at = kept + pre + __builtin_popcountll(bt & below);  // kept pages before j
    kept += tot;
    if (j < max_pages) {
      const int dst = j >= n ? j : take ? at : keep + j - at;
      out_row[dst] = row[j];
      for (int h = 0; h < hkv; ++h) {
        const int64_t base = int64_t(h) * max_pages;
        out_w[base + dst] = take ? w[base + j] : 0.f;
      }
    }
  }
}

}  // namespace ifn

extern "C" int ifn_evict_pages(int32_t* out_tables, int32_t* out_lens, float* out_weights, int32_t* num_evicted,
                               const int32_t* block_tables, int32_t max_pages_per_seq, const int32_t* seq_lens,
                               const uint8_t* active_mask, const float* page_weights, int32_t batch,
                               int32_t num_kv_heads, int32_t block_size, int32_t keep_pages, int32_t sink_pages,
                               int32_t recent_pages, void* stream) {
  using namespace ifn;
  if (out_tables == nullptr || out_lens == nullptr || out_weights == nullptr || num_evicted == nullptr ||
      block_tables == nullptr || seq_lens == nullptr || page_weights == nullptr)
    return IFN_ERR_INVALID_ARGUMENT;
  if (batch < 0 || max_pages_per_seq < 1 || num_kv_heads < 1 || block_size < 1 || sink_pages < 0 || recent_pages < 1 ||
      int64_t(keep_pages) < int64_t(sink_pages) + recent_pages)
    return IFN_ERR_INVALID_ARGUMENT;
  if (block_size != 16 || max_pages_per_seq > kEvictMaxPages) return IFN_ERR_UNSUPPORTED;
  if (batch == 0) return IFN_OK;
  evict_pages_kernel<<<dim3(unsigned(batch)), dim3(kEvictThreads), size_t(max_pages_per_seq) * 4,
                       static_cast<hipStream_t>(stream)>>>(
      out_tables, out_lens, out_weights, num_evicted, block_tables, max_pages_per_seq, seq_lens, active_mask,
      page_weights, num_kv_heads, keep_pages, sink_pages, recent_pages);
  return ifn_launch_status();
}
