// Eviction of cache pages by accumulated attention weight (evict_pages).
//
// No counterpart in the reference, whose cache rows never shrink; it works on the tables of its documented
// paged layout (docs/architecture.md:225-240).  A row of n = ceil(len / 16) pages with n > keep keeps its first
// `sink` and last `recent` pages and, of the others, the keep - sink - recent of largest weight: the sum over
// kv heads of weights[b][h][j], in 64 bits and rounded to fp32 (NaN counts as the lowest, ties go to the lower
// j).  The row's table and weights close up in order; the evicted ids follow the kept ones.
//
// A row's first workgroup chooses: the sums become integers that order as the floats do; a radix select, at most three
// passes of 11 bits over LDS, finds the smallest kept one and how many of its equals are kept; one prefix sum over the
// threads, each with a run of the row's pages, gives every page its place, and the row is written through that
// permutation.  Further workgroups, one per kv head, write what no choice is needed for: the zeros behind the kept
// weights, or all the weights of a row that is not cut.  Counts are integers, so LDS atomics leave no trace of their
// order.
//
// What bounds it: latency -- lengths, sums, up to three passes, the scan, the row, one after the other.  32 rows of 8-256
// pages, 8 heads: 6.7 us (ranking by counting instead of the passes: 1.3-2.3 more); 64 rows of 1250-4096 pages (17 MB
// read and written): 12.8 us, where one workgroup a row that also wrote the zeros took 24.
#include <algorithm>

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

constexpr int kEvictBits = 11;   // of a digit
constexpr int kEvictBins = 1 << kEvictBits;

// Exclusive prefix sum of x over the workgroup's threads, and the total (s_sum: one word per wave; two barriers).
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* s_sum, uint32_t& total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  uint32_t y = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  if (lane == kWave - 1) s_sum[wave] = y;
  __syncthreads();
  uint32_t pre = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    const uint32_t v = s_sum[w];
    pre += w < wave ? v : 0u;
    total += v;
  }
  __syncthreads();
  return pre + y - x;
}

__global__ __launch_bounds__(kEvictThreads) void evict_pages_kernel(
    const int32_t* __restrict__ lens, const uint8_t* __restrict__ active, const float* __restrict__ weights,
    int32_t max_pages, int32_t hkv, int32_t keep, int32_t sink, int32_t recent,
    const int32_t* __restrict__ tables,  // (up to here in registers at dispatch: build.py)
    int32_t* __restrict__ out_tables, int32_t* __restrict__ out_lens, float* __restrict__ out_weights,
    int32_t* __restrict__ num_evicted) {
  extern __shared__ uint32_t s_key[];  // max_pages: the keys, then the row's permutation
  __shared__ int s_hist[kEvictBins];
  __shared__ uint32_t s_sum[kEvictWaves];
  __shared__ int s_pick[3];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  const int len = lens[b];
  const bool on = active == nullptr || active[b] != 0;
  const int n = (max(0, min(len, max_pages * 16)) + 15) / 16;
  const bool cut = on && n > keep;
  const float* w = weights + b * hkv * max_pages;
  float* out_w = out_weights + b * hkv * max_pages;
  if (blockIdx.y > 0) {
    for (int h = int(blockIdx.y) - 1; h < hkv; h += int(gridDim.y) - 1) {
      const int64_t at = int64_t(h) * max_pages;
      for (int j = (cut ? keep : 0) + tid; j < max_pages; j += kEvictThreads) out_w[at + j] = !cut && j < n ? w[at + j] : 0.f;
    }
    return;
  }
  const int gone = cut ? n - keep : 0;
  const int32_t* row = tables + b * max_pages;
  int32_t* out_row = out_tables + b * max_pages;
  if (tid == 0) {
    out_lens[b] = len - 16 * gone;
    num_evicted[b] = gone;
  }
  for (int j = (cut ? n : 0) + tid; j < max_pages; j += kEvictThreads) out_row[j] = row[j];
  if (!cut) return;

  // keys of the candidates [lo, hi): four pages of eight heads a thread are in flight
  const int lo = sink, hi = n - recent;
  for (int j0 = lo; j0 < hi; j0 += 4 * kEvictThreads) {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    for (int h0 = 0; h0 < hkv; h0 += 8) {
      float v[4][8];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = min(j0 + c * kEvictThreads + tid, hi - 1);
        if (j0 + c * kEvictThreads >= hi) continue;  // (uniform)
#pragma unroll
        for (int x = 0; x < 8; ++x) v[c][x] = w[int64_t(min(h0 + x, hkv - 1)) * max_pages + j];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (j0 + c * kEvictThreads >= hi) continue;
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (h0 + x < hkv) sum[c] += double(v[c][x]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = j0 + c * kEvictThreads + tid;
      if (j < hi) s_key[j] = order_key(float(sum[c]));
    }
  }
  // the left-th largest key, digit by digit; left: how many of those equal to it (under mask) are kept
  int left = keep - sink - recent;
  uint32_t prefix = 0, mask = 0;
  for (int shift = 32 - kEvictBits; left > 0; shift = max(shift - kEvictBits, 0)) {
    const uint32_t digit = shift == 0 ? ~mask : uint32_t(kEvictBins - 1) << shift;
    s_hist[tid] = 0;
    s_hist[tid + kEvictThreads] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kEvictThreads) {
      const uint32_t k = s_key[j];
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k & digit) >> shift], 1);
    }
    __syncthreads();
    // thread i: bins 2047 - 2 i and 2046 - 2 i
    const int c0 = s_hist[kEvictBins - 1 - 2 * tid], c1 = s_hist[kEvictBins - 2 - 2 * tid];
    uint32_t total;
    const int before = int(block_scan(uint32_t(c0 + c1), s_sum, total));
    if (before < left && before + c0 + c1 >= left) {  // (one thread)
      const bool second = before + c0 < left;
      s_pick[0] = kEvictBins - 1 - 2 * tid - (second ? 1 : 0);
      s_pick[1] = left - before - (second ? c0 : 0);
      s_pick[2] = second ? c1 : c0;
    }
    __syncthreads();
    prefix |= uint32_t(s_pick[0]) << shift;
    mask |= digit;
    left = s_pick[1];
    if (shift == 0 || left == s_pick[2]) break;  // (all of the bin's are kept: its lower digits do not matter)
  }
  // Each thread: a run of `per` pages.  Kept: over the key, or one of the first `left` equal to it.
  const int per = (n + kEvictThreads - 1) / kEvictThreads, first = tid * per;  // (per <= 32)
  uint32_t over = 0, same = 0;
  for (int k = 0; k < per; ++k) {
    const int j = first + k;
    if (j >= n) break;
    if (j < lo || j >= hi) {
      over |= 1u << k;
    } else if (left > 0) {
      const uint32_t key = s_key[j] & mask;
      over |= uint32_t(key > prefix) << k;
      same |= uint32_t(key == prefix) << k;
    }
  }
  uint32_t total;
  const uint32_t before = block_scan(uint32_t(__popc(over)) << 16 | uint32_t(__popc(same)), s_sum, total);
  int over_before = int(before >> 16), same_before = int(before & 0xffffu);
  for (int k = 0; k < per; ++k) {  // (every key has been read: the scan's barriers)
    const int j = first + k;
    if (j >= n) break;
    const bool s = (same >> k) & 1u, take = ((over >> k) & 1u) != 0 || (s && same_before < left);
    const int at = over_before + min(same_before, left);  // kept pages before j
    s_key[take ? at : keep + j - at] = uint32_t(j);
    over_before += (over >> k) & 1u;
    same_before += s ? 1 : 0;
  }
  __syncthreads();
  for (int j = tid; j < n; j += kEvictThreads) out_row[j] = row[s_key[j]];
  for (int x = tid; x < keep * hkv; x += kEvictThreads) {
    const int64_t at = int64_t(x / keep) * max_pages;
    out_w[at + x % keep] = w[at + s_key[x % keep]];
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
  if (block_size != 16 || max_pages_per_seq > kEvictMaxPages ||
      int64_t(std::min(keep_pages, max_pages_per_seq)) * num_kv_heads >= int64_t(1) << 31)
    return IFN_ERR_UNSUPPORTED;
  if (batch == 0) return IFN_OK;
  evict_pages_kernel<<<dim3(unsigned(batch), unsigned(1 + std::min<int32_t>(num_kv_heads, 32))), dim3(kEvictThreads),
                       size_t(max_pages_per_seq) * 4, static_cast<hipStream_t>(stream)>>>(
      seq_lens, active_mask, page_weights, max_pages_per_seq, num_kv_heads, keep_pages, sink_pages, recent_pages,
      block_tables, out_tables, out_lens, out_weights, num_evicted);
  return ifn_launch_status();
}
