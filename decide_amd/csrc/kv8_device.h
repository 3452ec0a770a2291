// Device helpers of the 8-bit cache's kernels: where a page's parts lie, which sequence a work item belongs to.
#pragma once

#include "kv8.h"
#include "tile_common.h"

namespace dh {

// The parts of head h in a page: K codes [64][D], V codes [D][64], the 4 K scales and the 4 V scales.
template <int D>
__device__ __forceinline__ uint32_t kv_k_at(uint32_t h) { return h * (kKvPage * D); }
template <int D>
__device__ __forceinline__ uint32_t kv_v_at(uint32_t h, uint32_t kv_heads) { return (kv_heads + h) * (kKvPage * D); }
template <int D>
__device__ __forceinline__ uint32_t kv_scale_at(uint32_t h, uint32_t kv_heads) {
  return 2 * kv_heads * (kKvPage * D) + h * 32;
}

// Work items are numbered so that sequence s's start at first(s) = row0[s] * mul / div + s * extra, whatever the others
// hold: item i belongs to the last s with first(s) <= i. All 64 lanes look at once: one read for up to 64 sequences,
// two for 4,096 (a search that halves would wait for six reads one after another).
// Returns seqs where i lies before every sequence.
__device__ __forceinline__ uint32_t kv_find_seq(const uint32_t* __restrict__ row0, uint32_t seqs, uint32_t rows,
                                                uint64_t i, uint32_t mul, uint32_t div, uint32_t extra) {
  const uint32_t lane = __lane_id();
  uint32_t lo = 0, hi = seqs;  // the answer lies in [lo, hi)
  for (;;) {
    const uint32_t step = (hi - lo + 63) / 64;
    const uint32_t at = lo + lane * step;
    bool le = false;
    if (at < hi) le = (uint64_t)min(row0[at], rows) * mul / div + (uint64_t)at * extra <= i;
    const uint64_t vote = __ballot(le);
    const uint32_t n = __builtin_ctzll(~vote | (1ull << 63));  // lanes before the first that lies behind i
    const uint32_t cnt = vote == ~0ull ? 64 : n;
    if (cnt == 0) return seqs;
    lo += (cnt - 1) * step;
    hi = min(hi, lo + step);
    if (step == 1) return lo;
  }
}

}  // namespace dh
