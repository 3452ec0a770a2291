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
// hold: item i belongs to the last s with first(s) <= i. All 64 lanes look at once: one read for up to 63 sequences,
// two for 3,969 (a search that halves would wait for six reads one after another), and the sequence's rows, begin .. end
// - 1 (at most `rows`), come with it. Returns seqs where i lies before every sequence.
__device__ __forceinline__ uint32_t kv_find_seq(const uint32_t* __restrict__ row0, uint32_t seqs, uint32_t rows,
                                                uint64_t i, uint32_t mul, uint32_t div, uint32_t extra, uint32_t& begin,
                                                uint32_t& end) {
  const uint32_t lane = __lane_id();
  uint32_t lo = 0, hi = seqs;  // the answer lies in [lo, hi)
  for (;;) {
    const uint32_t step = (hi - lo + 62) / 63;
    const uint32_t at = min(lo + lane * step, seqs), first = min(row0[at], rows);
    const bool le = lane < 63 && at < hi && (uint64_t)first * mul / div + (uint64_t)at * extra <= i;
    const uint32_t n = (uint32_t)__builtin_ctzll(~__ballot(le));  // lanes before the first that lies behind i, at most 63
    if (n == 0) return seqs;
    if (step == 1) {
      begin = (uint32_t)__builtin_amdgcn_readlane((int)first, n - 1);
      end = (uint32_t)__builtin_amdgcn_readlane((int)first, n);
      return lo + n - 1;
    }
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
}

}  // namespace dh
