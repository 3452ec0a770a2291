// What the two attention kernels over the 8-bit cache share (kv8_attention.hip, kv8_wide.hip): codes to fp16, tiles of
// (row, head) pairs, and the runs of pages that workgroups take. Device code only.
#pragma once

#include <type_traits>

#include "kv8_device.h"

namespace dh {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr float kLazy = 8.0f;  // log2 headroom of the softmax reference point (weights up to 256)
constexpr float kLog2e = 1.4426950408889634f;

// 8 code bytes (two words) as fp16 numbers, exactly.
template <bool INT8>
__device__ __forceinline__ h8 numbers(uint32_t a, uint32_t b) {
  h2 p[4];
  if constexpr (INT8) {
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    auto two = [&](uint32_t x, uint32_t sel) {
      return __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, sel)) - bias;
    };
    p[0] = two(a, 0x04010400u), p[1] = two(a, 0x04030402u), p[2] = two(b, 0x04010400u), p[3] = two(b, 0x04030402u);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
  }
  h8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[2 * i] = p[i][0], r[2 * i + 1] = p[i][1];
  return r;
}

// Combined over the four lanes (n, 0 .. 3) that hold one pair's scores.
__device__ __forceinline__ float max_groups(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  auto with = [&](auto lanes) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(lanes)::value, 0xf, 0xf, false));
  };
  with(std::integral_constant<int, 0xb1>{});   // the neighbour's
  with(std::integral_constant<int, 0x4e>{});   // the neighbouring pair's
  with(std::integral_constant<int, 0x141>{});  // mirrored within 8 lanes: the other four's
  with(std::integral_constant<int, 0x140>{});  // within 16: the other eight's
  auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)max(a[0], a[1]));
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// How many tokens row r sees (0 .. 2^32 - 1): its position and those before it; no position wraps to none.
__device__ __forceinline__ uint32_t seen_by(const KvArgs& a, uint32_t r) { return a.qpos[r] + 1u; }

struct Tile {
  uint32_t seq;         // sequence
  uint32_t pairs;       // pairs (rows x group) from the tile's first on, in the sequence
  uint32_t row, extra;  // the first pair's row, and its head in the group
};

struct AttnArgs {
  const _Float16* q;
  const float* gate;  // or null
  _Float16* y;
  float* ws;  // the runs' states (KvAttnPlan)
  uint32_t ldq, ldg, ldy, heads, group;
  uint32_t group_inv;  // 2^21 / group, rounded up
  uint32_t slots;  // tiles are numbered below it
  uint32_t runs;   // of each kv head; 0: a workgroup per tile
  uint32_t min_run;
  float scale;
};

// Tile `slot` of a kv head: sequences' tiles start at row0 * group / TILE + s, which leaves room for all of them.
template <uint32_t TILE>
__device__ __forceinline__ bool tile_of(const KvArgs& a, uint32_t group, uint32_t slot, uint32_t seq, uint32_t begin,
                                        uint32_t end, Tile& t) {
  const uint32_t r0 = min(begin, a.rows), r1 = min(end, a.rows);
  if (r1 <= r0) return false;
  const uint32_t pairs = (r1 - r0) * group, first = (slot - (uint32_t)((uint64_t)r0 * group / TILE) - seq) * TILE;
  if (first >= pairs) return false;
  t = Tile{seq, pairs - first, r0 + first / group, first % group};
  return true;
}
template <uint32_t TILE>
__device__ __forceinline__ bool find_tile(const KvArgs& a, uint32_t group, uint32_t slot, Tile& t) {
  uint32_t begin, end;
  const uint32_t s = kv_find_seq(a.row0, a.seqs, a.rows, slot, group, TILE, 1, begin, end);
  return s < a.seqs && tile_of<TILE>(a, group, slot, s, begin, end, t);
}
// Row and head of the tile's pair k < 128. For x = extra + k < group + 128, x times the rounded 2^21 / group is off by
// less than x, and x group < 2^21 for groups of at most 1,024: the quotient is exact. (The product stays below 2^32.)
__device__ __forceinline__ void pair_at(const AttnArgs& t, const Tile& tile, uint32_t kvh, uint32_t k, uint32_t& row,
                                        uint32_t& head) {
  const uint32_t x = tile.extra + k, q = x * t.group_inv >> 21;
  row = tile.row + q;
  head = kvh * t.group + (x - q * t.group);
}

// Pages of `seen` tokens. One page past the table is enough to make the row NaN.
__device__ __forceinline__ uint32_t pages_of(const KvArgs& a, uint32_t seen) {
  const uint32_t n = seen / kKvPage + (seen % kKvPage != 0);  // at most 2^26
  return n > a.ld_table ? a.ld_table + 1 : n;
}

// The runs: run w of `share` pages each, over the tiles' pages one after another.
__device__ __forceinline__ uint32_t share_of(uint32_t total, const AttnArgs& t) {
  return max((total + t.runs - 1) / t.runs, t.min_run);
}
// Where a run leaves a tile's state: its first tile's at 0, another's that goes on in the next run at 1.
template <int D, uint32_t TILE>
__device__ __forceinline__ float* state_of(const AttnArgs& t, uint32_t kvh, uint32_t run, uint32_t which) {
  return t.ws + ((size_t)(kvh * t.runs + run) * 2 + which) * (TILE * (D + 2));
}
// The pages before each tile, left behind the states for the combine.
template <int D, uint32_t TILE>
__device__ __forceinline__ uint32_t* starts_of(const KvArgs& a, const AttnArgs& t) {
  return (uint32_t*)(t.ws + (size_t)a.kv_heads * t.runs * 2 * (TILE * (D + 2)));
}

// What a workgroup that takes runs keeps in LDS: the pages before each tile, the tile's sequence, the sequences' rows.
template <uint32_t SLOTS>
struct Deal {
  uint32_t before[SLOTS + 1], seq[SLOTS + 1], row0[SLOTS + 1], sums[8];
};

// Adds up the pages of all tiles, every workgroup for itself (the reads are the same for all and few: each row's position
// once), and says which pages are this run's.
template <int D, uint32_t TILE, uint32_t SLOTS, uint32_t THREADS>
__device__ __forceinline__ void deal_runs(const KvArgs& a, const AttnArgs& t, uint32_t run, Deal<SLOTS>& d, uint32_t& u,
                                          uint32_t& u1) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (uint32_t i = tid; i <= a.seqs; i += THREADS) d.row0[i] = min(a.row0[i], a.rows);
  __syncthreads();
#pragma unroll 1
  for (uint32_t slot = tid; slot < t.slots; slot += THREADS) {
    uint32_t lo = 0, hi = a.seqs;  // the last sequence that starts at or before the slot
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if ((uint64_t)d.row0[mid] * t.group / TILE + mid <= slot)
        lo = mid;
      else
        hi = mid;
    }
    Tile tile;
    uint32_t most = 0;
    if ((uint64_t)d.row0[lo] * t.group / TILE + lo <= slot &&
        tile_of<TILE>(a, t.group, slot, lo, d.row0[lo], d.row0[lo + 1], tile)) {
      const uint32_t rows = (tile.extra + min(TILE, tile.pairs) - 1) / t.group + 1;
#pragma unroll 4
      for (uint32_t r = tile.row; r < tile.row + rows; ++r) most = max(most, seen_by(a, r));
    }
    d.seq[slot] = lo;
    d.before[slot] = pages_of(a, most);
  }
  __syncthreads();
  // running sums: each thread some consecutive tiles, then the lanes, then the waves
  const uint32_t per = (t.slots + THREADS - 1) / THREADS, at0 = min(tid * per, t.slots), at1 = min(at0 + per, t.slots);
  uint32_t mine = 0;
#pragma unroll 1
  for (uint32_t i = at0; i < at1; ++i) mine += d.before[i];
  uint32_t sum = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t v = (uint32_t)__shfl_up((int)sum, o, 64);
    if (lane >= (uint32_t)o) sum += v;
  }
  if (lane == 63) d.sums[wave] = sum;
  __syncthreads();
  uint32_t at = sum - mine, total = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; ++w) {
    at += w < wave ? d.sums[w] : 0;
    total += d.sums[w];
  }
#pragma unroll 1
  for (uint32_t i = at0; i < at1; ++i) {
    const uint32_t n = d.before[i];
    d.before[i] = at;
    at += n;
  }
  if (tid == 0) d.before[t.slots] = total;
  __syncthreads();
  total = (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
  if (blockIdx.x == 0) {
    uint32_t* const out = starts_of<D, TILE>(a, t);
#pragma unroll 1
    for (uint32_t i = tid; i <= t.slots; i += THREADS) out[i] = d.before[i];
  }
  const uint32_t share = share_of(total, t);
  u = (uint32_t)min((uint64_t)run * share, (uint64_t)total);
  u1 = min(u + share, total);
}

// A value that all lanes have, in a scalar register.
__device__ __forceinline__ uint32_t same(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// The tile that holds page u of a kv head: the last that starts at or before it (empty ones start where the next does).
template <uint32_t SLOTS>
__device__ __forceinline__ uint32_t tile_at(const Deal<SLOTS>& d, uint32_t slots, uint32_t u) {
  uint32_t lo = 0, hi = slots;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (d.before[mid] <= u)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Four outputs of row r: O over its sum, times the sigmoid of the gate where there is one. A row that sees nothing is zero
// whatever its gate; one that sees only scores of -infinity has the sum 0 and is NaN, as its softmax is.
__device__ __forceinline__ void store_out(const AttnArgs& t, uint32_t r, uint32_t col, const f4& acc, float sum,
                                          uint32_t sees, const f4& gate) {
  f4 v = f4{0.f, 0.f, 0.f, 0.f};
  if (sees) {
    v = acc * (1.0f / sum);
    if (t.gate) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= sigmoid(gate[e]);
    }
  }
  *(h4*)(t.y + (size_t)r * t.ldy + col) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}
// eight dims, already over their sum (zeros, and the gate one too, for a row that sees nothing)
__device__ __forceinline__ void store_out8(const AttnArgs& t, uint32_t r, uint32_t col, f4 v0, f4 v1, const f4& g0,
                                           const f4& g1) {
  typedef _Float16 h8u __attribute__((ext_vector_type(8), aligned(8)));
  if (t.gate) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v0[e] *= sigmoid(g0[e]), v1[e] *= sigmoid(g1[e]);
  }
  *(h8u*)(t.y + (size_t)r * t.ldy + col) = h8u{(_Float16)v0[0], (_Float16)v0[1], (_Float16)v0[2], (_Float16)v0[3],
                                               (_Float16)v1[0], (_Float16)v1[1], (_Float16)v1[2], (_Float16)v1[3]};
}

// weight of a state whose reference point is m among those whose largest is top; none where it met no score
__device__ __forceinline__ float state_weight(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// Masks the scores of a block of which a pair sees `mine` tokens. They are scaled in the exponent, as where all is seen, so
// that a mask that is there for another pair of the tile rounds nothing twice: `unit` is what they are yet to be multiplied
// by. A factor that is 0 or NaN goes in beforehand: it would make NaN of the masked ones' -infinity.
template <typename V>
__device__ __forceinline__ void mask_scores(V& s, float cs, uint32_t mine, float& unit) {
  const bool early = mine != 0 && !(cs > 0.f);
  if (__any(early)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= early ? cs : 1.0f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = i < (int)mine ? s[i] : -INFINITY;
  unit = mine != 0 && cs > 0.f ? cs : 1.0f;
}

// V's scales differ from block to block, so what a pair rounds to fp16 is the product of a token's weight and its block's
// scale, relative to `vref`: at least the largest block's share (its largest weight times its scale) over 2^8 among the
// blocks that this pair sees, and at most the largest. So the products stay at most 2^8, and each is off by 2^-11 of
// itself or 2^-25 of the largest share, whatever scales unseen blocks or those of next to no weight have. (A block that is
// seen in part counts with its whole scale, which its seen tokens are coded in: a code's half step is 2^-10 of it at least.)
// Relative to the largest scale alone, a block of values 2^20 larger behind a row's position took 5 % of that row.
constexpr float kNoScale = 0x1p-100f;   // no block's scale is smaller
constexpr float kMostScale = 0x1p126f;  // vref's, and a ratio's, largest: the reciprocal and the products stay finite
__device__ __forceinline__ float block_share(float top, float m, float vs) {
  return __builtin_amdgcn_exp2f(top - (m == -INFINITY ? 0.f : m)) * vs;
}
// Whether a page whose largest score and share are bm and vm moves the pair's reference points.
__device__ __forceinline__ bool moves(float bm, float m, float vm, float vref) {
  return bm > m + kLazy || vm > 256.0f * vref;
}
// (blocks that were never written, with scales of zero, leave it where it was)
__device__ __forceinline__ float next_reference(float vold, float share) {
  return fminf(fmaxf(fmaxf(vold, share), kNoScale), kMostScale);
}
__device__ __forceinline__ float scale_ratio(float vs, float vref) {
  const float r = vs * __builtin_amdgcn_rcpf(vref);  // off by 2^-23 at most
  return r > kMostScale ? kMostScale : r;  // (where weights vanish; a NaN scale stays)
}

// kv8_wide.hip: the kernel for many rows, over t.runs runs or t.slots tiles
hipError_t launch_kv8_wide(const KvArgs& a, const AttnArgs& t, uint32_t head_dim, bool int8, hipStream_t s);

}  // namespace dh
