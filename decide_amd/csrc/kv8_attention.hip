// Attention over the 8-bit paged cache, for gfx950 MFMA:
//   y[r, h] = softmax_t(scale * q[r, h] . K[t]) . V[t] (x sigmoid(gate)), tokens t = 0 ..= qpos[r] of the row's sequence.
//
// kv8_attention_kernel, tiles of 16 (row, head) pairs of one kv head:
//   * Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_16x16x32_f16: lane (n, g), n = lane
//     % 16, g = lane / 16, holds scores of ONE pair n. The key rows that a product takes are dealt so that over a page
//     (64 tokens, four products) lane group g gets the 16 scores of the page's block g: one K scale and one V scale a
//     lane, and the scores are, in order, the operand that P^T V needs when the products run over tokens 16 g + 8 e + j.
//     V lies transposed in the page, so the other operand's 16 tokens are 16 consecutive bytes. Nothing of K, V, S or P
//     goes through LDS.
//   * Codes become fp16 exactly (e4m3: one conversion for two; int8: a byte next to 0x64 is 1024 + b as fp16, then one
//     subtraction for two). The K scale joins the softmax's factor; the V scale, relative to the largest that the wave
//     has met, multiplies the weight in fp32 before its rounding to fp16, so weights stay at most 2^8 and one page's small
//     scale cannot push another's weights out of fp16's range.
//   * The eight waves of a workgroup take every eighth page and meet at the end of a tile, through LDS.
//   * Sequences of one call may differ in length by any factor, and the host does not know them. So the workgroups of a
//     kv head (one per CU in all) add up the pages of all tiles, each for itself, and take equal runs of them: a run may
//     end one tile and begin another. A tile that lies in several runs leaves a state (largest score, sum, O) per run, and
//     kv8_combine_kernel merges them in order. With pieces of a fixed length instead, sized by the longest sequence, 64
//     sequences of up to 8,192 tokens made 2,560 workgroups, 2,100 of them empty, and took 77 us against XX.
#include <algorithm>

#include "kv8_device.h"

namespace dh {

namespace {
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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// How many tokens row r sees (0 .. 2^32 - 1): its position and those before it; no position wraps to none.
__device__ __forceinline__ uint32_t seen_by(const KvArgs& a, uint32_t r) { return a.qpos[r] + 1u; }

struct Tile {
  uint32_t seq, r0, pairs, first;  // sequence, its first row, its pairs (rows x group), the tile's first pair
};

struct AttnArgs {
  const _Float16* q;
  const float* gate;  // or null
  _Float16* y;
  float* ws;  // the runs' states (KvAttnPlan)
  uint32_t ldq, ldg, ldy, heads, group;
  uint32_t slots;  // tiles are numbered below it
  uint32_t runs;   // of each kv head; 0: a workgroup per tile
  float scale;
};

// Tile `slot` of a kv head: sequences' tiles start at row0 * group / 16 + s, which leaves room for all of them.
__device__ __forceinline__ bool tile_of(const KvArgs& a, uint32_t group, uint32_t slot, uint32_t seq, uint32_t begin,
                                        uint32_t end, Tile& t) {
  t.seq = seq;
  t.r0 = min(begin, a.rows);
  const uint32_t r1 = min(end, a.rows);
  if (r1 <= t.r0) return false;
  t.pairs = (r1 - t.r0) * group;
  t.first = (slot - (uint32_t)((uint64_t)t.r0 * group / kKvTile) - seq) * kKvTile;
  return t.first < t.pairs;
}
__device__ __forceinline__ bool find_tile(const KvArgs& a, uint32_t group, uint32_t slot, Tile& t) {
  const uint32_t s = kv_find_seq(a.row0, a.seqs, a.rows, slot, group, kKvTile, 1);
  return s < a.seqs && tile_of(a, group, slot, s, a.row0[s], a.row0[s + 1], t);
}

// Pages of `seen` tokens. One page past the table is enough to make the row NaN.
__device__ __forceinline__ uint32_t pages_of(const KvArgs& a, uint32_t seen) {
  return min(seen / kKvPage + (seen % kKvPage != 0), a.ld_table + 1);
}

// The runs: run w of `share` pages each, over the tiles' pages one after another.
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t runs) {
  return max((total + runs - 1) / runs, kKvMinRun);
}
// Where a run leaves a tile's state: its first tile's at 0, another's that goes on in the next run at 1.
template <int D>
__device__ __forceinline__ float* state_of(const AttnArgs& t, uint32_t kvh, uint32_t run, uint32_t which) {
  return t.ws + ((size_t)(kvh * t.runs + run) * 2 + which) * (kKvTile * (D + 2));
}
// The pages before each tile, left behind the states for the combine.
template <int D>
__device__ __forceinline__ uint32_t* starts_of(const KvArgs& a, const AttnArgs& t) {
  return (uint32_t*)(t.ws + (size_t)a.kv_heads * t.runs * 2 * (kKvTile * (D + 2)));
}

__device__ __forceinline__ void store_out(const AttnArgs& t, uint32_t r, uint32_t col, const f4& acc, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  f4 v = acc * inv;
  if (t.gate) {
    const f4 gt = *(const f4*)(t.gate + (size_t)r * t.ldg + col);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= sigmoid(gt[e]);
  }
  *(h4*)(t.y + (size_t)r * t.ldy + col) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

// weight of a state whose reference point is m among those whose largest is top; none where it met no score
__device__ __forceinline__ float state_weight(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}
}  // namespace

template <int D, bool INT8>
__global__ __launch_bounds__(512) void kv8_attention_kernel(KvArgs a, AttnArgs t) {
  constexpr int S = D / 64;    // 64-byte quarters of a key: two products each
  constexpr int DT = D / 16;   // 16-dim tiles of O
  constexpr int kPad = D + 4;  // floats of a pair's O in LDS
  constexpr int kWaves = 8;
  __shared__ __attribute__((aligned(16))) float lds[kWaves * kKvTile * kPad];
  __shared__ f2 ml[kWaves * kKvTile];
  __shared__ uint32_t before[kKvMaxSlots + 1];  // pages of the tiles before each
  __shared__ uint32_t seq_of[kKvMaxSlots], row0[kKvMaxSlots + 1];
  __shared__ uint32_t sums[kWaves];
  const uint32_t kvh = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = lane & 15, g = lane >> 4;
  uint32_t u = 0, u1 = 1;  // pages of the run
  if (t.runs) {
    for (uint32_t i = tid; i <= a.seqs; i += 512) row0[i] = min(a.row0[i], a.rows);
    __syncthreads();
    // each thread counts the pages of some consecutive tiles
    constexpr uint32_t kPer = kKvMaxSlots / 512;
    const uint32_t per = (t.slots + 511) / 512;
    uint32_t count[kPer], mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      count[i] = 0;
      const uint32_t slot = tid * per + i;
      if (i >= per || slot >= t.slots) continue;
      seq_of[slot] = 0;
      uint32_t lo = 0, hi = a.seqs;  // the last sequence that starts at or before the slot
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint64_t)row0[mid] * t.group / kKvTile + mid <= slot)
          lo = mid;
        else
          hi = mid;
      }
      Tile tile;
      if ((uint64_t)row0[lo] * t.group / kKvTile + lo > slot ||
          !tile_of(a, t.group, slot, lo, row0[lo], row0[lo + 1], tile))
        continue;
      seq_of[slot] = lo;
      uint32_t most = 0;
      const uint32_t ra = tile.r0 + tile.first / t.group,
                     rb = tile.r0 + (min(tile.first + kKvTile, tile.pairs) - 1) / t.group;
#pragma unroll 4
      for (uint32_t r = ra; r <= rb; ++r) most = max(most, seen_by(a, r));
      count[i] = pages_of(a, most);
      mine += count[i];
    }
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = (uint32_t)__shfl_up((int)sum, o, 64);
      if (lane >= (uint32_t)o) sum += v;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    uint32_t at = sum - mine, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      at += w < wave ? sums[w] : 0;
      total += sums[w];
    }
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      const uint32_t slot = tid * per + i;
      if (i < per && slot < t.slots) before[slot] = at;
      at += count[i];
    }
    if (tid == 0) before[t.slots] = total;
    __syncthreads();
    if (blockIdx.x == 0) {
      uint32_t* const out = starts_of<D>(a, t);
      for (uint32_t i = tid; i <= t.slots; i += 512) out[i] = before[i];
    }
    const uint32_t share = share_of(total, t.runs);
    u = (uint32_t)min((uint64_t)run * share, (uint64_t)total);
    u1 = min(u + share, total);
  }
  const uint32_t first_u = u;
  const float c = t.scale * kLog2e;
  const uint32_t ktok = (n >> 2) * 16 + (n & 3);  // this lane's key of a product: token ktok + 4 T

  while (u < u1) {
    uint32_t slot = run, tile_u = 0;
    Tile tile;
    if (t.runs) {  // the tile that holds page u: the last that starts at or before it (empty ones start where the next does)
      uint32_t lo = 0, hi = t.slots;
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (before[mid] <= u)
          lo = mid;
        else
          hi = mid;
      }
      slot = lo;
      tile_u = before[lo];
      const uint32_t s = seq_of[lo];
      if (!tile_of(a, t.group, lo, s, row0[s], row0[s + 1], tile)) return;  // it has pages, so it has rows
    } else if (!find_tile(a, t.group, slot, tile)) {
      return;
    }
    const uint32_t pair = min(tile.first + n, tile.pairs - 1);
    const uint32_t row = tile.r0 + pair / t.group, head = kvh * t.group + pair % t.group;
    const uint32_t seen = seen_by(a, row);
    const uint32_t most = wave_max_u32(seen);
    const uint32_t least = ~wave_max_u32(~seen);
    const uint32_t npages = pages_of(a, most);
    const uint32_t b0 = u - tile_u, b1 = t.runs ? min(npages, u1 - tile_u) : npages;
    if (t.runs && b1 <= b0) return;  // positions that changed under the call
    const bool whole = b0 == 0 && b1 == npages;
    const uint32_t* const table = a.table + (size_t)tile.seq * a.ld_table;

    // Q: dims 64 j + 16 g + 8 e .. + 7 of pair n
    h8 q[2 * S];
    {
      const _Float16* qp = t.q + (size_t)row * t.ldq + head * D + 16 * g;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        q[2 * j] = *(const h8*)(qp + 64 * j);
        q[2 * j + 1] = *(const h8*)(qp + 64 * j + 8);
      }
    }
    f4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    float vref = 0x1p-100f, inv_vref = 0x1p100f;  // the largest V scale met; o is relative to it

    for (uint32_t b = b0 + wave; b < b1; b += kWaves) {
      const uint32_t id0 = b < a.ld_table ? table[b] : 0xffffffffu;
      const bool bad = id0 >= a.pages;
      const uint8_t* const rec = a.pool + (bad ? 0 : id0) * a.page_bytes;
      const uint8_t* const kp = rec + kv_k_at<D>(kvh) + ktok * D + 16 * g;
      const uint8_t* const vp = rec + kv_v_at<D>(kvh, a.kv_heads) + n * kKvPage + 16 * g;
      const float* const sp = (const float*)(rec + kv_scale_at<D>(kvh, a.kv_heads));
      const float ks0 = sp[g], vs0 = sp[4 + g];
      u4 kc[4][S], vc[DT];
#pragma unroll
      for (int T = 0; T < 4; ++T)
#pragma unroll
        for (int j = 0; j < S; ++j) kc[T][j] = *(const u4*)(kp + 4 * T * D + 64 * j);
#pragma unroll
      for (int i = 0; i < DT; ++i) vc[i] = *(const u4*)(vp + i * 16 * kKvPage);
      f4 st[4];
#pragma unroll
      for (int T = 0; T < 4; ++T) {
        st[T] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < S; ++j) {
          st[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(kc[T][j][0], kc[T][j][1]), q[2 * j], st[T], 0, 0,
                                                         0);
          st[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(kc[T][j][2], kc[T][j][3]), q[2 * j + 1], st[T],
                                                         0, 0, 0);
        }
      }
      float sv[16];
      const float cs = c * (bad ? NAN : ks0);
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = st[i / 4][i % 4] * cs;
      float vs = vs0;
      bool blind = false;  // the pair sees nothing of the lane's block
      const uint64_t tok0 = (uint64_t)b * kKvPage + 16 * g;
      if ((uint64_t)(b + 1) * kKvPage > least) {  // some pair does not see all of the page
        const uint32_t mine = seen > tok0 ? (uint32_t)min((uint64_t)seen - tok0, (uint64_t)16) : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) sv[i] = i < (int)mine ? sv[i] : -INFINITY;
        blind = mine == 0;
        if (tok0 >= most) vs = 0.f;  // the scale of a block that none sees may be anything
        if ((uint64_t)(b + 1) * kKvPage > most) {  // bytes behind the last seen token may be anything
          const uint32_t have = most > tok0 ? (uint32_t)min((uint64_t)most - tok0, (uint64_t)16) : 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int left = (int)have - 4 * w;
            const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1u;
#pragma unroll
            for (int i = 0; i < DT; ++i) vc[i][w] &= keep;
          }
        }
      }
      float bm = sv[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) bm = fmaxf(bm, sv[i]);
      bm = max_groups(bm);
      const float vm = max_groups(vs);  // the same in every lane
      if (__any(bm > m + kLazy) || vm > vref) {
        const float mnew = bm > m + kLazy ? bm : m;
        const float alpha = state_weight(m, mnew);
        const float vnew = fmaxf(vref, vm);
        l *= alpha;
        m = mnew;
        const float both = alpha * (vref / vnew);
        vref = vnew;
        inv_vref = 1.0f / vnew;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= both;
      }
      const float mref = m == -INFINITY ? 0.f : m;
      const float ratio = blind ? 0.f : vs * inv_vref;
      h8 p[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w = __builtin_amdgcn_exp2f(sv[i] - mref);
        l += w;
        p[i / 8][i % 8] = (_Float16)(w * ratio);
      }
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(vc[i][0], vc[i][1]), p[0], o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(vc[i][2], vc[i][3]), p[1], o[i], 0, 0, 0);
      }
    }

    // The waves meet: each leaves its O relative to the largest of their reference points.
    const uint32_t pairs = min(kKvTile, tile.pairs - tile.first);
    l = sum_groups(l);
    if (g == 0) ml[wave * kKvTile + n] = f2{m, l};
    __syncthreads();
    if (n < pairs) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w * kKvTile + n][0]);
      const float mine = state_weight(m, top) * vref;
#pragma unroll
      for (int i = 0; i < DT; ++i) *(f4*)(lds + (wave * kKvTile + n) * kPad + 16 * i + 4 * g) = o[i] * mine;
    }
    __syncthreads();
    float* const state = whole ? nullptr : state_of<D>(t, kvh, run, u == first_u ? 0 : 1);
    for (uint32_t i = tid; i < pairs * (D / 4); i += 512) {
      const uint32_t pr = i / (D / 4), d = 4 * (i % (D / 4));
      f4 acc = f4{0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w * kKvTile + pr][0]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f2 v = ml[w * kKvTile + pr];
        lt += v[0] == -INFINITY ? v[1] : v[1] * __builtin_amdgcn_exp2f(v[0] - top);  // a NaN sum stays
        acc += *(const f4*)(lds + (w * kKvTile + pr) * kPad + d);
      }
      if (whole) {
        store_out(t, tile.r0 + (tile.first + pr) / t.group, (kvh * t.group + (tile.first + pr) % t.group) * D + d, acc,
                  lt);
      } else {
        *(f4*)(state + pr * D + d) = acc;
        if (d == 0) *(f2*)(state + kKvTile * D + 2 * pr) = f2{top, lt};
      }
    }
    if (!t.runs) return;
    __syncthreads();  // the next tile's states go where these lay
    u = tile_u + b1;
  }
}

// Merges the states of every tile that lies in more than one run, in the runs' order, and writes the rows that see
// nothing. A workgroup per tile and kv head: D / 4 lanes a pair, and where the pairs leave lanes over, several groups take
// every so many runs of a pair.
template <int D>
__global__ __launch_bounds__(512) void kv8_combine_kernel(KvArgs a, AttnArgs t) {
  constexpr uint32_t L = D / 4;
  __shared__ __attribute__((aligned(16))) f4 sum[512];
  __shared__ float lsum[512];
  const uint32_t kvh = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads, tid = threadIdx.x;
  const uint32_t* const before = starts_of<D>(a, t);
  const uint32_t u0 = before[slot], u1 = before[slot + 1], share = share_of(before[t.slots], t.runs);
  const uint32_t w0 = u0 / share, w1 = u1 > u0 ? (u1 - 1) / share : w0;
  if (u1 > u0 && w0 == w1) return;  // written by the attention kernel itself
  Tile tile;
  if (!find_tile(a, t.group, slot, tile)) return;
  const uint32_t pairs = min(kKvTile, tile.pairs - tile.first);
  const uint32_t items = pairs * L;
  // `ways` groups of `items` lanes, or several rounds of one group
  const uint32_t ways = items <= 256 ? 512 / items : 1;
  const uint32_t way = ways > 1 ? tid / items : 0;
  for (uint32_t i0 = 0; i0 < items; i0 += 512) {
    const uint32_t i = ways > 1 ? tid % items : i0 + tid;
    const uint32_t pr = i / L, d = 4 * (i % L);
    const bool on = i < items && way < ways;
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (on && u1 > u0) {
      auto state = [&](uint32_t w) { return state_of<D>(t, kvh, w, w == w0 && u0 != w0 * share ? 1 : 0); };
      float top = -INFINITY;
#pragma unroll 8
      for (uint32_t w = w0; w <= w1; ++w) top = fmaxf(top, state(w)[kKvTile * D + 2 * pr]);
#pragma unroll 4
      for (uint32_t w = w0 + way; w <= w1; w += ways) {
        const float* const s = state(w);
        const f2 v = *(const f2*)(s + kKvTile * D + 2 * pr);
        const float x = state_weight(v[0], top);
        l += v[0] == -INFINITY ? v[1] : v[1] * x;
        acc += *(const f4*)(s + pr * D + d) * x;
      }
    }
    if (ways > 1) {
      sum[tid] = acc;
      lsum[tid] = l;
      __syncthreads();
      if (way == 0)
        for (uint32_t j = 1; j < ways; ++j) {
          acc += sum[j * items + i];
          l += lsum[j * items + i];
        }
    }
    if (on && way == 0)
      store_out(t, tile.r0 + (tile.first + pr) / t.group, (kvh * t.group + (tile.first + pr) % t.group) * D + d, acc, l);
  }
}

KvAttnPlan kv8_attention_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                              uint32_t ld_table, uint32_t max_tokens, uint32_t cus) {
  KvAttnPlan p;
  const uint32_t group = heads / kv_heads;
  const uint64_t slots = (uint64_t)rows * group / kKvTile + seqs;
  p.slots = (uint32_t)slots;
  const uint64_t pages = std::min<uint64_t>(((uint64_t)max_tokens + kKvPage - 1) / kKvPage, ld_table);
  if (pages <= 16 || slots > kKvMaxSlots || slots * (ld_table + 1ull) > UINT32_MAX) return p;
  p.runs = std::max<uint32_t>(1, cus / kv_heads);
  p.ws_bytes = ((uint64_t)kv_heads * p.runs * 2 * (kKvTile * (head_dim + 2)) + kKvMaxSlots + 1) * sizeof(float);
  return p;
}

namespace {
template <int D>
hipError_t attention_dim(const KvArgs& a, bool int8, const AttnArgs& t, hipStream_t s) {
  const dim3 grid(a.kv_heads * (t.runs ? t.runs : t.slots));
  if (int8)
    hipLaunchKernelGGL((kv8_attention_kernel<D, true>), grid, dim3(512), 0, s, a, t);
  else
    hipLaunchKernelGGL((kv8_attention_kernel<D, false>), grid, dim3(512), 0, s, a, t);
  if (t.runs) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv8_combine_kernel<D>), dim3(a.kv_heads * t.slots), dim3(512), 0, s, a, t);
  }
  return hipGetLastError();
}
}  // namespace

hipError_t launch_kv8_attention(const KvArgs& a, uint32_t head_dim, bool int8, const _Float16* q, uint32_t ldq,
                                uint32_t heads, float scale, const float* gate, uint32_t ldg, _Float16* y,
                                uint32_t ldy, float* ws, const KvAttnPlan& p, hipStream_t s) {
  if (a.rows == 0 || a.seqs == 0) return hipSuccess;
  if (p.runs && (!ws || p.slots > kKvMaxSlots)) return hipErrorInvalidValue;
  const AttnArgs t{q, gate, y, ws, ldq, ldg, ldy, heads, heads / a.kv_heads, p.slots, p.runs, scale};
  if (head_dim == 64) return attention_dim<64>(a, int8, t, s);
  if (head_dim == 128) return attention_dim<128>(a, int8, t, s);
  return attention_dim<256>(a, int8, t, s);
}

}  // namespace dh
