// Device helpers of attention over packed sequences: types, tiles of (row, head) pairs, the softmax's steps.
#pragma once

#include "kv8_device.h"
#include "packed.h"

namespace dh {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr float kPackLazy = 8.0f;  // log2 headroom of the softmax's reference point (weights up to 256)
constexpr float kPackLog2e = 1.4426950408889634f;
// A weight is 2^(score c - m) with the product unrounded, while the reference point m is the largest one's rounded: half a step
// of m apart. From |m| = 2^20 on, where that is 2^-4 and grows with m until weights overflow, a pair's products are rounded too,
// so that the largest weighs 2^0 again.
constexpr float kPackFar = 0x1p20f;

// fp16 or bf16, eight to an operand
template <bool BF16>
__device__ __forceinline__ f16v mfma_16bit(const s8& a, const s8& b, const f16v& c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// Rounded to nearest: outputs, and the softmax's weights as the operand of P V, which is what the matrix instruction takes at
// full rate: a weight is off by half a step of its type, as a value of V is, and sums and scores stay fp32. Against 64 bits
// outputs are 2.5e-4 off in fp16 and 2.2e-3 in bf16 (2-norm), rounding them alone 2.1e-4 and 1.7e-3.
template <bool BF16>
__device__ __forceinline__ s8 pack8(const float* v) {
  if constexpr (BF16) {
    b8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)v[i];
    return __builtin_bit_cast(s8, r);
  } else {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)v[i];
    return __builtin_bit_cast(s8, r);
  }
}

// What a scale leaves to be done to Q: a negative one's sign goes to it, so that the largest score is the largest product; and
// so does zero, which would make NaN of a masked score's -infinity. Returns the factor of the exponent, a subnormal one among
// them: bf16's products reach 2^128.
template <bool BF16, int N>
__device__ __forceinline__ float scale_into(s8 (&q)[N], float scale) {
  const float c = fabsf(scale) * kPackLog2e;
  if (scale < 0.f) {
#pragma unroll
    for (int x = 0; x < N; ++x) q[x] ^= (short)0x8000;
  }
  if (c > 0.f) return c;
  constexpr short kExp = BF16 ? 0x7f80 : 0x7c00;
#pragma unroll
  for (int x = 0; x < N; ++x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[x][e] = (q[x][e] & kExp) == kExp ? (short)0x7fff : (short)0;
  }
  return 1.0f;
}

// Chunk c of 16 bytes of K's row t lies at c ^ pack_k_key(t): both 8 lanes and 16 that read chunk c of as many rows read
// different banks. Of V's row at c ^ pack_v_key(t): a transposing read takes 64 bytes of each of four rows.
template <int D>
__device__ __forceinline__ uint32_t pack_k_key(uint32_t t) {
  return D == 64 ? (t & 7) ^ (t >> 3 & 1) : t & 15;
}
template <int D>
__device__ __forceinline__ uint32_t pack_v_key(uint32_t t) {
  return D == 64 ? (t >> 1 & 1) * 4 : (t & 3) * 4;
}
// Combined over the two halves of a wave: lanes r and r + 32 hold one pair's scores.
__device__ __forceinline__ float max_of_halves(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ uint32_t max_of_wave(uint32_t v) {
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
// weight of a state whose reference point is m among those whose largest is top; none where it met no score
__device__ __forceinline__ float weight_of_state(float m, float top) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
}
// For a pair whose reference point is `m`: rounds the products where it lies far out; returns what is left of the factor c.
template <int N>
__device__ __forceinline__ float round_far(f16v* st, float c, float m) {
  if (!__any(fabsf(m) >= kPackFar)) return c;
  const bool far = fabsf(m) >= kPackFar;
  const float f = far ? c : 1.0f;  // (the tile's other pairs keep their bits)
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) st[t][e] *= f;
  return far ? 1.0f : c;
}
__device__ __forceinline__ float sigmoid_of(float x) { return 1.0f / (1.0f + __expf(-x)); }

// Masked weights are zero, and zero times an infinity or NaN is NaN: where some pair does not see all keys of a block, their
// values are looked through first (two VALU operations for two of them), and where one is not finite, infinities are added for the
// pairs that see it and zero takes its place. Infinities are made as products of bfloat16's largest number and the same again,
// which overflow; a NaN is an infinity of either sign.
// Is any of the 16 N bytes of LDS a lane, from `at` on, 1,024 apart, not finite?
template <bool BF16, int N>
__device__ __forceinline__ bool any_not_finite(const char* at) {
  typedef unsigned short u2s __attribute__((ext_vector_type(2)));
  u2s most = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const s8 v = *(const s8*)(at + i * 1024);
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      most = __builtin_elementwise_max(most, u2s{(unsigned short)v[e], (unsigned short)v[e + 1]} & (unsigned short)0x7fff);
    if (i % 4 == 3) asm volatile("" : "+v"(most) : : "memory");
  }
  return __any(max(most[0], most[1]) >= (BF16 ? 0x7f80 : 0x7c00));
}
// Zero in their place.
template <bool BF16, int N>
__device__ __forceinline__ void clear_not_finite(char* at) {
#pragma unroll 1
  for (int i = 0; i < N; ++i) {
    s8 v = *(const s8*)(at + i * 1024);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (v[e] & 0x7fff) >= (BF16 ? 0x7f80 : 0x7c00) ? (short)0 : v[e];
    *(s8*)(at + i * 1024) = v;
  }
}
// The infinities; value(d, x) is V's operand, sees(x, e) whether the lane's pair sees key e of operand x.
template <bool BF16, int X, int DT, class Value, class Sees>
__device__ __forceinline__ void add_infinities(f16v (&o)[DT], Value value, Sees sees) {
  constexpr short kInf = BF16 ? 0x7f80 : 0x7c00, kNegInf = (short)(kInf | 0x8000);
  constexpr short kLargest = 0x7f7f, kNegLargest = (short)0xff7f;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
#pragma unroll
    for (int x = 0; x < X; ++x) {
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        s8 v = value(d, x), w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = (v[e] & 0x7fff) >= kInf && v[e] != (part ? kInf : kNegInf) ? (part ? kNegLargest : kLargest) : (short)0;
          w[e] = sees(x, e) ? kLargest : (short)0;
        }
        o[d] = mfma_16bit<true>(v, w, o[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// Pairs (row, head of the group) of one kv head, row by row, from the tile's first on.
struct PackTile {
  uint32_t seq;
  uint32_t pairs;       // to the sequence's end
  uint32_t row, extra;  // the first pair's row, and its head in the group
  uint32_t q_begin, q_end, k_begin, keys;
};

// Tile `slot` of a kv head: sequence s's tiles start at q0[s] * group / TILE + s, which leaves room for all before it.
template <uint32_t TILE>
__device__ __forceinline__ bool pack_tile_of(const PackArgs& a, uint32_t slot, uint32_t s, uint32_t begin, uint32_t end,
                                             PackTile& t) {
  if (end <= begin) return false;
  const uint32_t pairs = (end - begin) * a.group;
  const uint32_t first = (slot - (uint32_t)((uint64_t)begin * a.group / TILE) - s) * TILE;
  if (first >= pairs) return false;
  const uint32_t kb = min(a.k0[s], a.k_rows), ke = min(a.k0[s + 1], a.k_rows);
  t = PackTile{s, pairs - first, begin + first / a.group, first % a.group, begin, end, kb, ke > kb ? ke - kb : 0};
  return true;
}
template <uint32_t TILE>
__device__ __forceinline__ bool find_pack_tile(const PackArgs& a, uint32_t slot, PackTile& t) {
  uint32_t begin, end;
  const uint32_t s = kv_find_seq(a.q0, a.seqs, a.q_rows, slot, a.group, TILE, 1, begin, end);
  return s < a.seqs && pack_tile_of<TILE>(a, slot, s, begin, end, t);
}
// Row and head of the tile's pair k < 256. For x = extra + k < group + 256, x times the rounded 2^21 / group is off by less
// than x, and x group < 2^21 for groups of at most 1,024: the quotient is exact. (The product stays below 2^32.)
__device__ __forceinline__ void pack_pair(const PackArgs& a, const PackTile& t, uint32_t kvh, uint32_t k, uint32_t& row,
                                          uint32_t& head) {
  const uint32_t x = t.extra + k, q = x * a.group_inv >> 21;
  row = t.row + q;
  head = kvh * a.group + (x - q * a.group);
}
// How many keys a row of the tile's sequence sees: the last row all of them, each before it one less.
__device__ __forceinline__ uint32_t pack_seen(const PackTile& t, uint32_t row) {
  const uint32_t behind = t.q_end - 1 - row;
  return t.keys > behind ? t.keys - behind : 0;
}

// Eight dims of a pair's output, already over its sum, and of its gates, which are read long before they are wanted.
struct Gate8 {
  f4 g0, g1;
  __device__ __forceinline__ void load(const PackArgs& a, uint32_t row, uint32_t col) {
    const f4* const g = (const f4*)(a.gate + (size_t)row * a.ldg + col);
    g0 = g[0], g1 = g[1];
  }
};
template <bool BF16>
__device__ __forceinline__ void store_pack8(const PackArgs& a, uint32_t row, uint32_t col, f4 v0, f4 v1, const Gate8& g,
                                            bool sees) {
  if (a.gate) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (sees) v0[e] *= sigmoid_of(g.g0[e]), v1[e] *= sigmoid_of(g.g1[e]);
    }
  }
  const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
  typedef short s8u __attribute__((ext_vector_type(8), aligned(8)));
  *(s8u*)(a.y + (size_t)row * a.ldy + col) = pack8<BF16>(v);
}

}  // namespace dh
