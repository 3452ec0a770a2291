// Attention over the 8-bit paged cache, for gfx950 MFMA:
//   y[r, h] = softmax_t(scale * q[r, h] . K[t]) . V[t] (x sigmoid(gate)), tokens t = 0 ..= qpos[r] of the row's sequence.
//
// kv8_attention_kernel, 16 (row, head) pairs of one kv head a tile:
//   * Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_16x16x32_f16: lane (n, g), n = lane
//     % 16, g = lane / 16, holds scores of ONE pair n. The key rows that a product takes are dealt so that over a page
//     (64 tokens, four products) lane group g gets the 16 scores of the page's block g: one K scale and one V scale a
//     lane, and the scores are, in order, the operand that P^T V needs when the products run over tokens 16 g + 8 e + j.
//     V lies transposed in the page, so the other operand's 16 tokens are 16 consecutive bytes. Nothing of K, V, S or P
//     goes through LDS.
//   * Codes become fp16 exactly (e4m3: one conversion for two; int8: a byte next to 0x64 is 1024 + b as fp16, then one
//     subtraction for two). The K scale joins the softmax's factor; the V scale, relative to the largest of the
//     workgroup's pages, multiplies the weight in fp32 before its rounding to fp16, so weights stay at most 2^8 and one
//     page's small scale cannot push another's weights out of fp16's range.
//   * The four waves take every fourth page and meet once at the end, through LDS; long sequences are cut into pieces,
//     a workgroup each, that kv8_combine_kernel merges in order.
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
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// How many tokens row r sees (0 .. 2^32 - 1): its position and those before it; no position wraps to none.
__device__ __forceinline__ uint32_t seen_by(const KvArgs& a, uint32_t r) { return a.qpos[r] + 1u; }

struct Tile {
  uint32_t seq, r0, pairs, first;  // sequence, its first row, its pairs (rows x group), the tile's first pair
};

// Tile `slot` of a kv head: sequences' tiles start at row0 * group / rows + s, which leaves room for all of them.
__device__ __forceinline__ bool find_tile(const KvArgs& a, uint32_t slot, uint32_t group, uint32_t tile_rows, Tile& t) {
  t.seq = kv_find_seq(a.row0, a.seqs, a.rows, slot, group, tile_rows, 1);
  if (t.seq >= a.seqs) return false;
  t.r0 = min(a.row0[t.seq], a.rows);
  const uint32_t r1 = min(a.row0[t.seq + 1], a.rows);
  if (r1 <= t.r0) return false;
  t.pairs = (r1 - t.r0) * group;
  t.first = (slot - (uint32_t)((uint64_t)t.r0 * group / tile_rows) - t.seq) * tile_rows;
  return t.first < t.pairs;
}

struct AttnArgs {
  const _Float16* q;
  const float* gate;  // or null
  _Float16* y;
  float* ws;  // pieces: O [np][rows][heads][D] as weights x values, then (max, sum) [np][rows][heads]
  uint32_t ldq, ldg, ldy, heads, group, tiles, piece, np;
  float scale;
};
}  // namespace

template <int D, bool INT8>
__global__ __launch_bounds__(256) void kv8_attention_kernel(KvArgs a, AttnArgs t) {
  constexpr int S = D / 64;   // 64-byte quarters of a key: two products each
  constexpr int DT = D / 16;  // 16-dim tiles of O
  constexpr int kPad = D + 4; // floats of a pair's O in LDS
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * kPad + 4 * 16 * 2];
  const uint32_t kvh = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads % t.tiles,
                 piece = blockIdx.x / a.kv_heads / t.tiles;
  Tile tile;
  if (!find_tile(a, slot, t.group, 16, tile)) return;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n = lane & 15, g = lane >> 4;
  const uint32_t pair = min(tile.first + n, tile.pairs - 1);
  const uint32_t row = tile.r0 + pair / t.group, head = kvh * t.group + pair % t.group;
  const uint32_t seen = seen_by(a, row);
  const uint32_t most = wave_max_u32(seen);
  const uint32_t least = ~wave_max_u32(~seen);
  const uint32_t npages = (uint32_t)(((uint64_t)most + kKvPage - 1) / kKvPage);
  const uint32_t npieces = min(t.np, max(1u, (npages + t.piece - 1) / t.piece));
  if (piece >= npieces) return;
  const uint32_t b0 = piece * t.piece, b1 = piece + 1 == npieces ? npages : b0 + t.piece;
  const uint32_t* const table = a.table + (size_t)tile.seq * a.ld_table;
  auto page_of = [&](uint32_t b) -> uint32_t { return b < a.ld_table ? table[b] : 0xffffffffu; };

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
  // the largest V scale of the piece's seen blocks, a page per lane
  float vref = 0x1p-100f;
  for (uint32_t b = b0 + lane; b < b1; b += 64) {
    const uint32_t id = page_of(b);
    if (id >= a.pages) continue;
    const f4 vs = *(const f4*)(a.pool + id * a.page_bytes + kv_scale_at<D>(kvh, a.kv_heads) + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((uint64_t)b * kKvPage + i * kKvBlock < most) vref = fmaxf(vref, vs[i]);
  }
  vref = wave_max_f32(vref);
  const float inv_vref = 1.0f / vref;

  f4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const float c = t.scale * kLog2e;
  const uint32_t ktok = (n >> 2) * 16 + (n & 3);  // this lane's key of a product: token ktok + 4 T

  for (uint32_t b = b0 + wave; b < b1; b += 4) {
    const uint32_t id0 = page_of(b);
    const bool bad = id0 >= a.pages;
    const uint8_t* const rec = a.pool + (bad ? 0 : id0) * a.page_bytes;
    const uint8_t* const kp = rec + kv_k_at<D>(kvh) + ktok * D + 16 * g;
    const uint8_t* const vp = rec + kv_v_at<D>(kvh, a.kv_heads) + n * kKvPage + 16 * g;
    const float* const sp = (const float*)(rec + kv_scale_at<D>(kvh, a.kv_heads));
    const float ks = bad ? NAN : sp[g], vs = sp[4 + g];
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
        st[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(kc[T][j][0], kc[T][j][1]), q[2 * j], st[T], 0, 0, 0);
        st[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(numbers<INT8>(kc[T][j][2], kc[T][j][3]), q[2 * j + 1], st[T], 0,
                                                       0, 0);
      }
    }
    float sv[16];
    const float cs = c * ks;
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[i] = st[i / 4][i % 4] * cs;
    float ratio = vs * inv_vref;
    const uint64_t tok0 = (uint64_t)b * kKvPage + 16 * g;
    if ((uint64_t)(b + 1) * kKvPage > least) {  // some pair does not see all of the page
      const uint32_t mine = seen > tok0 ? (uint32_t)min((uint64_t)seen - tok0, (uint64_t)16) : 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = i < (int)mine ? sv[i] : -INFINITY;
      if (mine == 0) ratio = 0.f;  // the scale of a block that is not seen may be anything
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
    if (__any(bm > m + kLazy)) {
      const float mnew = bm > m + kLazy ? bm : m;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
      m = mnew;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= alpha;
    }
    const float mref = m == -INFINITY ? 0.f : m;
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
  l = sum_groups(l);
  f2* const ml = (f2*)(lds + 4 * 16 * kPad);
  if (g == 0) ml[wave * 16 + n] = f2{m, l};
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * 16 + n][0]);
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top) * vref;
#pragma unroll
  for (int i = 0; i < DT; ++i) *(f4*)(lds + (wave * 16 + n) * kPad + 16 * i + 4 * g) = o[i] * mine;
  __syncthreads();
  const uint32_t pairs = min(16u, tile.pairs - tile.first);
  const bool whole = npieces == 1;
  for (uint32_t i = threadIdx.x; i < pairs * (D / 4); i += 256) {
    const uint32_t pr = i / (D / 4), d = 4 * (i % (D / 4));
    const uint32_t r = tile.r0 + (tile.first + pr) / t.group, h = kvh * t.group + (tile.first + pr) % t.group;
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ml[w * 16 + pr][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f2 v = ml[w * 16 + pr];
      lt += v[0] == -INFINITY ? v[1] : v[1] * __builtin_amdgcn_exp2f(v[0] - mt);  // a NaN sum stays
      acc += *(const f4*)(lds + (w * 16 + pr) * kPad + d);
    }
    if (!whole) {
      const size_t at = ((size_t)piece * a.rows + r) * t.heads + h;
      *(f4*)(t.ws + at * D + d) = acc;
      if (d == 0) *(f2*)(t.ws + (size_t)t.np * a.rows * t.heads * D + 2 * at) = f2{mt, lt};
      continue;
    }
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    f4 v = acc * inv;
    if (t.gate) {
      const f4 gt = *(const f4*)(t.gate + (size_t)r * t.ldg + h * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= sigmoid(gt[e]);
    }
    *(h4*)(t.y + (size_t)r * t.ldy + h * D + d) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
}

// Merges the pieces of every tile that has more than one, in their order: a group of D / 4 lanes per (row, head).
template <int D>
__global__ __launch_bounds__(256) void kv8_combine_kernel(KvArgs a, AttnArgs t, uint32_t tile_rows) {
  constexpr uint32_t kPer = 1024 / D;  // pairs of a workgroup
  const uint32_t kvh = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads % t.tiles;
  const uint32_t part = blockIdx.x / a.kv_heads / t.tiles;
  Tile tile;
  if (!find_tile(a, slot, t.group, tile_rows, tile)) return;
  const uint32_t lane = threadIdx.x & 63;
  uint32_t most = 0;
  const uint32_t pairs = min(tile_rows, tile.pairs - tile.first);
  for (uint32_t i = lane; i < pairs; i += 64) most = max(most, seen_by(a, tile.r0 + (tile.first + i) / t.group));
  most = wave_max_u32(most);
  const uint32_t npages = (uint32_t)(((uint64_t)most + kKvPage - 1) / kKvPage);
  const uint32_t npieces = min(t.np, max(1u, (npages + t.piece - 1) / t.piece));
  if (npieces <= 1) return;  // written by the attention kernel itself
  const uint32_t pr = part * kPer + threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
  if (pr >= pairs) return;
  const uint32_t r = tile.r0 + (tile.first + pr) / t.group, h = kvh * t.group + (tile.first + pr) % t.group;
  const size_t at = (size_t)r * t.heads + h, step = (size_t)a.rows * t.heads;
  const f2* const ml = (const f2*)(t.ws + (size_t)t.np * step * D) + at;
  float top = -INFINITY;
  for (uint32_t p = 0; p < npieces; ++p) top = fmaxf(top, ml[p * step][0]);
  f4 acc = f4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (uint32_t p = 0; p < npieces; ++p) {
    const f2 v = ml[p * step];
    const float w = v[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v[0] - top);
    l += v[0] == -INFINITY ? v[1] : v[1] * w;
    acc += *(const f4*)(t.ws + (p * step + at) * D + d) * w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  f4 v = acc * inv;
  if (t.gate) {
    const f4 gt = *(const f4*)(t.gate + (size_t)r * t.ldg + h * D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= sigmoid(gt[e]);
  }
  *(h4*)(t.y + (size_t)r * t.ldy + h * D + d) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

KvAttnPlan kv8_attention_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                              uint32_t max_tokens, uint32_t cus) {
  KvAttnPlan p;
  const uint32_t group = heads / kv_heads;
  p.tile_rows = 16;
  p.tiles = (uint32_t)((uint64_t)rows * group / p.tile_rows + seqs);
  // tiles that hold rows, at least: every sequence that has any has one
  const uint64_t likely = std::max<uint64_t>(1, ((uint64_t)rows * group + p.tile_rows - 1) / p.tile_rows);
  const uint32_t pages = (uint32_t)(((uint64_t)max_tokens + kKvPage - 1) / kKvPage);
  const uint64_t wanted = std::max<uint64_t>(1, 2 * (uint64_t)cus / std::max<uint64_t>(1, likely * kv_heads));
  const uint64_t bytes = (uint64_t)rows * heads * (head_dim + 2) * sizeof(float);  // of one piece
  const uint64_t room = std::max<uint64_t>(1, (256ull << 20) / std::max<uint64_t>(1, bytes));
  const uint64_t np = std::min({wanted, room, (uint64_t)kKvMaxPieces, (uint64_t)std::max(1u, pages / 16)});
  p.piece = std::max<uint32_t>(1, (uint32_t)((pages + np - 1) / np));
  p.np = std::max<uint32_t>(1, (pages + p.piece - 1) / p.piece);
  p.ws_bytes = p.np > 1 ? bytes * p.np : 0;
  return p;
}

namespace {
template <int D>
hipError_t attention_dim(const KvArgs& a, bool int8, const AttnArgs& t, const KvAttnPlan& p, hipStream_t s) {
  const dim3 grid(a.kv_heads * p.tiles * p.np);
  if (int8)
    hipLaunchKernelGGL((kv8_attention_kernel<D, true>), grid, dim3(256), 0, s, a, t);
  else
    hipLaunchKernelGGL((kv8_attention_kernel<D, false>), grid, dim3(256), 0, s, a, t);
  if (p.np > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint32_t parts = (p.tile_rows + 1024 / D - 1) / (1024 / D);
    hipLaunchKernelGGL((kv8_combine_kernel<D>), dim3(a.kv_heads * p.tiles * parts), dim3(256), 0, s, a, t, p.tile_rows);
  }
  return hipGetLastError();
}
}  // namespace

hipError_t launch_kv8_attention(const KvArgs& a, uint32_t head_dim, bool int8, const _Float16* q, uint32_t ldq,
                                uint32_t heads, float scale, const float* gate, uint32_t ldg, _Float16* y,
                                uint32_t ldy, float* ws, const KvAttnPlan& p, hipStream_t s) {
  if (a.rows == 0 || a.seqs == 0) return hipSuccess;
  if (p.np > 1 && !ws) return hipErrorInvalidValue;
  const AttnArgs t{q, gate, y, ws, ldq, ldg, ldy, heads, heads / a.kv_heads, p.tiles, p.piece, p.np, scale};
  if (head_dim == 64) return attention_dim<64>(a, int8, t, p, s);
  if (head_dim == 128) return attention_dim<128>(a, int8, t, p, s);
  return attention_dim<256>(a, int8, t, p, s);
}

}  // namespace dh
