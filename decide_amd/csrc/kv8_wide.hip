// Attention over the 8-bit paged cache where many rows share their tokens (prompts, long follow-ups), for gfx950 MFMA.
//
// kv8_attention_wide_kernel, tiles of 128 (row, head) pairs: eight waves, four groups of 32 pairs x the two halves of a
// page's blocks, on v_mfma_f32_32x32x16_f16.
//   * Pages go into LDS as they are, by DMA, into a ring of four; a wave reads the codes of its half from there and turns
//     them into fp16 in registers, 128 conversions and 32 products of 32 clocks a page.
//   * The same deal of tokens as in kv8_attention_kernel, for two lane groups: lane (r, f), r = lane % 32, f = lane / 32,
//     of half T gets the 16 scores of pair r and block 2 T + f, which are P^T V's operand as they are.
//   * 16-byte chunk x of K's token t lies at chunk x ^ key(t), of V's dim d at x ^ (d / 2 % 4), so that eight lanes
//     that read at once read 128 different bytes' banks.
//   * A page takes 2.1 to 2.5 us with every CU busy (2,040 rows behind 8,192 tokens against 4,096). The two waves of a SIMD
//     have 375 vector instructions each a page (35 more where a row is masked), 4 clocks apart at best and 16 for the 20
//     transcendental ones, 3,500 clocks together, beside 2,048 of products: at 2.4 GHz 1.45 and 0.85 us, overlapped in
//     part. What the rest is was not taken apart. The halves are kept half a page apart, so that one is at its products
//     while the other is at its softmax, and the one at its products has priority.
//   * The two halves meet once, at a tile's end, through LDS: each takes half of the dims.
#include "kv8_attention.h"

namespace dh {

namespace {
typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f16v mfma32(const h8& a, const h8& b, const f16v& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float max_halves(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// token t's swizzle of its D / 16 chunks
template <int D>
__device__ __forceinline__ uint32_t k_key(uint32_t t) {
  if constexpr (D == 256) return (t & 15) ^ (t >> 4 & 1) << 3;
  if constexpr (D == 128) return (t & 3) | (t >> 4 & 1) << 2;
  return (t >> 1 & 1) | (t >> 4 & 1) << 1;
}
// memory that nothing writes while the kernel runs, by a pointer that all lanes share: a scalar read
typedef const __attribute__((address_space(4))) uint32_t* scalar_words;
}  // namespace

template <int D, bool INT8, bool RUNS>
__global__ __launch_bounds__(512) void kv8_attention_wide_kernel(KvArgs a, AttnArgs t) {
  constexpr int C = D / 32;   // pairs of 16-byte chunks of a key
  constexpr int DT = D / 32;  // 32-dim tiles of O
  constexpr uint32_t kBytes = kKvPage * D;  // of a page's K, or V
  constexpr uint32_t kPieces = kBytes / 4096;
  constexpr int kAhead = D == 256 ? 2 : 3;  // LDS reads ahead of their products (registers allow no third)
  // four pages (K, V); at a tile's end the halves' O: [wave][DT / 2 x 4 pieces of 4 dims][64 lanes]
  __shared__ __attribute__((aligned(1024))) char lds[8 * kBytes];
  static_assert(8 * (DT / 2 * 4) * 64 * 16 <= sizeof(lds), "the halves' exchange fits the pages");
  __shared__ __attribute__((aligned(1024))) float scales[4][256];  // of the pages: K's 4, V's 4 (a DMA's room)
  __shared__ f4 meet[8 * 32];  // largest score, sum, V reference of each wave's pairs, and whether they see anything
  __shared__ Deal<RUNS ? kKvWideSlots : 0> deal;
  __shared__ uint32_t seen_most[8];
  const uint32_t kvh = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave & 3, T = wave >> 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t scales0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)scales;
  uint32_t u = 0, u1 = 1;
  if constexpr (RUNS) deal_runs<D, kKvWideTile, kKvWideSlots, 512>(a, t, run, deal, u, u1);
  const uint32_t first_u = u;
  const float c = fabsf(t.scale) * kLog2e;  // a negative scale's sign goes to Q: the largest score is then the largest product
  // What follows from the lane is formed where it is used, again and again: kept over the pages it would spill, and a
  // spill's reload waits for the DMAs.
  auto thread = [] {
    uint32_t x = threadIdx.x;
    asm volatile("" : "+v"(x));
    return x;
  };

  while (u < u1) {
    uint32_t slot = t.slots - 1 - run, tile_u = 0;  // one tile each: the last, longest ones first
    Tile tile;
    if constexpr (RUNS) {
      slot = same(tile_at(deal, t.slots, u));
      tile_u = same(deal.before[slot]);
      const uint32_t q0 = same(deal.seq[slot]);
      if (!tile_of<kKvWideTile>(a, t.group, slot, q0, same(deal.row0[q0]), same(deal.row0[q0 + 1]), tile)) return;
    } else if (!find_tile<kKvWideTile>(a, t.group, slot, tile)) {
      return;
    }
    uint32_t row, head;
    pair_at(t, tile, kvh, min(32 * group + (thread() & 31), tile.pairs - 1), row, head);
    const uint32_t seen = seen_by(a, row);
    const uint32_t wmost = wave_max_u32(seen), wleast = ~wave_max_u32(~seen);
    if ((thread() & 63) == 0) seen_most[wave] = wmost;
    // Q: dims 32 x + 16 f + 8 e .. + 7 of pair r
    h8 q[2 * C];
    {
      const _Float16* qp = t.q + (size_t)row * t.ldq + head * D + 16 * (thread() >> 5 & 1);
#pragma unroll
      for (int x = 0; x < C; ++x) {
        q[2 * x] = *(const h8*)(qp + 32 * x);
        q[2 * x + 1] = *(const h8*)(qp + 32 * x + 8);
      }
      if (t.scale < 0.f) {
#pragma unroll
        for (int x = 0; x < 2 * C; ++x) q[x] = -q[x];
      }
    }
    __syncthreads();
    const uint32_t most =
        __builtin_amdgcn_readfirstlane(max(max(seen_most[0], seen_most[1]), max(seen_most[2], seen_most[3])));
    const uint32_t npages = pages_of(a, most);
    const uint32_t b0 = u - tile_u, b1 = RUNS ? min(npages, u1 - tile_u) : npages;
    if (RUNS && b1 <= b0) return;  // positions that changed under the call
    const bool whole = !RUNS || (b0 == 0 && b1 == npages);
    const scalar_words table = (scalar_words)(a.table + (size_t)tile.seq * a.ld_table);
    auto page_id = [&](uint32_t b) -> uint32_t { return b < a.ld_table ? table[b] : 0xffffffffu; };
    auto record = [&](uint32_t id) { return a.pool + (id < a.pages ? id : 0) * a.page_bytes; };
    // a page's K, V and scales into place `to` (0 .. 3), in kPieces DMAs of 1 KB a wave; the scales by one wave
    auto stage_piece = [&](const uint8_t* rec, uint32_t to, uint32_t i) {
      constexpr uint32_t kRow = D / 16;  // chunks of a token
      const uint32_t lane = thread() & 63, at = (8 * i + wave) * 1024;
      if (at < kBytes) {
        const uint32_t tok = at / D + lane / kRow, x = lane % kRow ^ k_key<D>(tok);
        dma16(lds0 + to * 2 * kBytes + at, tok * D + x * 16, rec + kv_k_at<D>(kvh));
      } else {
        const uint32_t dim = (at - kBytes) / 64 + lane / 4, x = lane % 4 ^ (dim >> 1 & 3);
        dma16(lds0 + to * 2 * kBytes + at, dim * 64 + x * 16, rec + kv_v_at<D>(kvh, a.kv_heads));
      }
    };
    auto stage_scales = [&](const uint8_t* rec, uint32_t to) {
      const uint32_t lane = thread() & 63;
      if (wave == to && lane < 2) dma16(scales0 + to * 1024, lane * 16, rec + kv_scale_at<D>(kvh, a.kv_heads));
    };
    auto stage = [&](uint32_t id, uint32_t to) {
      stage_scales(record(id), to);
#pragma unroll
      for (uint32_t i = 0; i < kPieces; ++i) stage_piece(record(id), to, i);
    };

    // O: o[i] holds dims 32 i' .., i' = i for half 0, i ^ DT / 2 for half 1: what a wave keeps at the end comes first
    f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    float vref = kNoScale;

    auto id_of = [&](uint32_t b) { return b < b1 ? page_id(b) : 0; };
    uint32_t id0 = id_of(b0), id1 = id_of(b0 + 1), id2 = id_of(b0 + 2), id3 = id_of(b0 + 3);  // of pages b .. b + 3
    if (b0 < b1) stage(id0, 0);
    if (b0 + 1 < b1) stage(id1, 1);
    if (b0 + 2 < b1) stage(id2, 2);
    wait_vm<0>();
#pragma unroll
    for (int x = 0; x < 2 * C; ++x) tie(q[x]);  // no wait for Q in the loop: it would wait for the DMAs too
    __syncthreads();
    // One barrier a page. Half 0 meets it before the page's first products, half 1 between the page's softmax and its
    // products with V, a page's work ahead: so of the two waves of a SIMD one is at its products while the other is at its
    // softmax. At barrier b pages up to b + 1 have landed and page b - 1 is done with: behind it page b + 3 is sent for.
    auto meet_at = [&](uint32_t b) {
      if (b + 2 < b1)
        wait_vm<kPieces>();  // all but page b + 2
      else
        wait_vm<0>();
      __syncthreads();
    };
    for (uint32_t b = b0; b < b1; ++b) {
      const uint32_t at = (b - b0) & 3;
      if (T == 0) {
        // Bytes behind the last seen token may be anything, and what stands in for a bad page too.
        if (b * kKvPage + (kKvPage - 1) >= most || id0 >= a.pages) {
          char* const vb = lds + (at * 2 + 1) * kBytes;
          const uint32_t have = id0 >= a.pages ? 0 : most % kKvPage;
          for (uint32_t i = thread(); i < D * 4; i += 256) {
            const uint32_t dim = i / 4, x = i % 4, left = have > 16 * x ? min(have - 16 * x, 16u) : 0;
            u4* const to = (u4*)(vb + dim * 64 + (x ^ (dim >> 1 & 3)) * 16);
            u4 v = *to;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int n = (int)left - 4 * w;
              v[w] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << 8 * n) - 1u;
            }
            *to = v;
          }
        }
        meet_at(b);
        if (b + 3 < b1) stage(id3, (at + 3) & 3);
      }
      const bool on = b * kKvPage + 32 * T < wmost;  // some pair of the wave sees the half
      h8 p[2];
      if (on) {
        const bool bad = id0 >= a.pages;
        const uint32_t lane = thread() & 63, r = lane & 31, f = lane >> 5;
        // the key of row m = 8 x + 4 y + i is token 16 (2 T + y) + 4 x + i
        const uint32_t tok = 16 * (2 * T + (r >> 2 & 1)) + 4 * (r >> 3) + (r & 3);
        const char* const kb = lds + at * 2 * kBytes + tok * D;
        uint32_t sw = (f ^ k_key<D>(tok)) * 16;  // chunk 2 x + f of the token lies at byte 32 x ^ sw
        asm volatile("" : "+v"(sw));             // formed here: hoisted addresses would spill
        __builtin_amdgcn_s_setprio(1);  // the wave at its products goes first: 2,307 causal rows 101 us against 93
        f16v st;
#pragma unroll
        for (int e = 0; e < 16; ++e) st[e] = 0.f;
        // reads run kAhead products ahead; the barriers keep the compiler from moving them to their use
        u4 kf[kAhead + 1];
#pragma unroll
        for (int x = 0; x < (kAhead < C ? kAhead : C); ++x) kf[x] = *(const u4*)(kb + ((32 * x) ^ sw));
#pragma unroll
        for (int x = 0; x < C; ++x) {
          if (x + kAhead < C) kf[(x + kAhead) % (kAhead + 1)] = *(const u4*)(kb + ((32 * (x + kAhead)) ^ sw));
          __builtin_amdgcn_sched_barrier(0);
          const u4 k = kf[x % (kAhead + 1)];
          st = mfma32(numbers<INT8>(k[0], k[1]), q[2 * x], st);
          st = mfma32(numbers<INT8>(k[2], k[3]), q[2 * x + 1], st);
        }
        __builtin_amdgcn_s_setprio(0);
        const float ks = scales[at][2 * T + f];
        float vs = scales[at][4 + 2 * T + f];
        const float cs = c * (bad ? NAN : ks);
        float unit = cs;  // scores are st * unit
        bool blind = false;
        if (b * kKvPage + 32 * T + 31 >= wleast) {  // some pair does not see all of the half
          const uint32_t tok0 = b * kKvPage + 16 * (2 * T + f);  // below 2^32, as seen is
          const uint32_t mine = seen > tok0 ? min(seen - tok0, 16u) : 0;
          mask_scores(st, cs, mine, unit);
          blind = mine == 0;
          if (tok0 >= most || bad) vs = 0.f;
        }
        float top = st[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, st[i]);
        top *= unit;  // of the lane's block
        const float bm = max_halves(top);
        auto share = [&](float ref) { return max_halves(blind ? 0.f : block_share(top, ref, vs)); };
        const float vm = share(m);
        if (__any(moves(bm, m, vm, vref))) {
          const bool mine = moves(bm, m, vm, vref);  // a pair's own: the others of the tile keep their bits
          const float mnew = higher(bm, m) ? bm : m;
          const float alpha = state_weight(m, mnew), vold = alpha * vref;
          const float vnew = mine ? next_reference(vold, share(mnew)) : vref;
          const float both = mine ? vold / vnew : 1.0f;
          l *= alpha;
          m = mnew;
          vref = vnew;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] *= both;
        }
        const float mref = m == -INFINITY ? 0.f : m;
        round_far(st, mref, unit);
        const float ratio = blind ? 0.f : scale_ratio(vs, vref);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float w = __builtin_amdgcn_exp2f(fmaf(st[i], unit, -mref));
          l += w;
          p[i / 8][i % 8] = (_Float16)(w * ratio);
        }
      }
      if (T == 1) meet_at(b);
      if (on) {
        // V: 32 dims on are 2,048 bytes, with the same swizzle
        const uint32_t lane = thread() & 63, r = lane & 31, f = lane >> 5;
        const char* const vt = lds + (at * 2 + 1) * kBytes + r * 64 + ((2 * T + f) ^ (r >> 1 & 3)) * 16;
        const char* const v0 = vt + T * (kBytes / 2);
        const char* const v1 = vt + (1 - T) * (kBytes / 2) - kBytes / 2;
        auto read_v = [&](int i) { return *(const u4*)((i < DT / 2 ? v0 : v1) + 2048 * i); };
        __builtin_amdgcn_s_setprio(1);
        u4 vf[kAhead + 1];
#pragma unroll
        for (int i = 0; i < (kAhead < DT ? kAhead : DT); ++i) vf[i] = read_v(i);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          if (i + kAhead < DT) vf[(i + kAhead) % (kAhead + 1)] = read_v(i + kAhead);
          __builtin_amdgcn_sched_barrier(0);
          const u4 v = vf[i % (kAhead + 1)];
          o[i] = mfma32(numbers<INT8>(v[0], v[1]), p[0], o[i]);
          o[i] = mfma32(numbers<INT8>(v[2], v[3]), p[1], o[i]);
        }
      }
      if (T == 1 && b + 3 < b1) stage(id3, (at + 3) & 3);
      __builtin_amdgcn_s_setprio(0);
      id0 = id1, id1 = id2, id2 = id3, id3 = id_of(b + 4);
    }
    __syncthreads();  // the states go where the pages lie

    // The halves' states meet: each wave keeps its first o's and gives its partner the rest.
    constexpr uint32_t kPer = DT / 2 * 4;  // pieces of four dims that a lane keeps: dims D/2 T + 32 (i / 4) + 8 (i % 4) + 4 f
    const uint32_t lane = thread() & 63, r = lane & 31, f = lane >> 5;
    f4* const xo = (f4*)lds;
    // piece i of lane x: the swizzle spreads one pair's pieces over the banks
    auto piece = [](uint32_t of, uint32_t i, uint32_t x) { return (of * kPer + i) * 64 + (x ^ i); };
    l = sum_halves(l);
    if (f == 0) meet[wave * 32 + r] = f4{m, l, vref, seen ? 1.f : 0.f};
#pragma unroll
    for (int i = 0; i < (int)kPer; ++i) {
      const f16v& v = o[DT / 2 + i / 4];
      const int e = 4 * (i % 4);
      xo[piece(wave, i, lane)] = f4{v[e], v[e + 1], v[e + 2], v[e + 3]};
    }
    // What a lane writes in the end: dims D/2 T + 8 x .. + 7 of pairs first + 64 / kPer k.
    const uint32_t x = lane % kPer, first = 32 * group + lane / kPer, d = T * (D / 2) + 8 * x;
    auto read_gate = [&](uint32_t k, f4* to) {
      pair_at(t, tile, kvh, min(first + 64 / kPer * k, tile.pairs - 1), row, head);
      const f4* const g = (const f4*)(t.gate + (size_t)row * t.ldg + head * D + d);
      to[0] = g[0];
      to[1] = g[1];
    };
    f4 gate[RUNS ? 2 : kPer];
    if (!RUNS && t.gate) {  // while the exchange runs (in runs they would spill)
#pragma unroll
      for (uint32_t k = 0; k < kPer / 2; ++k) read_gate(k, gate + 2 * k);
    }
    __syncthreads();
    {
      const f4 other = meet[(wave ^ 4) * 32 + r];
      const float top = fmaxf(m, other[0]);
      const float wm = state_weight(m, top), wo = state_weight(other[0], top);
      // (a NaN sum stays: a state without a score has weight 0 and, but for NaN, the sum 0)
      const float lt = (m == -INFINITY ? l : l * wm) + (other[0] == -INFINITY ? other[1] : other[1] * wo);
      const float factor = !whole ? 1.0f : seen ? 1.0f / lt : 0.f;
      const float fm = wm * vref * factor, fo = wo * other[2] * factor;
#pragma unroll
      for (int i = 0; i < (int)kPer; ++i) {
        f4& to = xo[piece(wave ^ 4, i, lane)];  // (read by this lane only)
        const f4 po = to;
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(po[e], fo, o[i / 4][4 * (i % 4) + e] * fm);
        to = v;
      }
      if (!whole && T == 0 && f == 0 && 32 * group + r < tile.pairs) {
        float* const state = state_of<D, kKvWideTile>(t, kvh, run, u == first_u ? 0 : 1);
        *(f2*)(state + kKvWideTile * D + 2 * (32 * group + r)) = f2{top, lt};
      }
    }
    // From LDS once more, now eight dims a lane and a pair's half in kPer lanes: gates, results and states in whole lines.
    // Straight from the products' layout, 32 bytes of a line at a time, a tile's end took 11,000 to 29,000 clocks.
    asm volatile("" ::: "memory");  // the wave's own writes, read by its other lanes: LDS keeps a wave's order
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t k = 0; k < kPer / 2; ++k) {
      const uint32_t pair = first + 64 / kPer * k;
      const f4 v0 = xo[piece(wave ^ 4, x, pair % 32)], v1 = xo[piece(wave ^ 4, x, pair % 32 + 32)];
      if (pair >= tile.pairs) continue;
      if (whole) {
        if (RUNS && t.gate) read_gate(k, gate);
        f4 &g0 = gate[RUNS ? 0 : 2 * k], &g1 = gate[RUNS ? 1 : 2 * k + 1];
        if (t.gate && meet[wave * 32 + pair % 32][3] == 0.f) g0 = g1 = f4{0.f, 0.f, 0.f, 0.f};
        pair_at(t, tile, kvh, pair, row, head);
        store_out8(t, row, head * D + d, v0, v1, g0, g1);
      } else {
        float* const to = state_of<D, kKvWideTile>(t, kvh, run, u == first_u ? 0 : 1) + pair * D + d;
        *(f4*)to = v0;
        *(f4*)(to + 4) = v1;
      }
    }
    if constexpr (!RUNS) return;
    __syncthreads();  // the next tile's pages go where the states lay
    u = tile_u + b1;
  }
}

namespace {
template <int D>
void wide_kernels(const KvArgs& a, const AttnArgs& t, bool int8, hipStream_t s) {
  const dim3 grid(a.kv_heads * (t.runs ? t.runs : t.slots));
  auto go = [&](auto i8, auto runs) {
    hipLaunchKernelGGL((kv8_attention_wide_kernel<D, decltype(i8)::value, decltype(runs)::value>), grid, dim3(512), 0, s,
                       a, t);
  };
  auto with = [&](auto i8) {
    if constexpr (D != 64) {
      if (t.runs) return go(i8, std::true_type{});
    }
    go(i8, std::false_type{});
  };
  int8 ? with(std::true_type{}) : with(std::false_type{});
}
}  // namespace

hipError_t launch_kv8_wide(const KvArgs& a, const AttnArgs& t, uint32_t head_dim, bool int8, hipStream_t s) {
  if (head_dim == 64)
    wide_kernels<64>(a, t, int8, s);
  else if (head_dim == 128)
    wide_kernels<128>(a, t, int8, s);
  else
    wide_kernels<256>(a, t, int8, s);
  return hipGetLastError();
}

}  // namespace dh
