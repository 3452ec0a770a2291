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
//     subtraction for two). The K scale joins the softmax's factor; the V scale multiplies the weight in fp32 before its
//     rounding to fp16, relative to the largest such product that the pair has met (block_share in kv8_attention.h).
//   * The eight waves of a workgroup take every eighth page and meet at the end of a tile, through LDS.
//   * Sequences of one call may differ in length by any factor, and the host does not know them. So the workgroups of a
//     kv head (one per CU in all) add up the pages of all tiles, each for itself, and take equal runs of them: a run may
//     end one tile and begin another. A tile that lies in several runs leaves a state (largest score, sum, O) per run, and
//     kv8_combine_kernel merges them in order. With pieces of a fixed length instead, sized by the longest sequence, 64
//     sequences of up to 8,192 tokens made 2,560 workgroups, 2,100 of them empty, and took 77 us against 52.
//   * Long sequences: bound by HBM (one row behind 131,072 tokens, 8 heads of 128, 52 us: 5.1 TB/s). Short ones: by the
//     chain of reads row range, position, Q, page number, page, and the waves' merge (603 tokens 12 us, any number of heads).
#include <algorithm>

#include "kv8_attention.h"

namespace dh {

template <int D, bool INT8, bool RUNS>
__global__ __launch_bounds__(512) void kv8_attention_kernel(KvArgs a, AttnArgs t) {
  constexpr int S = D / 64;    // 64-byte quarters of a key: two products each
  constexpr int DT = D / 16;   // 16-dim tiles of O
  constexpr int kPad = D + 4;  // floats of a pair's O in LDS
  constexpr int kWaves = 8;
  __shared__ __attribute__((aligned(16))) float lds[kWaves * kKvTile * kPad];
  __shared__ f2 ml[kWaves * kKvTile];
  __shared__ uint32_t sees[kKvTile];  // how many tokens
  __shared__ Deal<RUNS ? kKvMaxSlots : 0> deal;
  const uint32_t kvh = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = lane & 15, g = lane >> 4;
  uint32_t u = 0, u1 = 1;  // pages of the run
  if constexpr (RUNS) deal_runs<D, kKvTile, kKvMaxSlots, 512>(a, t, run, deal, u, u1);
  const uint32_t first_u = u;
  const float c = fabsf(t.scale) * kLog2e;  // a negative scale's sign goes to Q: the largest score is then the largest product
  const uint32_t ktok = (n >> 2) * 16 + (n & 3);  // this lane's key of a product: token ktok + 4 T

  while (u < u1) {
    uint32_t slot = run, tile_u = 0;
    Tile tile;
    if constexpr (RUNS) {
      slot = same(tile_at(deal, t.slots, u));
      tile_u = same(deal.before[slot]);
      const uint32_t q0 = same(deal.seq[slot]);
      // (it has pages, so it has rows)
      if (!tile_of<kKvTile>(a, t.group, slot, q0, same(deal.row0[q0]), same(deal.row0[q0 + 1]), tile)) return;
    } else if (!find_tile<kKvTile>(a, t.group, slot, tile)) {
      return;
    }
    uint32_t row, head;
    pair_at(t, tile, kvh, min(n, tile.pairs - 1), row, head);
    const uint32_t seen = seen_by(a, row);
    const uint32_t* const table = a.table + (size_t)tile.seq * a.ld_table;
    auto id_of = [&](uint32_t b) { return b < a.ld_table ? table[b] : 0xffffffffu; };
    uint32_t next = id_of(u - tile_u + wave);  // with the position and Q, not behind them; later ids a page ahead

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
    const uint32_t most = wave_max_u32(seen);
    const uint32_t least = ~wave_max_u32(~seen);
    const uint32_t npages = pages_of(a, most);
    const uint32_t b0 = u - tile_u, b1 = RUNS ? min(npages, u1 - tile_u) : npages;
    if (RUNS && b1 <= b0) return;  // positions that changed under the call
    const bool whole = !RUNS || (b0 == 0 && b1 == npages);
    if (t.scale < 0.f) {
#pragma unroll
      for (int j = 0; j < 2 * S; ++j) q[j] = -q[j];
    }
    // the gate of the thread's first four outputs, in flight through the pages
    const uint32_t pairs = min(kKvTile, tile.pairs);
    f4 gate = f4{0.f, 0.f, 0.f, 0.f};
    if (t.gate && whole && tid < pairs * (D / 4)) {
      uint32_t r, h;
      pair_at(t, tile, kvh, tid / (D / 4), r, h);
      gate = *(const f4*)(t.gate + (size_t)r * t.ldg + h * D + 4 * (tid % (D / 4)));
    }
    f4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    float vref = kNoScale;  // what the pair's o is relative to

    for (uint32_t b = b0 + wave; b < b1; b += kWaves) {
      const uint32_t id0 = next;
      next = id_of(b + kWaves);
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
      float unit = cs;  // scores are sv * unit
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = st[i / 4][i % 4];
      float vs = vs0;
      bool blind = false;  // the pair sees nothing of the lane's block
      const uint32_t tok0 = b * kKvPage + 16 * g;  // below 2^32, as seen is
      if (b * kKvPage + (kKvPage - 1) >= least) {  // some pair does not see all of the page
        const uint32_t mine = seen > tok0 ? min(seen - tok0, 16u) : 0;
        mask_scores(sv, cs, mine, unit);
        blind = mine == 0;
        // What none sees may be anything, and so may what stands in for a bad page, for those that do not see it.
        if (tok0 >= most || bad) vs = 0.f;
        if (b * kKvPage + (kKvPage - 1) >= most || bad) {
          const uint32_t have = most > tok0 && !bad ? min(most - tok0, 16u) : 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int left = (int)have - 4 * w;
            const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1u;
#pragma unroll
            for (int i = 0; i < DT; ++i) vc[i][w] &= keep;
          }
        }
      }
      float top = sv[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, sv[i]);
      top *= unit;  // of the lane's block
      const float bm = max_groups(top);
      auto share = [&](float ref) { return max_groups(blind ? 0.f : block_share(top, ref, vs)); };
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
      round_far(sv, mref, unit);
      const float ratio = blind ? 0.f : scale_ratio(vs, vref);
      h8 p[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w = __builtin_amdgcn_exp2f(fmaf(sv[i], unit, -mref));
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
    if (g == 0) ml[wave * kKvTile + n] = f2{m, l};
    if (tid < kKvTile) sees[n] = seen;
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
    float* const state = whole ? nullptr : state_of<D, kKvTile>(t, kvh, run, u == first_u ? 0 : 1);
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
        uint32_t r, h;
        pair_at(t, tile, kvh, pr, r, h);
        if (t.gate && i != tid) gate = *(const f4*)(t.gate + (size_t)r * t.ldg + h * D + d);
        store_out(t, r, h * D + d, acc, lt, sees[pr], gate);
      } else {
        *(f4*)(state + pr * D + d) = acc;
        if (d == 0) *(f2*)(state + kKvTile * D + 2 * pr) = f2{top, lt};
      }
    }
    if constexpr (!RUNS) return;
    __syncthreads();  // the next tile's states go where these lay
    u = tile_u + b1;
  }
}

// Merges the states of every tile that lies in more than one run, in the runs' order, and writes the rows that see
// nothing. A workgroup takes PAIRS pairs of a tile, D / 4 lanes a pair, and the 512 / (PAIRS D / 4) groups of lanes that a
// pair has take every so many of its states, merged as they come: each state is one read behind the others', whatever
// their number.
template <int D, uint32_t TILE, uint32_t PAIRS>
__global__ __launch_bounds__(512) void kv8_combine_kernel(KvArgs a, AttnArgs t) {
  constexpr uint32_t L = D / 4, kParts = TILE / PAIRS, kItems = PAIRS * L, kWays = 512 / kItems;
  static_assert(kItems * kWays == 512 && TILE % PAIRS == 0, "a pair's lanes and ways fill the workgroup");
  __shared__ __attribute__((aligned(16))) f4 sums[512];
  __shared__ f2 mls[512];
  const uint32_t kvh = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads % kParts,
                 slot = blockIdx.x / a.kv_heads / kParts, tid = threadIdx.x;
  const uint32_t* const before = starts_of<D, TILE>(a, t);
  const uint32_t u0 = before[slot], u1 = before[slot + 1], total = before[t.slots];
  Tile tile;
  if (!find_tile<TILE>(a, t.group, slot, tile) || PAIRS * part >= tile.pairs) return;
  const uint32_t share = share_of(total, t);
  const uint32_t w0 = u0 / share, w1 = u1 > u0 ? (u1 - 1) / share : w0;
  if (u1 > u0 && w0 == w1) return;  // written by the attention kernel itself
  const uint32_t item = tid % kItems, way = tid / kItems, d = 4 * (item % L);
  const uint32_t pr = min(PAIRS * part + item / L, tile.pairs - 1);
  uint32_t r, h;
  pair_at(t, tile, kvh, pr, r, h);
  f4 gate = f4{0.f, 0.f, 0.f, 0.f};
  if (t.gate && way == 0) gate = *(const f4*)(t.gate + (size_t)r * t.ldg + h * D + d);  // with the states, not behind them
  f4 acc = f4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, l = 0.f;
  // N states of a thread on their way at once
  auto merge = [&](uint32_t w, auto count) {
    constexpr int N = decltype(count)::value;
    f4 o[N];
    f2 v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t at = min(w + j * kWays, w1);
      const float* const s = state_of<D, TILE>(t, kvh, at, at == w0 && u0 != w0 * share ? 1 : 0);
      v[j] = *(const f2*)(s + TILE * D + 2 * pr);
      o[j] = *(const f4*)(s + pr * D + d);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (w + j * kWays > w1) v[j] = f2{-INFINITY, 0.f};  // (the last state again: nothing of it)
      const float both = fmaxf(top, v[j][0]), x = state_weight(top, both), y = state_weight(v[j][0], both);
      l = (top == -INFINITY ? l : l * x) + (v[j][0] == -INFINITY ? v[j][1] : v[j][1] * y);  // a NaN sum stays
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(o[j][e], y, acc[e] * x);
      top = both;
    }
  };
  // 8 at once where there are as many, 32 states 7.1 us against 4.8; for 2 each they cost 5.6 against 4.6. Where many tiles
  // are merged, in two ways, registers for 8 would halve the workgroups on a CU: 64 tiles 7.6 against 6.9 with 4.
  constexpr int kMost = kWays > 2 ? 8 : 4;
  if (u1 > u0) {
    if (w1 - w0 < 2 * kWays)
      merge(w0 + way, std::integral_constant<int, 2>{});
    else
      for (uint32_t w = w0 + way; w <= w1; w += kMost * kWays) merge(w, std::integral_constant<int, kMost>{});
  }
  if constexpr (kWays > 1) {
    sums[tid] = acc;
    mls[tid] = f2{top, l};
    __syncthreads();
    if (way != 0) return;
#pragma unroll
    for (uint32_t j = 1; j < kWays; ++j) {
      const f2 v = mls[j * kItems + item];
      const f4 o = sums[j * kItems + item];
      const float both = fmaxf(top, v[0]), x = state_weight(top, both), y = state_weight(v[0], both);
      l = (top == -INFINITY ? l : l * x) + (v[0] == -INFINITY ? v[1] : v[1] * y);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(o[e], y, acc[e] * x);
      top = both;
    }
  }
  if (PAIRS * part + item / L >= tile.pairs) return;
  // (the position only where it matters: beside the states it would cost the merge of 256 rows behind 7,744 tokens 0.7 us)
  store_out(t, r, h * D + d, acc, l, l == 0.f ? seen_by(a, r) : 1u, gate);
}

namespace {
uint64_t least_pages(bool wide, uint32_t head_dim) {
  return wide ? 64 : head_dim == 256 ? 17 : head_dim == 128 ? 25 : 57;
}

// Many rows: tiles of 128 pairs. 16 heads over 4 of 256: 496 causal rows 33 us against 25 with tiles of 16, 603 rows 32
// against 32, 1,000 rows 44 against 54, 8 x 128 rows 46 against 70; 32 over 8 of 128: 256 rows behind 544 tokens 25
// against 18, 496 rows 22 against 26. Heads of 64 dims leave the narrow kernel room for two workgroups a CU: 8 heads over
// one, 1,500 causal rows 30 against 14, 4,000 rows 69 against 54, 8,000 rows 141 against 155, 16 x 512 rows behind 2,000
// tokens 61 against 84. Few rows behind many tokens, where the narrow kernel reads them once for every 16 pairs: 256 rows
// of 4 heads behind 7,744 tokens 72 against 91, 128 rows behind 3,972 tokens 48 against 44.
// More pairs, fewer sequences and more pages only ever turn to wide tiles.
bool wide_tiles(uint64_t pairs, uint32_t seqs, uint32_t kv_heads, uint32_t head_dim, uint64_t pages, uint32_t cus) {
  const uint64_t full = pairs / kKvTile * kv_heads;  // narrow tiles that are surely full
  if (head_dim == 64) return full >= 10ull * cus;
  return full >= 5ull * cus / 2 || (pages >= least_pages(true, head_dim) && pairs >= 512ull * seqs);
}

// Two states for each run, and where each slot's runs start.
uint64_t run_bytes(bool wide, uint64_t runs, uint64_t slots, uint32_t kv_heads, uint32_t head_dim) {
  return (kv_heads * runs * 2 * ((wide ? kKvWideTile : kKvTile) * (head_dim + 2)) + slots + 1) * sizeof(float);
}
}  // namespace

constexpr uint32_t kMinRun = 8;

KvAttnPlan kv8_attention_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                              uint32_t ld_table, uint32_t max_tokens, uint32_t cus) {
  KvAttnPlan p;
  const uint64_t pairs = (uint64_t)rows * (heads / kv_heads);
  const uint64_t pages = std::min<uint64_t>(((uint64_t)max_tokens + kKvPage - 1) / kKvPage, ld_table);
  const uint64_t full = pairs / kKvTile * kv_heads;  // narrow tiles that are surely full
  p.wide = wide_tiles(pairs, seqs, kv_heads, head_dim, pages, cus);
  const uint32_t tile = p.wide ? kKvWideTile : kKvTile;
  const uint64_t slots = pairs / tile + seqs;
  p.slots = (uint32_t)slots;
  // Runs, where whole tiles would leave most CUs idle behind long sequences, at the price of the count of their pages and
  // of the merge. One row, 16 heads over 4 of 256: 1,100 tokens 15.0 us against 17.1 with a workgroup per tile, 8,000
  // tokens 16 against 87; heads of 128: 1,100 tokens 11.9 against 10.3, 2,000 12.1 against 15.6; heads of 64: 3,000
  // tokens 10.6 against 10.2, 8,000 11.1 against 19.8. 1,500 rows in runs: 341 against 95. Wide tiles of 4 heads of 256:
  // 256 rows behind 7,744 tokens 72 against 212, 1,000 rows of 8,000 169 against 214, 1,000 causal rows 95 against 45.
  if (pages < least_pages(p.wide, head_dim) || (p.wide ? slots * kv_heads : full) >= cus ||
      (p.wide && head_dim == 64) || slots > (p.wide ? kKvWideSlots : kKvMaxSlots) ||
      slots * (ld_table + 1ull) > UINT32_MAX - std::max(cus, kMinRun))  // all pages, rounded up to whole runs, in 32 bits
    return p;
  p.runs = std::max<uint32_t>(1, cus / kv_heads);
  p.min_run = p.wide ? 4 : kMinRun;  // a page for each wave; fewer, and the states' share grows
  p.ws_bytes = run_bytes(p.wide, p.runs, p.slots, kv_heads, head_dim);
  return p;
}

// What any call of at most these sizes takes: in runs, wide tiles if such a call may have them.
uint64_t kv8_attention_ws_bytes(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_tokens,
                                uint32_t cus) {
  const uint64_t pages = ((uint64_t)max_tokens + kKvPage - 1) / kKvPage;
  if (pages < least_pages(false, head_dim)) return 0;
  const bool wide = head_dim != 64 && pages >= least_pages(true, head_dim) &&
                    wide_tiles((uint64_t)rows * (heads / kv_heads), 1, kv_heads, head_dim, pages, cus);
  return run_bytes(wide, std::max<uint32_t>(1, cus / kv_heads), kKvMaxSlots, kv_heads, head_dim);
}

namespace {
template <int D>
void narrow_kernels(const KvArgs& a, const AttnArgs& t, bool int8, hipStream_t s) {
  const dim3 grid(a.kv_heads * (t.runs ? t.runs : t.slots));
  auto go = [&](auto i8, auto runs) {
    hipLaunchKernelGGL((kv8_attention_kernel<D, decltype(i8)::value, decltype(runs)::value>), grid, dim3(512), 0, s, a,
                       t);
  };
  auto with = [&](auto i8) { t.runs ? go(i8, std::true_type{}) : go(i8, std::false_type{}); };
  int8 ? with(std::true_type{}) : with(std::false_type{});
}
template <int D>
hipError_t attention_of(const KvArgs& a, const AttnArgs& t, bool int8, bool wide, uint32_t cus, hipStream_t s) {
  if (!wide) narrow_kernels<D>(a, t, int8, s);
  const hipError_t e = wide ? launch_kv8_wide(a, t, D, int8, s) : hipGetLastError();
  if (!t.runs || e != hipSuccess) return e;
  constexpr uint32_t kPairs = 512 / D;  // of a workgroup of the combine: four ways a pair
  if (wide) {
    if constexpr (D != 64)
      hipLaunchKernelGGL((kv8_combine_kernel<D, kKvWideTile, kPairs>),
                         dim3(a.kv_heads * t.slots * (kKvWideTile / kPairs)), dim3(512), 0, s, a, t);
  } else if (a.kv_heads * t.slots * (kKvTile / kPairs) <= 4 * cus)
    hipLaunchKernelGGL((kv8_combine_kernel<D, kKvTile, kPairs>), dim3(a.kv_heads * t.slots * (kKvTile / kPairs)),
                       dim3(512), 0, s, a, t);
  else
    hipLaunchKernelGGL((kv8_combine_kernel<D, kKvTile, 2 * kPairs>), dim3(a.kv_heads * t.slots * (kKvTile / (2 * kPairs))),
                       dim3(512), 0, s, a, t);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_kv8_attention(const KvArgs& a, uint32_t head_dim, bool int8, const _Float16* q, uint32_t ldq,
                                uint32_t heads, float scale, const float* gate, uint32_t ldg, _Float16* y,
                                uint32_t ldy, float* ws, const KvAttnPlan& p, uint32_t cus, hipStream_t s) {
  if (a.rows == 0 || a.seqs == 0) return hipSuccess;
  if (p.runs && (!ws || p.min_run == 0 || (p.wide && head_dim == 64) || p.slots > (p.wide ? kKvWideSlots : kKvMaxSlots))) return hipErrorInvalidValue;
  const uint32_t group = heads / a.kv_heads;
  const AttnArgs t{q,     gate,    y,      ws,        ldq,  ldg, ldy, heads, group, ((1u << 21) + group - 1) / group,
                   p.slots, p.runs, p.min_run, scale};
  if (head_dim == 64) return attention_of<64>(a, t, int8, p.wide, cus, s);
  if (head_dim == 128) return attention_of<128>(a, t, int8, p.wide, cus, s);
  return attention_of<256>(a, t, int8, p.wide, cus, s);
}

}  // namespace dh
