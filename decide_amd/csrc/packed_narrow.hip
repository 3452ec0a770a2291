// Causal attention over packed sequences where few rows share their keys (single tokens, short prompts and chunks), for gfx950
// MFMA. The products and their layouts are those of packed_wide.hip.
//
// Tiles of 32 (row, head) pairs of one kv head. The waves of a workgroup share the pairs and deal the keys, 32 of every 32 WAVES
// a wave, each with a ring of its own in LDS and no barrier among them; they meet at a tile's end.
//   * Sequences of one call differ in length by any factor, and the host does not know them. In runs, the workgroups of a kv head
//     add up the steps (of 32 WAVES keys) of all tiles, each for itself, and take equal runs of them, so that long sequences lie
//     over many workgroups and short ones share one. A tile that lies in several runs leaves a state (largest score, sum, O) per
//     run, and packed_merge_kernel merges them in order. Without runs a workgroup takes a tile.
#include <algorithm>

#include "packed_device.h"

namespace dh {

namespace {
constexpr uint32_t kTile = kPackTile;

// How many keys the tile's last pair sees: the most of them.
__device__ __forceinline__ uint32_t tile_most(const PackArgs& a, const PackTile& t) {
  return pack_seen(t, t.row + (t.extra + min(kTile, t.pairs) - 1) / a.group);
}
__device__ __forceinline__ uint32_t share_of(uint32_t total, const PackArgs& a) {
  return max((total + a.runs - 1) / a.runs, a.min_run);
}
// Where a run leaves a tile's state: its first tile's at 0, another's that goes on in the next run at 1.
template <int D>
__device__ __forceinline__ float* state_of(const PackArgs& a, uint32_t kvh, uint32_t run, uint32_t which) {
  return a.ws + ((size_t)(kvh * a.runs + run) * 2 + which) * (kTile * (D + 2));
}
// The steps before each tile, left behind the states for the merge.
template <int D>
__device__ __forceinline__ uint32_t* starts_of(const PackArgs& a) {
  return (uint32_t*)(a.ws + (size_t)a.kv_heads * a.runs * 2 * (kTile * (D + 2)));
}
}  // namespace

template <int D, bool BF16, int WAVES, bool RUNS>
__global__ __launch_bounds__(WAVES * 64, 1) void packed_narrow_kernel(PackArgs a) {
  constexpr uint32_t kRow = 2 * D, kBytes = 32 * kRow;  // of a key, of K (or V) of 32 keys
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kRing = packed_ring(D);
  constexpr int kPieces = kBytes / 1024;
  constexpr uint32_t kChunks = D / 8, kRowsEach = 64 / kChunks, kStep = 32 * WAVES;
  __shared__ __attribute__((aligned(1024))) char lds[WAVES * kRing * 2 * kBytes];
  __shared__ f2 ml[WAVES * 32];
  __shared__ uint32_t before[RUNS ? kPackSlots + 1 : 1], sums[WAVES];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t kvh = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t r = lane & 31, h = lane >> 5;
  auto same = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };

  uint32_t u = 0, u1 = 1;  // steps of the run
  if constexpr (RUNS) {
    constexpr uint32_t kThreads = WAVES * 64;
    for (uint32_t slot = tid; slot < a.slots; slot += kThreads) {
      // (a lane for itself: find_pack_tile asks the whole wave)
      uint32_t lo = 0, hi = a.seqs;
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint64_t)min(a.q0[mid], a.q_rows) * a.group / kTile + mid <= slot)
          lo = mid;
        else
          hi = mid;
      }
      PackTile t;
      const uint32_t begin = min(a.q0[lo], a.q_rows), end = min(a.q0[lo + 1], a.q_rows);
      uint32_t most = 0;
      if ((uint64_t)begin * a.group / kTile + lo <= slot && pack_tile_of<kTile>(a, slot, lo, begin, end, t)) most = tile_most(a, t);
      before[slot] = (most + kStep - 1) / kStep;
    }
    __syncthreads();
    // running sums: each thread some consecutive tiles, then the lanes, then the waves
    const uint32_t per = (a.slots + kThreads - 1) / kThreads, at0 = min(tid * per, a.slots), at1 = min(at0 + per, a.slots);
    uint32_t mine = 0;
    for (uint32_t i = at0; i < at1; ++i) mine += before[i];
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
    for (uint32_t w = 0; w < WAVES; ++w) {
      at += w < wave ? sums[w] : 0;
      total += sums[w];
    }
    for (uint32_t i = at0; i < at1; ++i) {
      const uint32_t n = before[i];
      before[i] = at;
      at += n;
    }
    if (tid == 0) before[a.slots] = total;
    __syncthreads();
    total = same(total);
    if (blockIdx.x == 0)
      for (uint32_t i = tid; i <= a.slots; i += kThreads) starts_of<D>(a)[i] = before[i];
    const uint32_t share = share_of(total, a);
    u = (uint32_t)min((uint64_t)run * share, (uint64_t)total);
    u1 = min(u + share, total);
  }
  const uint32_t first_u = u;

  while (u < u1) {
    uint32_t slot = a.slots - 1 - run, tile_u = 0;  // a tile each: the last, longest ones first
    if constexpr (RUNS) {  // the last tile that starts at or before step u (empty ones start where the next does)
      uint32_t lo = 0, hi = a.slots;
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (before[mid] <= u)
          lo = mid;
        else
          hi = mid;
      }
      slot = same(lo), tile_u = same(before[slot]);
    }
    PackTile tile;
    if (!find_pack_tile<kTile>(a, slot, tile)) return;
    const uint32_t most = tile_most(a, tile), steps = (most + kStep - 1) / kStep;
    const uint32_t s0 = u - tile_u, s1 = RUNS ? min(steps, u1 - tile_u) : steps;
    if (RUNS && s1 <= s0) return;  // (offsets that changed under the call)
    const bool whole = !RUNS || (s0 == 0 && s1 == steps);
    const uint32_t pairs = min(kTile, tile.pairs);
    uint32_t row, head;
    pack_pair(a, tile, kvh, min(r, pairs - 1), row, head);
    const uint32_t seen = pack_seen(tile, row), least = ~max_of_wave(~seen);

    const uint8_t* const kp = (const uint8_t*)(a.k + (size_t)tile.k_begin * a.ldk + kvh * D);
    const uint8_t* const vp = (const uint8_t*)(a.v + (size_t)tile.k_begin * a.ldv + kvh * D);
    // the wave's 32 keys of step s; keys past the sequence's end are its last one again
    auto stage = [&](uint32_t s, bool of_v) {
      const uint32_t first = s * kStep + 32 * wave, last = tile.keys - 1 - first;
      const uint32_t to = lds0 + ((wave * kRing + s % kRing) * 2 + (of_v ? 1 : 0)) * kBytes, ld = of_v ? a.ldv : a.ldk;
      const uint8_t* const base = (of_v ? vp : kp) + (size_t)first * ld * 2;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t t = i * kRowsEach + lane / kChunks;
        const uint32_t chunk = lane % kChunks ^ (of_v ? pack_v_key<D>(t) : pack_k_key<D>(t));
        dma16(to + i * 1024, min(t, last) * ld * 2 + chunk * 16, base);
      }
    };
    auto mine = [&](uint32_t s) { return s < s1 && s * kStep + 32 * wave < most; };  // the wave has keys of the step

    s8 q[KS];
    {
      const uint16_t* const qp = a.q + (size_t)row * a.ldq + head * D + 8 * h;
#pragma unroll
      for (int x = 0; x < KS; ++x) q[x] = *(const s8*)(qp + 16 * x);
    }
#pragma unroll
    for (int i = 0; i < kRing; ++i)
      if (mine(s0 + i)) {
        stage(s0 + i, false);
        stage(s0 + i, true);
      }
    const float c = scale_into<BF16>(q, a.scale);
#pragma unroll
    for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(q[x]));  // no wait for Q in the loop: it would wait for the DMAs too

    f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (uint32_t s = s0; mine(s); ++s) {
      const uint32_t k0 = s * kStep + 32 * wave;
      // Younger than K of step s: its V, and K and V of up to kRing - 1 more steps.
      const bool ahead = kRing > 1 && mine(s + kRing - 1);
      if (ahead)
        wait_vm<(2 * kRing - 1) * kPieces>();
      else if (kRing > 2 && mine(s + 1))
        wait_vm<3 * kPieces>();
      else
        wait_vm<kPieces>();
      const char* const ks = lds + (wave * kRing + s % kRing) * 2 * kBytes;
      f16v st;
#pragma unroll
      for (int e = 0; e < 16; ++e) st[e] = 0.f;
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const s8 k = *(const s8*)(ks + r * kRow + ((32 * x) ^ ((h ^ pack_k_key<D>(r)) * 16)));  // chunk 2 x + h
        st = mfma_16bit<BF16>(k, q[x], st);
      }
      asm volatile("" : "+v"(st));
      if (mine(s + kRing)) {
        wait_lgkm<0>();
        stage(s + kRing, false);
      }
      if (k0 + 31 >= least) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + 4 * h + 8 * (e / 4) + e % 4 >= seen) st[e] = -INFINITY;
      }
      float top = st[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, st[e]);
      top = max_of_halves(top) * c;
      if (__any(top - m > kPackLazy)) {
        const float mnew = top - m > kPackLazy ? top : m;  // a pair's own: the others of the tile keep their bits
        const float alpha = weight_of_state(m, mnew);
        l *= alpha;
        m = mnew;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
      }
      const float mref = m == -INFINITY ? 0.f : m, factor = round_far<1>(&st, c, mref);
      s8 p[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(fmaf(st[8 * x + e], factor, -mref));
          l += w[e];
        }
        p[x] = pack8<BF16>(w);
      }
      // Younger than V of step s: what is behind it.
      if (mine(s + kRing))
        wait_vm<(2 * kRing - 1) * kPieces>();
      else if (kRing > 1 && mine(s + kRing - 1))
        wait_vm<(2 * kRing - 2) * kPieces>();
      else if (kRing > 2 && mine(s + 1))
        wait_vm<2 * kPieces>();
      else
        wait_vm<0>();
      const uint32_t i16 = lane & 15, vrow = 4 * h + i16 / 4;
      const char* const vb = ks + kBytes + vrow * kRow + (i16 & 1) * 8;
      const uint32_t vchunk = 2 * (lane >> 4 & 1) + (i16 >> 1 & 1);
      auto read_v = [&](int d, int x) {
        typedef __attribute__((address_space(3))) s4* lds_s4;
        const char* const vd = vb + d / 4 * 256 + ((4 * (d % 4) + vchunk) ^ pack_v_key<D>(vrow)) * 16 + 16 * x * kRow;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)vd);
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(vd + 8 * kRow));
        return s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      if (k0 + 31 >= least) {  // values that not all pairs see
        char* const at = lds + ((wave * kRing + s % kRing) * 2 + 1) * kBytes + lane * 16;
        if (any_not_finite<BF16, kPieces>(at)) {
          const int ahead = (int)(seen - k0 - 4 * h);  // keys that the lane sees from its first on
          add_infinities<BF16, 2>(o, read_v, [&](int x, int e) { return 16 * x + 8 * (e / 4) + e % 4 < ahead; });
          clear_not_finite<BF16, kPieces>(at);
          asm volatile("" ::: "memory");  // the wave's own keys: LDS keeps its order
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 2; ++x) o[d] = mfma_16bit<BF16>(read_v(d, x), p[x], o[d]);
      if (mine(s + kRing)) {
        wait_lgkm<0>();
        stage(s + kRing, true);
      }
    }

    // The waves meet, 64 dims at a time: each leaves its O relative to the largest of their reference points, four dims of pair r
    // at chunk x ^ r % 16.
    l = sum_of_halves(l);
    if (h == 0) ml[wave * 32 + r] = f2{m, l};
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml[w * 32 + r][0]);
    const float weight = weight_of_state(m, top);
    float* const state = whole ? nullptr : state_of<D>(a, kvh, run, u == first_u ? 0 : 1);
    constexpr uint32_t kItems = kTile * 8 / (WAVES * 64);  // of a thread: eight of a pair's 64 dims
    uint32_t rows[kItems], cols[kItems];
    Gate8 gates[DT / 2][kItems];
#pragma unroll
    for (uint32_t j = 0; j < kItems; ++j) {
      const uint32_t i = tid + j * WAVES * 64;
      pack_pair(a, tile, kvh, min(i / 8, pairs - 1), rows[j], cols[j]);
      cols[j] = cols[j] * D + 8 * (i % 8);
      if (whole && a.gate) {
#pragma unroll
        for (int g = 0; g < DT / 2; ++g) gates[g][j].load(a, rows[j], cols[j] + 64 * g);
      }
    }
#pragma unroll
    for (int g = 0; g < DT / 2; ++g) {
      if (g) __syncthreads();
      char* const to = lds + wave * 8192 + r * 256;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const f16v& v = o[2 * g + x / 4];
        const int e = 4 * (x % 4);
        *(f4*)(to + ((2 * x + h) ^ (r & 15)) * 16) = f4{v[e], v[e + 1], v[e + 2], v[e + 3]} * weight;
      }
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kItems; ++j) {
        const uint32_t i = tid + j * WAVES * 64, pair = i / 8, x = 2 * (i % 8);
        if (pair >= pairs) break;
        float pt = -INFINITY, lt = 0.f;
        f4 v0 = f4{0.f, 0.f, 0.f, 0.f}, v1 = v0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) pt = fmaxf(pt, ml[w * 32 + pair][0]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const f2 s = ml[w * 32 + pair];
          lt += s[0] == -INFINITY ? s[1] : s[1] * __builtin_amdgcn_exp2f(s[0] - pt);  // a NaN sum stays
          const char* const from = lds + w * 8192 + pair * 256;
          v0 += *(const f4*)(from + (x ^ (pair & 15)) * 16);
          v1 += *(const f4*)(from + ((x + 1) ^ (pair & 15)) * 16);
        }
        if (whole) {
          const bool sees = pack_seen(tile, rows[j]) != 0;
          const float inv = sees ? 1.0f / lt : 0.f;
          store_pack8<BF16>(a, rows[j], cols[j] + 64 * g, v0 * inv, v1 * inv, gates[g][j], sees);
        } else {
          const uint32_t dim = 64 * g + 8 * (i % 8);
          *(f4*)(state + pair * D + dim) = v0;
          *(f4*)(state + pair * D + dim + 4) = v1;
          if (dim == 0) *(f2*)(state + kTile * D + 2 * pair) = f2{pt, lt};
        }
      }
    }
    if constexpr (!RUNS) return;
    __syncthreads();  // the next tile's keys go where the states lay
    u = tile_u + s1;
  }
}

// Merges the states of every tile that lies in more than one run, in the runs' order, and writes the rows that see nothing.
// A workgroup takes eight pairs of a tile, D / 8 lanes a pair, and the groups of lanes that a pair has take every so many of its
// states.
template <int D, bool BF16>
__global__ __launch_bounds__(512) void packed_merge_kernel(PackArgs a) {
  constexpr uint32_t kPairs = 8, L = D / 8, kItems = kPairs * L, kWays = 512 / kItems;
  __shared__ f4 acc0[512], acc1[512];
  __shared__ f2 mls[512];
  const uint32_t kvh = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads % (kTile / kPairs),
                 slot = blockIdx.x / a.kv_heads / (kTile / kPairs), tid = threadIdx.x;
  const uint32_t* const before = starts_of<D>(a);
  const uint32_t u0 = before[slot], u1 = before[slot + 1], total = before[a.slots];
  PackTile tile;
  if (!find_pack_tile<kTile>(a, slot, tile) || kPairs * part >= min(kTile, tile.pairs)) return;
  const uint32_t share = share_of(total, a);
  const uint32_t w0 = u0 / share, w1 = u1 > u0 ? (u1 - 1) / share : w0;
  if (u1 > u0 && w0 == w1) return;  // written by the attention kernel itself
  const uint32_t item = tid % kItems, way = tid / kItems, d = 8 * (item % L);
  const uint32_t pr = min(kPairs * part + item / L, tile.pairs - 1);
  uint32_t row, head;
  pack_pair(a, tile, kvh, pr, row, head);
  Gate8 gate;
  if (a.gate) gate.load(a, row, head * D + d);
  f4 v0 = f4{0.f, 0.f, 0.f, 0.f}, v1 = v0;
  float top = -INFINITY, l = 0.f;
  auto add = [&](const f2& s, const f4& o0, const f4& o1) {
    const float both = fmaxf(top, s[0]), x = weight_of_state(top, both), y = weight_of_state(s[0], both);
    l = (top == -INFINITY ? l : l * x) + (s[0] == -INFINITY ? s[1] : s[1] * y);  // a NaN sum stays
    v0 = v0 * x + o0 * y;
    v1 = v1 * x + o1 * y;
    top = both;
  };
  if (u1 > u0) {
#pragma unroll 4
    for (uint32_t w = w0 + way; w <= w1; w += kWays) {
      const float* const s = state_of<D>(a, kvh, w, w == w0 && u0 != w0 * share ? 1 : 0);
      add(*(const f2*)(s + kTile * D + 2 * pr), *(const f4*)(s + pr * D + d), *(const f4*)(s + pr * D + d + 4));
    }
  }
  acc0[tid] = v0, acc1[tid] = v1, mls[tid] = f2{top, l};
  __syncthreads();
  if (way != 0 || kPairs * part + item / L >= tile.pairs) return;
#pragma unroll
  for (uint32_t j = 1; j < kWays; ++j) add(mls[j * kItems + item], acc0[j * kItems + item], acc1[j * kItems + item]);
  const bool sees = pack_seen(tile, row) != 0;
  const float inv = sees ? 1.0f / l : 0.f;
  store_pack8<BF16>(a, row, head * D + d, v0 * inv, v1 * inv, gate, sees);
}

namespace {
template <int D, bool BF16>
hipError_t narrow_kernels(const PackArgs& a, hipStream_t s) {
  constexpr int WAVES = 4;
  if (!a.runs) {
    hipLaunchKernelGGL((packed_narrow_kernel<D, BF16, WAVES, false>), dim3(a.kv_heads * a.slots), dim3(WAVES * 64), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((packed_narrow_kernel<D, BF16, WAVES, true>), dim3(a.kv_heads * a.runs), dim3(WAVES * 64), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((packed_merge_kernel<D, BF16>), dim3(a.kv_heads * a.slots * (kTile / 8)), dim3(512), 0, s, a);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_packed_narrow(const PackArgs& a, uint32_t head_dim, bool bf16, hipStream_t s) {
  if (head_dim == 64) return bf16 ? narrow_kernels<64, true>(a, s) : narrow_kernels<64, false>(a, s);
  if (head_dim == 128) return bf16 ? narrow_kernels<128, true>(a, s) : narrow_kernels<128, false>(a, s);
  return bf16 ? narrow_kernels<256, true>(a, s) : narrow_kernels<256, false>(a, s);
}

// Wide tiles once narrow ones would fill the device more than twice (narrow against wide, us): 32 heads over 8 of 128, 4 x 128
// rows behind 3,000 keys (512 tiles) 67 against 64, 4 x 200 (800 tiles) 120 against 65; 16 over 4 of 256, 1,000 rows (500) 33
// against 42, 1,500 rows (748) 60 against 60, 8 x 200 rows (800) 37 against 16; 8 of 64, 2,000 rows (496) 25 against 29, 3,000
// rows (744) 49 against 41. Where sequences are short a tile's fixed time weighs more, and a narrow one has a CU for itself:
// beyond one for each CU 32 heads over 8 of 128, 400 rows (400) 14.6 against 13.7, 603 rows (600) 23 against 18; of 64, 603 rows
// (600) 16 against 12, 8 of 64, 8 x 200 rows (400) 10.1 against 7.5; but 16 over 4 of 256, 603 rows (300) 22 against 28.
// Narrow tiles of two waves, two of them on a CU, lose: 16 over 4 of 256, 603 rows 26, 8 of 64, 2,000 rows 34.
// Runs, at the price of the deal and the merge, where narrow tiles leave half of the device idle over long sequences: one row, 32
// heads over 8 of 128, 600 keys 10.9 us against 9.9, 4,096 keys 12 against 38; 16 over 4 of 256, 8 rows of up to 1,000 keys 24
// against 21, one of 2,000 17 against 34; 200 rows behind 6,000 keys (100 tiles) 66 against 91; 32 over 8 of 128, 4 x 64 rows
// behind 3,000 keys (256 tiles) 43 against 33. More kv heads than half of the CUs would leave a head one run.
// Single tokens make a tile a sequence, however many pairs it lacks, and the count below (as if sequences shared tiles) takes
// many of them for few tiles and very many for a prompt. Measured, bf16, lengths of up to 4,096, wide | narrow | runs, us (* what
// this takes): 32 heads over 8 of 128, 64 tokens 98 | 89 | 81*, 128 163 | 141* | 148, 256 295 | 270* | 290; 64 over 8, 64 tokens
// 105 | 97* | 93, 256 304 | 281* | 277; 16 over 4 of 256, 64 tokens 159 | 100 | 77*, 256 298 | 273* | 252; 8 over 1 of 64, 256
// 53 | 43 | 40*; 640 tokens of these 68 to 650, the three within 5 %, but for runs of 64 dims (83); 32 over 8 of 128, 288 tokens of
// up to 200 37* | 54 | 88, of up to 1,000 100* | 114 | 156. All of 1,500: 32 over 8 of 128,
// 64 tokens 73 | 73 | 83*, 256 269 | 272* | 301; 16 over 4 of 256, 128 tokens 129 | 136 | 149*. The keys' bytes bound these; the
// choice costs at most 8 % where lengths differ, 15 % where they are all the same, which the host does not know.
PackPlan packed_plan(uint32_t q_rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_k,
                     uint32_t cus) {
  PackPlan p;
  const uint64_t pairs = (uint64_t)q_rows * (heads / kv_heads);
  const uint64_t full = pairs / kPackTile * kv_heads;  // narrow tiles that the rows fill if sequences share them
  p.wide = full >= (head_dim == 128 ? 9ull : 11ull) * cus / 4 || (head_dim < 256 && max_k <= 1024 && full > cus);
  p.slots = (uint32_t)(pairs / (p.wide ? kPackWideTile : kPackTile) + seqs);
  const uint32_t least = head_dim == 256 ? 1024 : head_dim == 128 ? 768 : 1536;
  if (p.wide || p.slots > kPackSlots || max_k < least || full >= cus / 2 || kv_heads > cus / 2) return p;
  p.runs = std::max(1u, cus / kv_heads);
  p.min_run = 2;
  p.ws_bytes = packed_run_bytes(p.runs, p.slots, kv_heads, head_dim);
  return p;
}

uint64_t packed_run_bytes(uint32_t runs, uint32_t slots, uint32_t kv_heads, uint32_t head_dim) {
  return ((uint64_t)kv_heads * runs * 2 * (kTile * (head_dim + 2)) + slots + 1) * sizeof(float);
}

}  // namespace dh
