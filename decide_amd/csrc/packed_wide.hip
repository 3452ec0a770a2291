// Causal attention over packed sequences where rows share their keys (prompts, chunks of them), for gfx950 MFMA.
//
//   y[r, h] = softmax_t(scale * q[r, h] . k[t, g]) . v[t, g] (x sigmoid(gate[r, h])),  t < keys - (rows behind r)
//
// Tiles of 128 (row, head) pairs of one kv head, 32 for each of four waves; keys in blocks of 32 T, which all waves read from LDS.
//   * Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_32x32x16: lane (r, h), r = lane % 32, h
//     = lane / 32, holds scores of ONE pair r, 16 of every 32 keys: 8 i + 4 h + j, i, j < 4. The largest and the sum of a
//     pair are in its two lanes, and the weights are, as they are, the operand of P^T: eight a lane for 16 keys, 4 h + j and
//     8 + 4 h + j. V's operand is to hold the same keys for each dim: two transposing reads of four rows of V each.
//   * K and V go into LDS by DMA, two blocks in turn, their chunks swizzled (packed_device.h). Two workgroups share a CU, and so
//     two waves a SIMD, which need not be in step: 8,192 rows of 32 heads over 8 of 128 dims 531 us (1,040 TF); when it took
//     585, eight waves in one workgroup on a ring of four blocks took 611, and with the two of a SIMD kept half a block apart
//     614; three workgroups with blocks of 32 keys 620. Matrix and vector instructions (the softmax) bound it, the matrix unit
//     busy 58 % of the cycles and vector instructions issued in 53 %.
//   * The softmax's reference point moves only where a score exceeds it by 2^8, so O is rarely rescaled.
//   * Of 256 dims, 24 prompts of up to 2,307 rows and 16 heads over 4, 21,864 rows in all, with gates: 375 us; there the bytes of
//     Q, y and the gates alone are 151 us. The matrix unit is busy 38 % of the cycles, and waves wait 32 %; this was not tried
//     with other blocks or tiles.
//   * Keys past the sequence's end are its last one again, masked: another sequence's values are never touched.
#include "packed_device.h"

namespace dh {

template <int D, bool BF16>
__global__ __launch_bounds__(256, 2) void packed_wide_kernel(PackArgs a) {
  constexpr int T = D == 64 ? 4 : D == 128 ? 2 : 1;  // 64 KB of LDS: two workgroups a CU
  constexpr uint32_t kTile = kPackWideTile, kWaves = kTile / 32, kBlock = 32 * T;
  constexpr uint32_t kRow = 2 * D, kBytes = kBlock * kRow;      // of a key, of a block's K (or V)
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kAhead = D == 256 ? 2 : 3;  // LDS reads ahead of their products: as many as registers are left for
  constexpr int kPieces = 2 * kBytes / 1024 / kWaves;           // DMAs of a wave for a block
  constexpr uint32_t kChunks = D / 8, kRowsEach = 64 / kChunks;  // 16-byte chunks of a row, rows of a DMA
  __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * kBytes];
  __shared__ uint32_t odd[kWaves];
  static_assert(2 * 2 * kBytes >= kWaves * 8192, "the outputs' exchange fits the ring");
  const uint32_t kvh = blockIdx.x % a.kv_heads, slot = a.slots - 1 - blockIdx.x / a.kv_heads;
  PackTile tile;
  if (!find_pack_tile<kTile>(a, slot, tile)) return;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 31, h = lane >> 5;
  auto same = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
  uint32_t row, head;
  pack_pair(a, tile, kvh, min(kTile, tile.pairs) - 1, row, head);
  const uint32_t most = pack_seen(tile, row), blocks = (most + kBlock - 1) / kBlock;
  pack_pair(a, tile, kvh, min(32 * wave + r, tile.pairs - 1), row, head);
  const uint32_t seen = pack_seen(tile, row), least = same(pack_seen(tile, tile.row));
  const uint32_t wmost = 32 * wave < tile.pairs ? max_of_wave(seen) : 0, wleast = ~max_of_wave(~seen);

  // Q: dims 16 x + 8 h .. + 7 of pair r
  s8 q[KS];
  {
    const uint16_t* const qp = a.q + (size_t)row * a.ldq + head * D + 8 * h;
#pragma unroll
    for (int x = 0; x < KS; ++x) q[x] = *(const s8*)(qp + 16 * x);
  }
  const float c = scale_into<BF16>(q, a.scale);

  const uint8_t* const kp = (const uint8_t*)(a.k + (size_t)tile.k_begin * a.ldk + kvh * D);
  const uint8_t* const vp = (const uint8_t*)(a.v + (size_t)tile.k_begin * a.ldv + kvh * D);
  // A DMA brings kRowsEach rows, a lane 16 bytes of one: piece p of a block's K (or V) its rows kRowsEach p on. A wave's pieces
  // are 4 apart, which leaves a lane's chunk the same (but for K of 256 dims,
  // where 8 rows on it is the other half's).
  constexpr int kEach = kPieces / 2;  // of K and of V each
  static_assert(kPieces % 2 == 0 && kEach * kWaves * kRowsEach == kBlock, "a wave's DMAs are K's, then V's");
  const uint32_t t0 = wave * kRowsEach + lane / kChunks;
  const uint32_t kchunk = (lane % kChunks ^ pack_k_key<D>(t0)) * 16, vchunk0 = (lane % kChunks ^ pack_v_key<D>(t0)) * 16;
  const uint32_t klane = lane / kChunks * a.ldk * 2, vlane = lane / kChunks * a.ldv * 2;
  auto stage = [&](uint32_t b) {
    const uint32_t to = lds0 + b % 2 * 2 * kBytes, left = tile.keys - b * kBlock;
    auto piece = [&](int i, const uint8_t* from, uint32_t ld, uint32_t row_at, uint32_t chunk) {
      const uint32_t first = (kWaves * (i % kEach) + wave) * kRowsEach, at = to + (i / kEach) * kBytes + (kWaves * (i % kEach) + wave) * 1024;
      const uint8_t* const base = from + (size_t)(b * kBlock) * ld * 2;
      if (left >= kBlock) {
        dma16(at, row_at + chunk, base + (size_t)first * ld * 2);
      } else {  // keys past the end are the last one again
        const uint32_t f = min(first, left - 1);
        dma16(at, min(row_at, (left - 1 - f) * ld * 2) + chunk, base + (size_t)f * ld * 2);
      }
    };
#pragma unroll
    for (int i = 0; i < kEach; ++i) piece(i, kp, a.ldk, klane, D == 256 ? kchunk ^ (i & 1) * 128 : kchunk);
#pragma unroll
    for (int i = kEach; i < kPieces; ++i) piece(i, vp, a.ldv, vlane, vchunk0);
  };

  f16v o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  if (blocks) stage(0);
#pragma unroll
  for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(q[x]));  // no wait for Q in the loop: it would wait for the DMAs too
  for (uint32_t b = 0; b < blocks; ++b) {
    wait_vm<0>();
    __syncthreads();  // block b has landed, and everyone is done with block b - 1
    if (b + 1 < blocks) stage(b + 1);
    const bool on = b * kBlock < wmost;  // some pair of the wave sees the block
    const char* const ks = lds + b % 2 * 2 * kBytes;
    s8 p[2 * T];
    if (on) {
      uint32_t sw = (h ^ pack_k_key<D>(r)) * 16;
      if (D == 256) asm volatile("" : "+v"(sw));  // formed here: the hoisted addresses would spill
      __builtin_amdgcn_s_setprio(1);
      f16v st[T];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[t][e] = 0.f;
      // Chunk 2 x + h of a key lies at byte 32 x ^ sw. Reads run kAhead products ahead; the barriers keep the compiler from
      // moving them to their use.
      auto read_k = [&](int i) { return *(const s8*)(ks + (32 * (i % T) + r) * kRow + ((32 * (i / T)) ^ sw)); };
      s8 k[kAhead + 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) k[i] = read_k(i);
#pragma unroll
      for (int i = 0; i < T * KS; ++i) {
        if (i + kAhead < T * KS) k[(i + kAhead) % (kAhead + 1)] = read_k(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        st[i % T] = mfma_16bit<BF16>(k[i % (kAhead + 1)], q[i / T], st[i % T]);
      }
      __builtin_amdgcn_s_setprio(0);
      const uint32_t k0 = b * kBlock;
      if (k0 + (kBlock - 1) >= wleast) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (k0 + 4 * h + 32 * t + 8 * (e / 4) + e % 4 >= seen) st[t][e] = -INFINITY;
      }
      float top = st[0][0];
#pragma unroll
      for (int e = 1; e < 16 * T; ++e) top = fmaxf(top, st[e / 16][e % 16]);
      top = max_of_halves(top) * c;
      if (__any(top - m > kPackLazy)) {
        const float mnew = top - m > kPackLazy ? top : m;  // a pair's own: the others of the tile keep their bits
        const float alpha = weight_of_state(m, mnew);
        l *= alpha;
        m = mnew;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
      }
      const float mref = m == -INFINITY ? 0.f : m, factor = round_far<T>(st, c, mref);
#pragma unroll
      for (int x = 0; x < 2 * T; ++x) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(fmaf(st[x / 2][8 * (x % 2) + e], factor, -mref));
          l += w[e];
        }
        p[x] = pack8<BF16>(w);
      }
    }
    // V: rows 16 x + 8 y + 4 h + i / 4 of lane i of 16, which gets four rows of dim 32 d + lane % 32
    auto read_v = [&](int i, uint32_t lane) {
      typedef __attribute__((address_space(3))) s4* lds_s4;
      const uint32_t i16 = lane & 15, vrow = 4 * (lane >> 5) + i16 / 4, vchunk = 2 * (lane >> 4 & 1) + (i16 >> 1 & 1);
      const int d = i / (2 * T);
      const char* const vd = ks + kBytes + vrow * kRow + (i16 & 1) * 8 + d / 4 * 256 +
                             ((4 * (d % 4) + vchunk) ^ pack_v_key<D>(vrow)) * 16 + 16 * (i % (2 * T)) * kRow;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)vd);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(vd + 8 * kRow));
      return s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    if (b * kBlock + (kBlock - 1) >= least) {  // values that not all pairs of the tile see: a quarter of them for each wave
      uint32_t here = lane;
      if (D == 256) asm volatile("" : "+v"(here));  // formed here: hoisted addresses and masks would spill
      char* const mine = lds + b % 2 * 2 * kBytes + kBytes + wave * (kBytes / kWaves) + here * 16;
      const bool found = any_not_finite<BF16, kBytes / kWaves / 1024>(mine);
      if (lane == 0) odd[wave] = found;
      wait_lgkm<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (same(odd[0] | odd[1] | odd[2] | odd[3])) {
        if (on) {
          int ahead = (int)(seen - b * kBlock - 4 * (here >> 5));  // keys that the lane sees from its first on
          add_infinities<BF16, 2 * T>(o,
                                      [&](int d, int x) {
                                        if (D == 256) asm volatile("" : "+v"(ahead));
                                        return read_v(2 * T * d + x, here);
                                      },
                                      [&](int x, int e) { return 16 * x + 8 * (e / 4) + e % 4 < ahead; });
        }
        __syncthreads();
        clear_not_finite<BF16, kBytes / kWaves / 1024>(mine);
        __syncthreads();
      }
    }
    if (on) {
      __builtin_amdgcn_s_setprio(1);
      s8 v[kAhead + 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = read_v(i, lane);
#pragma unroll
      for (int i = 0; i < 2 * T * DT; ++i) {
        if (i + kAhead < 2 * T * DT) v[(i + kAhead) % (kAhead + 1)] = read_v(i + kAhead, lane);
        __builtin_amdgcn_sched_barrier(0);
        o[i / (2 * T)] = mfma_16bit<BF16>(v[i % (kAhead + 1)], p[i % (2 * T)], o[i / (2 * T)]);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }
  __syncthreads();  // the outputs go where the blocks lay

  // Through LDS, 64 dims at a time, so that rows are written and gates read in whole lines. Four dims of pair r at chunk x
  // lie at x ^ r % 16.
  // The gates of the next 64 dims are read meanwhile.
  l = sum_of_halves(l);
  const float inv = seen ? 1.0f / l : 0.f;  // (a row that sees nothing is zero; one that sees only -infinity is NaN)
  char* const mine = lds + wave * 8192;
  auto at = [&](int k, uint32_t& row, uint32_t& col) {  // pair 8 k + lane / 8, dims 8 (lane % 8) .. + 7
    const uint32_t pair = 32 * wave + 8 * k + lane / 8;
    pack_pair(a, tile, kvh, min(pair, tile.pairs - 1), row, col);
    col = col * D + 8 * (lane % 8);
    return pair < tile.pairs;
  };
  Gate8 gates[2][4];
  auto read_gates = [&](int g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t row, col;
      if (at(k, row, col)) gates[g % 2][k].load(a, row, col + 64 * g);
    }
  };
  if (a.gate) read_gates(0);
#pragma unroll
  for (int g = 0; g < DT / 2; ++g) {
    if (a.gate && g + 1 < DT / 2) read_gates(g + 1);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const f16v& v = o[2 * g + x / 4];
      const int e = 4 * (x % 4);
      *(f4*)(mine + r * 256 + ((2 * x + h) ^ (r & 15)) * 16) = f4{v[e], v[e + 1], v[e + 2], v[e + 3]} * inv;
    }
    asm volatile("" ::: "memory");  // the wave's own writes, read by its other lanes: LDS keeps a wave's order
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t pair = 8 * k + lane / 8, x = 2 * (lane % 8);
      const f4 v0 = *(const f4*)(mine + pair * 256 + ((x ^ (pair & 15)) * 16));
      const f4 v1 = *(const f4*)(mine + pair * 256 + (((x + 1) ^ (pair & 15)) * 16));
      uint32_t row, col;
      if (at(k, row, col)) store_pack8<BF16>(a, row, col + 64 * g, v0, v1, gates[g % 2][k], pack_seen(tile, row) != 0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

namespace {
template <int D, bool BF16>
void wide_kernel(const PackArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_wide_kernel<D, BF16>), dim3(a.kv_heads * a.slots), dim3(256), 0, s, a);
}
}  // namespace

hipError_t launch_packed_wide(const PackArgs& a, uint32_t head_dim, bool bf16, hipStream_t s) {
  if (head_dim == 64)
    bf16 ? wide_kernel<64, true>(a, s) : wide_kernel<64, false>(a, s);
  else if (head_dim == 128)
    bf16 ? wide_kernel<128, true>(a, s) : wide_kernel<128, false>(a, s);
  else
    bf16 ? wide_kernel<256, true>(a, s) : wide_kernel<256, false>(a, s);
  return hipGetLastError();
}

}  // namespace dh
