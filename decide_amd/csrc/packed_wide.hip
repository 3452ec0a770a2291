// Causal attention over packed sequences where rows share their keys (prompts, chunks of them), for gfx950 MFMA.
//
//   y[r, h] = softmax_t(scale * q[r, h] . k[t, g]) . v[t, g] (x sigmoid(gate[r, h])),  t < keys - (rows behind r)
//
// Tiles of 32 WAVES (row, head) pairs of one kv head, 32 a wave; keys in blocks of 64, which all waves read from LDS.
//   * Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_32x32x16: lane (r, h), r = lane % 32, h
//     = lane / 32, holds scores of ONE pair r, 16 of every 32 keys: 8 i + 4 h + j, i, j < 4. The largest and the sum of a
//     pair are in its two lanes, and the weights are, as they are, the operand of P^T: eight a lane for 16 keys, 4 h + j and
//     8 + 4 h + j. V's operand is to hold the same keys for each dim: two transposing reads of four rows of V each.
//   * K and V go into LDS by DMA, a ring of NBUF blocks. 16-byte chunk c of K's row t lies at c ^ t % 8: eight lanes that
//     read chunk c of eight rows read different banks. Of V's row at c ^ 4 (t % 4) (64 dims: 4 (t / 2 % 2)): a transposing
//     read takes 64 bytes of each of four rows.
//   * The softmax's reference point moves only where a score exceeds it by 2^8, so O is rarely rescaled.
//   * Keys past the sequence's end are its last one again, masked: another sequence's values are never touched.
#include "packed_device.h"

namespace dh {

template <int D, bool BF16, int WAVES, int NBUF>
__global__ __launch_bounds__(WAVES * 64) void packed_wide_kernel(PackArgs a) {
  constexpr uint32_t kTile = 32 * WAVES, kBlock = 64;
  constexpr uint32_t kRow = 2 * D, kBytes = kBlock * kRow;         // of a key, of a block's K (or V)
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kAhead = 3;             // LDS reads ahead of their products
  constexpr int T = D == 256 ? 1 : 2;  // 32 T keys at a time (registers allow no more)
  constexpr int kPieces = 2 * kBytes / 1024 / WAVES;               // DMAs of a wave for a block
  constexpr uint32_t kChunks = D / 8, kRowsEach = 64 / kChunks;     // 16-byte chunks of a row, rows of a DMA
  __shared__ __attribute__((aligned(1024))) char lds[NBUF * 2 * kBytes];
  static_assert(NBUF * 2 * kBytes >= WAVES * 8192, "the outputs' exchange fits the ring");
  const uint32_t kvh = blockIdx.x % a.kv_heads, slot = a.slots - 1 - blockIdx.x / a.kv_heads;
  PackTile tile;
  if (!find_pack_tile<kTile>(a, slot, tile)) return;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 31, h = lane >> 5;
  uint32_t row, head;
  pack_pair(a, tile, kvh, min(kTile, tile.pairs) - 1, row, head);
  const uint32_t most = pack_seen(tile, row), blocks = (most + kBlock - 1) / kBlock;
  pack_pair(a, tile, kvh, min(32 * wave + r, tile.pairs - 1), row, head);
  const uint32_t seen = pack_seen(tile, row);
  const uint32_t wmost = 32 * wave < tile.pairs ? max_of_wave(seen) : 0, wleast = ~max_of_wave(~seen);

  // Q: dims 16 x + 8 h .. + 7 of pair r
  s8 q[KS];
  {
    const uint16_t* const qp = a.q + (size_t)row * a.ldq + head * D + 8 * h;
#pragma unroll
    for (int x = 0; x < KS; ++x) q[x] = *(const s8*)(qp + 16 * x);
  }
  const float c = scale_into<BF16>(q, a.scale);

  auto k_key = [](uint32_t t) { return t & 7; };
  auto v_key = [](uint32_t t) { return D == 64 ? (t >> 1 & 1) * 4 : (t & 3) * 4; };
  const uint8_t* const kp = (const uint8_t*)(a.k + (size_t)tile.k_begin * a.ldk + kvh * D);
  const uint8_t* const vp = (const uint8_t*)(a.v + (size_t)tile.k_begin * a.ldv + kvh * D);
  // What follows from the lane is formed where it is used: kept over the blocks it would spill, and a spill's reload waits for
  // the DMAs.
  auto lane_again = [] {
    uint32_t x = threadIdx.x;
    asm volatile("" : "+v"(x));
    return x & 63;
  };
  auto stage = [&](uint32_t b) {
    const uint32_t lane = D == 256 ? lane_again() : threadIdx.x & 63;
    const uint32_t to = lds0 + b % NBUF * 2 * kBytes, last = tile.keys - 1 - b * kBlock;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t piece = i * WAVES + wave;
      const bool of_k = piece < kBytes / 1024;
      const uint32_t t = piece % (kBytes / 1024) * kRowsEach + lane / kChunks;
      const uint32_t chunk = lane % kChunks ^ (of_k ? k_key(t) : v_key(t));
      const uint32_t ld = of_k ? a.ldk : a.ldv;
      dma16(to + piece * 1024, min(t, last) * ld * 2 + chunk * 16, (of_k ? kp : vp) + (size_t)b * kBlock * ld * 2);
    }
  };

  f16v o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m = -INFINITY, l = 0.f;

#pragma unroll
  for (uint32_t b = 0; b < NBUF - 1; ++b)
    if (b < blocks) stage(b);
#pragma unroll
  for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(q[x]));  // no wait for Q in the loop: it would wait for the DMAs too
  for (uint32_t b = 0; b < blocks; ++b) {
    if (b + NBUF - 2 < blocks)
      wait_vm<(NBUF - 2) * kPieces>();
    else
      wait_vm<0>();
    __syncthreads();  // block b has landed, and everyone is done with block b - 1
    if (b + NBUF - 1 < blocks) stage(b + NBUF - 1);
    const char* const kb = lds + b % NBUF * 2 * kBytes;
#pragma unroll 1
    for (uint32_t k0 = b * kBlock; k0 < min(wmost, (b + 1) * kBlock); k0 += 32 * T) {
      const char* const ks = kb + k0 % kBlock * kRow;
      f16v st[T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int e = 0; e < 16; ++e) st[t][e] = 0.f;
        auto read_k = [&](int x) { return *(const s8*)(ks + (32 * t + r) * kRow + x / 4 * 128 + (((2 * (x % 4) + h) ^ k_key(r)) * 16)); };
        s8 k[kAhead + 1];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) k[x] = read_k(x);
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          if (x + kAhead < KS) k[(x + kAhead) % (kAhead + 1)] = read_k(x + kAhead);
          if (D == 256) __builtin_amdgcn_sched_barrier(0);
          st[t] = mfma_16bit<BF16>(k[x % (kAhead + 1)], q[x], st[t]);
        }
      }
      if (k0 + (32 * T - 1) >= wleast) {
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
      if (__any(top > m + kPackLazy)) {
        const float mnew = top > m + kPackLazy ? top : m;  // a pair's own: the others of the tile keep their bits
        const float alpha = weight_of_state(m, mnew);
        l *= alpha;
        m = mnew;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
      }
      const float mref = m == -INFINITY ? 0.f : m;
      s8 p[2 * T];
#pragma unroll
      for (int x = 0; x < 2 * T; ++x) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(fmaf(st[x / 2][8 * (x % 2) + e], c, -mref));
          l += w[e];
        }
        p[x] = pack8<BF16>(w);
      }
      // V: rows 16 x + 8 y + 4 h + i / 4 of lane i of 16, which gets four rows of dim 32 d + lane % 32
      const uint32_t i16 = lane & 15, vrow = 4 * h + i16 / 4;
      const char* const vb = ks + kBytes + vrow * kRow + (i16 & 1) * 8;
      const uint32_t vchunk = 2 * (lane >> 4 & 1) + (i16 >> 1 & 1);
      auto read_v = [&](int i) {
        typedef __attribute__((address_space(3))) s4* lds_s4;
        const int d = i / (2 * T);
        const char* const vd = vb + d / 4 * 256 + ((4 * (d % 4) + vchunk) ^ v_key(vrow)) * 16 + 16 * (i % (2 * T)) * kRow;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)vd);
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(vd + 8 * kRow));
        return s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      s8 v[kAhead + 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = read_v(i);
#pragma unroll
      for (int i = 0; i < 2 * T * DT; ++i) {
        if (i + kAhead < 2 * T * DT) v[(i + kAhead) % (kAhead + 1)] = read_v(i + kAhead);
        if (D == 256) __builtin_amdgcn_sched_barrier(0);
        o[i / (2 * T)] = mfma_16bit<BF16>(v[i % (kAhead + 1)], p[i % (2 * T)], o[i / (2 * T)]);
      }
    }
  }
  __syncthreads();  // the outputs go where the blocks lay

  // Through LDS, 64 dims at a time, so that rows are written and gates read in whole lines. Four dims of pair r at chunk x
  // lie at x ^ r % 16.
  l = sum_of_halves(l);
  const float inv = seen ? 1.0f / l : 0.f;  // (a row that sees nothing is zero; one that sees only -infinity is NaN)
  char* const mine = lds + wave * 8192;
#pragma unroll
  for (int g = 0; g < DT / 2; ++g) {
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
      if (32 * wave + pair >= tile.pairs) continue;
      pack_pair(a, tile, kvh, 32 * wave + pair, row, head);
      store_pack8<BF16>(a, row, head * D + 64 * g + 8 * (lane % 8), v0, v1, pack_seen(tile, row) != 0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

namespace {
template <int D, bool BF16>
void wide_kernel(const PackArgs& a, hipStream_t s) {
  constexpr int NBUF = D == 256 ? 2 : D == 128 ? 3 : 4;
  hipLaunchKernelGGL((packed_wide_kernel<D, BF16, 8, NBUF>), dim3(a.kv_heads * a.slots), dim3(512), 0, s, a);
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
