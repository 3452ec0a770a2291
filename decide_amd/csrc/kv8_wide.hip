// Attention over the 8-bit paged cache where many rows share their tokens (prompts, long follow-ups), for gfx950 MFMA.
//
// kv8_attention_wide_kernel, tiles of 128 (row, head) pairs: four waves of 32 pairs, on v_mfma_f32_32x32x16_f16.
//   * The tile's pages go into LDS as they are, by DMA, two buffers; every wave reads all of a page's codes from there
//     and turns them into fp16 in registers. 32 pairs a wave make 64 products of 32 clocks of a page against 64 reads
//     of 16 bytes a lane (1,024 clocks a CU for two workgroups' ... ) and 256 conversions.
//   * The same deal of tokens as in kv8_attention_kernel, for two lane groups: over 32 keys (T = 0, 1) lane (r, f), r = lane % 32, f =
//     lane / 32, gets the 16 scores of pair r and block 2 T + f, which are P^T V's operand as they are.
//   * 16-byte chunk x of K's token t lies at chunk x ^ key(t), of V's dim d at x ^ (d / 2 % 4), so that eight lanes
//     that read at once read 128 different bytes' banks.
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
__global__ __launch_bounds__(256, 2) void kv8_attention_wide_kernel(KvArgs a, AttnArgs t) {
  constexpr int C = D / 32;  // pairs of 16-byte chunks of a key
  constexpr int DT = D / 32;  // 32-dim tiles of O
  constexpr uint32_t kBytes = kKvPage * D;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kBytes];  // two pages of K, two of V
  __shared__ Deal<RUNS ? kKvWideSlots : 0> deal;
  __shared__ __attribute__((aligned(1024))) float scales[2][256];  // of the two pages: K's 4, V's 4 (a DMA's room)
  __shared__ uint32_t seen_most[4];
  const uint32_t kvh = blockIdx.x % a.kv_heads, run = blockIdx.x / a.kv_heads;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t scales0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)scales;
  uint32_t u = 0, u1 = 1;
  if constexpr (RUNS) deal_runs<D, kKvWideTile, kKvWideSlots, 256>(a, t, run, deal, u, u1);
  const uint32_t first_u = u;
  const float c = fabsf(t.scale) * kLog2e;  // a negative scale's sign goes to Q: the largest score is then the largest product

  while (u < u1) {
    // What follows from the lane is formed where it is used, again and again: kept over the pages it would spill, and a
    // spill's reload waits for the DMAs.
    auto thread = [] {
      uint32_t x = threadIdx.x;
      asm volatile("" : "+v"(x));
      return x;
    };
    uint32_t slot = t.slots - 1 - run, tile_u = 0;  // one tile each: the last, longest ones first
    Tile tile;
    if constexpr (RUNS) {
      slot = tile_at(deal, t.slots, u);
      tile_u = deal.before[slot];
      const uint32_t q0 = deal.seq[slot];
      if (!tile_of<kKvWideTile>(a, t.group, slot, q0, deal.row0[q0], deal.row0[q0 + 1], tile)) return;
    } else if (!find_tile<kKvWideTile>(a, t.group, slot, tile)) {
      return;
    }
    uint32_t row, head;
    pair_at(t, tile, kvh, min(32 * wave + (thread() & 31), tile.pairs - 1), row, head);
    const uint32_t seen = seen_by(a, row);
    const uint32_t wmost = wave_max_u32(seen), wleast = ~wave_max_u32(~seen);
    if ((thread() & 63) == 0) seen_most[wave] = wmost;
    // Q: dims 32 c + 16 f + 8 e .. + 7 of pair r
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
    const uint32_t most = __builtin_amdgcn_readfirstlane(max(max(seen_most[0], seen_most[1]), max(seen_most[2], seen_most[3])));
    const uint32_t npages = pages_of(a, most);
    const uint32_t b0 = u - tile_u, b1 = RUNS ? min(npages, u1 - tile_u) : npages;
    if (RUNS && b1 <= b0) return;  // positions that changed under the call
    const bool whole = !RUNS || (b0 == 0 && b1 == npages);
    const scalar_words table = (scalar_words)(a.table + (size_t)tile.seq * a.ld_table);
    auto page_id = [&](uint32_t b) -> uint32_t { return b < a.ld_table ? table[b] : 0xffffffffu; };
    auto record = [&](uint32_t id) { return a.pool + (id < a.pages ? id : 0) * a.page_bytes; };
    // a page's K and V into buffer buf: 1 KB a wave and DMA. The swizzles of the i-th 4 KB are the first's, but for D = 256,
    // where K's odd ones have another bit of the key.
    auto stage = [&](uint32_t id, uint32_t buf) {
      const uint8_t* const kp = record(id) + kv_k_at<D>(kvh);
      const uint8_t* const vp = record(id) + kv_v_at<D>(kvh, a.kv_heads);
      constexpr uint32_t kRow = D / 16;  // chunks of a token
      const uint32_t lane = thread() & 63;
      const uint32_t tok = wave * (1024 / D) + lane / kRow, dim = wave * 16 + lane / 4;
      const uint32_t kx = tok * D + (lane % kRow ^ k_key<D>(tok)) * 16, vx = dim * 64 + (lane % 4 ^ (dim >> 1 & 3)) * 16;
#pragma unroll
      for (uint32_t i = 0; i < kBytes / 4096; ++i) {
        const uint32_t at = i * 4096 + wave * 1024;
        dma16(lds0 + buf * kBytes + at, D == 256 && i % 2 ? kx ^ 128 : kx, kp + i * 4096);
        dma16(lds0 + (2 + buf) * kBytes + at, vx, vp + i * 4096);
      }
      if (wave == 0 && lane < 2) dma16(scales0 + buf * 1024, lane * 16, record(id) + kv_scale_at<D>(kvh, a.kv_heads));
    };

    f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    float vref = 0x1p-100f, inv_vref = 0x1p100f;

    uint32_t id = b0 < b1 ? page_id(b0) : 0;
    if (b0 < b1) stage(id, 0);
    wait_vm<0>();
#pragma unroll
    for (int x = 0; x < 2 * C; ++x) tie(q[x]);  // no wait for Q in the loop: it would wait for the DMAs too
    __syncthreads();
    for (uint32_t b = b0, buf = 0; b < b1; ++b, buf ^= 1) {
      const uint32_t next = b + 1 < b1 ? page_id(b + 1) : 0;
      if (b + 1 < b1) stage(next, buf ^ 1);  // into the buffer every wave left before the last barrier
      const bool bad = id >= a.pages;
      char* const vb = lds + (2 + buf) * kBytes;
      if (b * kKvPage + (kKvPage - 1) >= most) {  // bytes behind the last seen token may be anything
        const uint32_t have = most % kKvPage;
        for (uint32_t i = thread(); i < D * 4; i += 256) {
          const uint32_t dim = i / 4, x = i % 4, left = have > 16 * x ? min(have - 16 * x, 16u) : 0;
          u4* const at = (u4*)(vb + dim * 64 + (x ^ (dim >> 1 & 3)) * 16);
          u4 v = *at;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int n = (int)left - 4 * w;
            v[w] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << 8 * n) - 1u;
          }
          *at = v;
        }
        __syncthreads();
      }
      if (b * kKvPage < wmost) {
#pragma unroll 1
        for (uint32_t T = 0; T < 2; ++T) {
          const uint32_t lane = thread() & 63, r = lane & 31, f = lane >> 5;
          // the key of row m = 8 x + 4 y + i is token 16 (2 T + y) + 4 x + i
          const uint32_t tok = 16 * (2 * T + (r >> 2 & 1)) + 4 * (r >> 3) + (r & 3);
          const char* const kb = lds + buf * kBytes + tok * D;
          uint32_t sw = (f ^ k_key<D>(tok)) * 16;  // chunk 2 x + f of the token lies at byte 32 x ^ sw
          asm volatile("" : "+v"(sw));             // formed here: hoisted addresses would spill
          f16v st;
#pragma unroll
          for (int e = 0; e < 16; ++e) st[e] = 0.f;
          // reads run two ahead of the products; the barriers keep the compiler from moving them to their use
          u4 kf[3];
#pragma unroll
          for (int x = 0; x < 2; ++x) kf[x] = *(const u4*)(kb + ((32 * x) ^ sw));
#pragma unroll
          for (int x = 0; x < C; ++x) {
            if (x + 2 < C) kf[(x + 2) % 3] = *(const u4*)(kb + ((32 * (x + 2)) ^ sw));
            __builtin_amdgcn_sched_barrier(0);
            const u4 k = kf[x % 3];
            st = mfma32(numbers<INT8>(k[0], k[1]), q[2 * x], st);
            st = mfma32(numbers<INT8>(k[2], k[3]), q[2 * x + 1], st);
          }
          const char* const vt = vb + r * 64 + ((2 * T + f) ^ (r >> 1 & 3)) * 16;  // 32 dims on: 2,048 bytes, the same swizzle
          u4 vf[3];
#pragma unroll
          for (int i = 0; i < 2; ++i) vf[i] = *(const u4*)(vt + 2048 * i);
          const float ks = scales[buf][2 * T + f];
          float vs = scales[buf][4 + 2 * T + f];
          const float cs = c * (bad ? NAN : ks);
          float unit = cs;  // scores are st * unit, or st where a mask has scaled them
          bool blind = false;
          if (b * kKvPage + (kKvPage - 1) >= wleast) {  // some pair does not see all of the page
            const uint32_t tok0 = b * kKvPage + 16 * (2 * T + f);  // below 2^32, as seen is
            const uint32_t mine = seen > tok0 ? min(seen - tok0, 16u) : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) st[i] = i < (int)mine ? st[i] * cs : -INFINITY;
            unit = 1.0f;
            blind = mine == 0;
            if (tok0 >= most) vs = 0.f;
          }
          float bm = st[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) bm = fmaxf(bm, st[i]);
          bm = max_halves(bm * unit);
          // the same in every lane: kept in scalar registers
          const float vm = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(max_halves(vs))));
          if (__any(bm > m + kLazy) || vm > vref) {
            const float mnew = bm > m + kLazy ? bm : m;
            const float alpha = state_weight(m, mnew);
            const float vnew = fmaxf(vref, vm);
            l *= alpha;
            m = mnew;
            const float both = alpha * (vref / vnew);
            vref = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(vnew)));
            inv_vref = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(1.0f / vnew)));
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= both;
          }
          const float mref = m == -INFINITY ? 0.f : m;
          const float ratio = blind ? 0.f : vs * inv_vref;
          h8 p[2];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float w = __builtin_amdgcn_exp2f(fmaf(st[i], unit, -mref));
            l += w;
            p[i / 8][i % 8] = (_Float16)(w * ratio);
          }
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            if (i + 2 < DT) vf[(i + 2) % 3] = *(const u4*)(vt + 2048 * (i + 2));
            __builtin_amdgcn_sched_barrier(0);
            const u4 v = vf[i % 3];
            o[i] = mfma32(numbers<INT8>(v[0], v[1]), p[0], o[i]);
            o[i] = mfma32(numbers<INT8>(v[2], v[3]), p[1], o[i]);
          }
        }
      }
      id = next;
      wait_vm<0>();
      __syncthreads();
    }

    l = sum_halves(l);
    const uint32_t r = thread() & 31, f = thread() >> 5 & 1;
    if (32 * wave + r < tile.pairs) {
      if (whole) {
        pair_at(t, tile, kvh, 32 * wave + r, row, head);
        const float factor = over_sum(l) * vref;
        auto store = [&](auto gate) {
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              store_out<decltype(gate)::value>(t, row, head * D + 32 * i + 8 * x + 4 * f,
                                               f4{o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]}, factor);
        };
        if (t.gate)
          store(std::true_type{});
        else
          store(std::false_type{});
      } else {
        float* const state = state_of<D, kKvWideTile>(t, kvh, run, u == first_u ? 0 : 1);
        float* const at = state + (32 * wave + r) * D + 4 * f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *(f4*)(at + 32 * i + 8 * x) =
                f4{o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]} * vref;
        if (f == 0) *(f2*)(state + kKvWideTile * D + 2 * (32 * wave + r)) = f2{m, l};
      }
    }
    if constexpr (!RUNS) return;
    __syncthreads();  // seen_most is written again
    u = tile_u + b1;
  }
}

namespace {
template <int D>
void wide_kernels(const KvArgs& a, const AttnArgs& t, bool int8, hipStream_t s) {
  const dim3 grid(a.kv_heads * (t.runs ? t.runs : t.slots));
  auto go = [&](auto i8, auto runs) {
    hipLaunchKernelGGL((kv8_attention_wide_kernel<D, decltype(i8)::value, decltype(runs)::value>), grid, dim3(256), 0, s,
                       a, t);
  };
  auto with = [&](auto i8) { t.runs ? go(i8, std::true_type{}) : go(i8, std::false_type{}); };
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
