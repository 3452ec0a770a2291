// Matrix product of 8-bit floating point codes with a power-of-two scale for each block of 128, for gfx950 MFMA.
//
//   y[m, n] = epi( sum_b 2^(ex[m, b] + ew[n / 128, b]) sum_{k in block b} x[m, k] w[n, k] )
//
// Two forms, by what y holds:
//   * fp16 outputs: v_mfma_scale_f32_32x32x64_f8f6f4, which takes the scales as operands, the exponent bytes of 32 of W's rows
//     and of 32 of X's rows for 64 columns. Products are exact, but the instruction adds eight neighbours' in a window that
//     ends 13 bits below the largest, cutting what lies lower towards zero; only these sums of eight meet in fp32. Measured
//     against 64 bits: 1.5e-5 of the result (2-norm) on normal operands, 4e-5 where columns differ by a factor of e. Rounding
//     to fp16 costs 2.1e-4.
//   * fp32 outputs: the codes times their scales as bf16, which holds them exactly where the scale's byte is 3 .. 246 (448 x 2^119
//     down to 2^-9 x 2^-124, bf16's smallest), on v_mfma_f32_32x32x16_bf16 at half the rate, whose sums are fp32's: 2e-7. (The
//     8-bit instruction without scales cuts just the same.)
//   * W is the first operand, so that a lane gets one row of y and four columns at a time, in four groups.
//   * K runs in stages of 128 columns, whole cache lines, through a ring of NBUF buffers in LDS, filled by DMA. Each half of a
//     stage is read into registers while the products of the half before it run, so a stage's buffer is free for another
//     when the products of its second half begin: there lies the barrier, one a stage.
//   * Chunk c of 16 bytes of row r lies at c ^ key(r), chosen so that both 8 lanes and 16 that read chunk c of as many rows
//     read different banks. Which of a slice's columns a lane takes as which operand
//     byte does not matter as long as both operands agree.
//   * The words of X's scales of 512 columns and the tile's rows lie in LDS, for up to kSegment columns at a time, and their
//     bytes are read with the slice.
// Measured: 16,384 x 18,432 x 2,560 with SwiGLU 639 us (2,420 TF, the matrix unit busy 66 % of the cycles), 8,192 x 2,560 x 9,216
// with fp32 outputs 308 (1,250 TF, 71 %; a large bf16 product runs at 1,540 to 1,610 TF), 16 x 18,432 x 2,560 10.5 (the weight at
// 4.5 TB/s).
#include <algorithm>
#include <cmath>

#include "fp8.h"
#include "tile_common.h"

namespace dh {

namespace {
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kStage = 128;  // columns (bytes) of a stage
constexpr uint32_t kSegmentWords = 12;
constexpr uint32_t kMostSplits = 16;
constexpr uint32_t kSegment = kSegmentWords * kFp8Word;  // columns whose scales are in LDS at a time

struct Fp8GemmArgs {
  const uint8_t* x;
  const uint8_t* w;
  const uint32_t* sx;
  const uint32_t* sw;
  void* y;
  float* ws;  // partial sums, or null
  uint32_t ldx, ldw, ldsx, ldsw, ldy;
  uint32_t m, n, k, kps, mtiles, ntiles, group, epi;
};

__device__ __forceinline__ f16v mfma_scaled(const i8v& a, const i8v& b, const f16v& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

__device__ __forceinline__ uint32_t row_key(uint32_t row) { return (row & 7) ^ (row >> 3 & 1); }

// As dma16, four bytes a lane.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma4(uint32_t m0, uint32_t voff, const void* sbase) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2 offset:0" ::"s"(m0), "v"(voff), "s"(sbase)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Eight codes times their scale, exactly within bf16's range.
__device__ __forceinline__ b8 widened(uint32_t lo, uint32_t hi, float scale) {
  const b2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false),
                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false),
                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
  return b8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

// Four columns from n on of row `row`, and for SwiGLU (gate v, u to be gated) of half as many columns.
__device__ __forceinline__ void put(const Fp8GemmArgs& a, uint32_t row, uint32_t n, const f4& v) {
  if (a.epi == 1u) {
    _Float16* const to = (_Float16*)a.y + (size_t)row * a.ldy + n;
    if (n + 4 <= a.n) {
      *(h4*)to = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (n + e < a.n) to[e] = (_Float16)v[e];
    }
  } else {
    float* const to = (float*)a.y + (size_t)row * a.ldy + n;
    if (n + 4 <= a.n) {
      *(f4*)to = a.epi == 2u ? *(const f4*)to + v : v;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (n + e < a.n) to[e] = a.epi == 2u ? to[e] + v[e] : v[e];
    }
  }
}
__device__ __forceinline__ void put_swiglu(const Fp8GemmArgs& a, uint32_t row, uint32_t col, const f4& g, const f4& u) {
  h4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (_Float16)swiglu_f(g[e], u[e]);
  *(h4*)((_Float16*)a.y + (size_t)row * a.ldy + col) = v;
}
// 16 bytes of row `row` from output column `col` on: fp32 (0; the partial sums' row where there are splits), fp16 (1, 2: SwiGLU).
template <int K>
__device__ __forceinline__ void put_chunk(const Fp8GemmArgs& a, uint32_t split, uint32_t row, uint32_t col, const u4& v) {
  if constexpr (K == 0) {
    const f4 f = __builtin_bit_cast(f4, v);
    if (a.ws) {
      const uint32_t ldp = (a.n + 3) / 4 * 4;
      if (col < ldp) *(f4*)(a.ws + ((size_t)split * a.m + row) * ldp + col) = f;
    } else if (col < a.n) {
      put(a, row, col, f);
    }
  } else {
    typedef u4 u4_8 __attribute__((aligned(8)));
    const uint32_t cols = K == 1 ? a.n : a.n / 2;
    _Float16* const to = (_Float16*)a.y + (size_t)row * a.ldy + col;
    if (col + 8 <= cols) {
      *(u4_8*)to = v;
    } else {
      const h8 f = __builtin_bit_cast(h8, v);
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        if (col + e < cols) to[e] = f[e];
    }
  }
}
}  // namespace

// A tile of BM of X's rows and BN of W's, waves WM x WN; EXACT: with sums in fp32 alone.
template <bool EXACT, int BM, int BN, int WM, int WN, int NBUF>
__global__ __launch_bounds__(WM * WN * 64, 1) void fp8_gemm_kernel(Fp8GemmArgs a) {
  constexpr int NW = WM * WN;
  constexpr int MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr uint32_t kXBytes = BM * kStage, kBytes = (BM + BN) * kStage;
  constexpr int kPieces = (BM + BN) / 8 / NW;  // DMAs of a wave for a stage
  static_assert((BM + BN) % (8 * NW) == 0 && BN / WN <= 128 && 128 % (BN / WN) == 0, "tile");
  constexpr uint32_t kWBlocks = (BN + 127) / 128;
  // [NBUF][X rows | W rows], X's scale words [kSegmentWords][BM], W's [kSegmentWords][kWBlocks]
  __shared__ __attribute__((aligned(1024))) char lds[NBUF * kBytes + kSegmentWords * 4 * (BM + kWBlocks)];
  uint32_t* const sx = (uint32_t*)(lds + NBUF * kBytes);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wm = wave / WN, wn = wave % WN, r = lane & 31, h = lane >> 5;

  // A DMA fetches 8 rows of 128 bytes, from[i] on, the wave's i-th of X's and then of W's; rows past the end are the last one
  // again. most[i]: how far the last of the eight lies from the first, at most 7 x 2^23 bytes (all the rows behind the first may
  // span more than 2^32).
  constexpr int kXPieces = BM / 8 / NW;
  static_assert(kXPieces * 8 * NW == BM && NW % 2 == 0, "a wave's DMAs are X's or W's as their number says");
  const uint8_t* from[kPieces];
  uint32_t most[kPieces];
  uint32_t m0, n0, split, kbegin, kend;
  auto set_tile = [&](uint32_t id) {
    const uint32_t tiles = a.mtiles * a.ntiles;
    split = id / tiles;
    id -= split * tiles;
    // stripes of `group` column tiles; within a stripe the columns fastest
    const uint32_t stripe = id / (a.mtiles * a.group), at = id - stripe * a.mtiles * a.group;
    const uint32_t wide = min(a.group, a.ntiles - stripe * a.group);
    m0 = at / wide * BM;
    n0 = (stripe * a.group + at % wide) * BN;
    kbegin = split * a.kps, kend = min(a.k, kbegin + a.kps);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const bool of_x = i < kXPieces;
      const uint32_t last = of_x ? a.m - 1 - m0 : a.n - 1 - n0, ld = of_x ? a.ldx : a.ldw;
      const uint32_t first = min(((of_x ? i : i - kXPieces) * NW + wave) * 8, last);
      from[i] = (of_x ? a.x + (size_t)m0 * ld : a.w + (size_t)n0 * ld) + (size_t)first * ld;
      most[i] = min(last - first, 7u) * ld;
    }
  };
  const uint32_t xlane = lane / 8 * a.ldx, wlane = lane / 8 * a.ldw, chunk = ((lane & 7) ^ row_key(8 * wave + lane / 8)) * 16;

  f16v acc[MT][NT];
  struct Frags {
    i8v x[MT], w[NT];
    int ex[MT], ew;  // the scales' bytes
  };
  // chunks 4 q + 2 h and the next of row r of each 32-row tile for half q
  const uint32_t key = row_key(r);
  const uint32_t xrow = (wm * (BM / WM) + r) * kStage, wrow = kXBytes + (wn * (BN / WN) + r) * kStage;
  const uint8_t* const xscale = (const uint8_t*)(sx + wm * (BM / WM) + r);
  const uint8_t* const wscale = (const uint8_t*)(sx + kSegmentWords * BM + wn * (BN / WN) / 128);
  // What half a stage takes to be read, in kReads parts: 16-byte chunks of the operands, then the scales.
  constexpr int kReads = 2 * (MT + NT) + 1;
  auto read_part = [&](Frags& f, uint32_t s, auto half, auto part) {
    constexpr int P = decltype(part)::value, q = decltype(half)::value;
    if constexpr (P < 2 * (MT + NT)) {
      constexpr int at = P / 2 < MT ? P / 2 : P / 2 - MT;
      const char* const p = lds + s % NBUF * kBytes + (P / 2 < MT ? xrow : wrow) + at * 32 * kStage;
      const u4 v = *(const u4*)(p + ((4 * q + 2 * h + P % 2) ^ key) * 16);
      i8v& to = P / 2 < MT ? f.x[at < MT ? at : 0] : f.w[at < NT ? at : 0];
#pragma unroll
      for (int e = 0; e < 4; ++e) to[4 * (P % 2) + e] = (int)v[e];
    } else {
      const uint32_t word = s / 4, byte = s % 4;
#pragma unroll
      for (int i = 0; i < MT; ++i) f.ex[i] = xscale[(word * BM + 32 * i) * 4 + byte];
      f.ew = wscale[word * kWBlocks * 4 + byte];
    }
  };

  auto stage_part = [&](uint32_t k0, uint32_t s, int i) {
    dma16(lds0 + s % NBUF * kBytes + (i * NW + wave) * 1024, min(i < kXPieces ? xlane : wlane, most[i]) + chunk,
          from[i] + k0 + s * kStage);
  };
  // The first stages of the segment from k0 on, and its scale words: four rows of X's a lane, one of W's.
  auto begin = [&](uint32_t k0) {
    const uint32_t k1 = min(kend, k0 + kSegment), stages = (k1 - k0 + kStage - 1) / kStage, word0 = k0 / kFp8Word;
    const uint32_t words = (k1 - k0 + kFp8Word - 1) / kFp8Word;
#pragma unroll
    for (uint32_t s = 0; s < NBUF; ++s)
      if (s < stages) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) stage_part(k0, s, i);
      }
    const uint32_t lane = threadIdx.x & 63, to = lds0 + NBUF * kBytes;
    for (uint32_t i = wave; i * 256 < words * BM; i += NW) {
      const uint32_t x = i * 64 + lane, j = min(x / (BM / 4), words - 1), g = min(x % (BM / 4) * 4, (a.m - 1 - m0) / 4 * 4);
      dma16(__builtin_amdgcn_readfirstlane(to + i * 1024), (j * a.ldsx + g) * 4, a.sx + (size_t)word0 * a.ldsx + m0);
    }
    if (wave == NW - 1 && lane < words * kWBlocks) {
      const uint32_t b = min(n0 / kFp8Block + lane % kWBlocks, (a.n - 1) / kFp8Block);
      dma4(to + kSegmentWords * BM * 4, (lane / kWBlocks * a.ldsw + b) * 4, a.sw + (size_t)word0 * a.ldsw);
    }
  };

  set_tile(xcd_remap(blockIdx.x, gridDim.x));
  if (kbegin < kend) begin(kbegin);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  for (uint32_t k0 = kbegin; k0 < kend; k0 += kSegment) {
    const uint32_t k1 = min(kend, k0 + kSegment), halves = (k1 - k0 + kStage / 2 - 1) / (kStage / 2), stages = (halves + 1) / 2;
    if (k0 != kbegin) begin(k0);
    wait_vm<0>();
    __syncthreads();

    Frags f0, f1;
    static_for<0, kReads>([&](auto part) { read_part(f0, 0, std::integral_constant<int, 0>{}, part); });
    // The products of half q of stage s, from `now`, while the next half comes to `next`.
    // `full`: there is a next half, and a stage to send for.
    auto step = [&](Frags& now, Frags& next, uint32_t s, auto half, auto full) {
      constexpr int q = decltype(half)::value;
      if constexpr (q == 1) {  // stage s + 1 has landed, and everyone has read stage s
        if (decltype(full)::value || s + NBUF - 1 < stages)
          wait_vm<(NBUF - 2) * kPieces>();
        else
          wait_vm<0>();
        wait_lgkm<0>();
        __syncthreads();
      }
      __builtin_amdgcn_s_setprio(q);  // the wave behind the barrier goes first: 241 us against 251 at 8,192 x 8,192 x 5,120
      // The products go first and the DMAs and reads between them: a wave that issued those first would leave the matrix unit
      // idle behind every barrier.
      const bool more = decltype(full)::value || s + NBUF < stages, another = decltype(full)::value || 2 * s + q + 1 < halves;
      constexpr int kItems = q ? kPieces + kReads : kReads, kProducts = MT * NT * (EXACT ? 4 : 1);
      auto items = [&](auto at) {  // what goes behind product `at`
        constexpr int P = decltype(at)::value;
        static_for<P * kItems / kProducts, (P + 1) * kItems / kProducts>([&](auto item) {
          constexpr int I = decltype(item)::value;
          if constexpr (I < kReads) {
            if (another) read_part(next, s + q, std::integral_constant<int, 1 - q>{}, item);
          } else {
            if constexpr (q == 1)
              if (more) stage_part(k0, s + NBUF, I - kReads);
          }
        });
        __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr (EXACT) {
        auto factor = [](int byte) { return __uint_as_float((uint32_t)byte << 23); };
        static_for<0, 4>([&](auto quarter) {
          constexpr int q = decltype(quarter)::value;
          b8 w[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) w[j] = widened(now.w[j][2 * q], now.w[j][2 * q + 1], factor(now.ew));
          static_for<0, MT>([&](auto row) {
            constexpr int i = decltype(row)::value;
            const b8 x = widened(now.x[i][2 * q], now.x[i][2 * q + 1], factor(now.ex[i]));
            static_for<0, NT>([&](auto col) {
              constexpr int j = decltype(col)::value;
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], x, acc[i][j], 0, 0, 0);
              items(std::integral_constant<int, (q * MT + i) * NT + j>{});
            });
          });
        });
      } else {
        static_for<0, MT * NT>([&](auto at) {
          constexpr int i = decltype(at)::value / NT, j = decltype(at)::value % NT;
          acc[i][j] = mfma_scaled(now.w[j], now.x[i], acc[i][j], now.ew, now.ex[i]);
          items(at);
        });
      }
    };
    uint32_t s = 0;
    const std::integral_constant<int, 0> first{};
    const std::integral_constant<int, 1> second{};
    for (; s + NBUF < stages; ++s) {
      step(f0, f1, s, first, std::true_type{});
      step(f1, f0, s, second, std::true_type{});
    }
#pragma unroll 1
    for (; s < stages; ++s) {
      step(f0, f1, s, first, std::false_type{});
      if (2 * s + 1 < halves) step(f1, f0, s, second, std::false_type{});
    }
    __syncthreads();  // the next segment's scales and slices go where these lay
  }

  // Outputs go through LDS and are written in whole lines: as they lie, 16 to 32 bytes of each of 32 rows at a time, they cost
  // 16,384 x 18,432 x 2,560 with SwiGLU 30 us more (700 against 670). kEach rows of each 32-row tile at a time; chunk c of row r at c ^ r.
  constexpr int kEach = MT * WM * 32 * BN * 4 <= (int)(NBUF * kBytes) ? MT : NBUF * kBytes / (WM * 32 * BN * 4);
  static_assert(kEach >= 1 && MT % kEach == 0, "the outputs' exchange fits the ring");
  auto write = [&](auto kind) {  // 0: fp32, 1: fp16, 2: SwiGLU
    constexpr int K = decltype(kind)::value;
    constexpr uint32_t kChunks = BN * (K == 0 ? 4 : K == 1 ? 2 : 1) / 16, kMask = kChunks < 16 ? kChunks - 1 : 15;
    static_for<0, MT / kEach>([&](auto pass) {
      constexpr int p = decltype(pass)::value * kEach;
      if (p) __syncthreads();
#pragma unroll
      for (int i = p; i < p + kEach; ++i) {
        const uint32_t lr = (wm * kEach + i - p) * 32 + r;
        char* const to = lds + lr * (kChunks * 16);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t col = wn * (BN / WN) + 32 * j;  // of the tile
          auto four = [&](int q) { return f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]}; };
          if constexpr (K == 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) *(f4*)(to + ((col / 4 + 2 * q + h) ^ (lr & kMask)) * 16) = four(q);
          } else if constexpr (K == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f4 v = four(q);
              *(h4*)(to + ((col / 8 + q) ^ (lr & kMask)) * 16 + 8 * h) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
            }
          } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const f4 g = four(q), u = four(q + 2);
              h4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = (_Float16)swiglu_f(g[e], u[e]);
              *(h4*)(to + ((col / 16 + q) ^ (lr & kMask)) * 16 + 8 * h) = v;
            }
          }
        }
      }
      __syncthreads();
#pragma unroll 4
      for (uint32_t x = threadIdx.x; x < WM * kEach * 32 * kChunks; x += NW * 64) {
        const uint32_t lr = x / kChunks, c = x % kChunks;
        const uint32_t row = m0 + lr / (32 * kEach) * (BM / WM) + 32 * p + lr % (32 * kEach);
        const u4 v = *(const u4*)(lds + lr * (kChunks * 16) + (c ^ (lr & kMask)) * 16);
        if (row < a.m) put_chunk<K>(a, split, row, K == 0 ? n0 + 4 * c : K == 1 ? n0 + 8 * c : n0 / 2 + 8 * c, v);
      }
    });
  };
  if (EXACT || a.ws)
    write(std::integral_constant<int, 0>{});
  else if (a.epi == 1u)
    write(std::integral_constant<int, 1>{});
  else
    write(std::integral_constant<int, 2>{});
}

// The partial sums in the order of their splits, and the epilogue: four columns a lane.
__global__ __launch_bounds__(256) void fp8_reduce_kernel(Fp8GemmArgs a, uint32_t splits) {
  const uint32_t ldp = (a.n + 3) / 4 * 4, cols = a.epi == 3u ? a.n / 2 : ldp;
  const size_t total = (size_t)a.m * (cols / 4), plane = (size_t)a.m * ldp;
  for (size_t t = (size_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (size_t)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / (cols / 4)), col = (uint32_t)(t % (cols / 4)) * 4;
    auto sum = [&](uint32_t n) {
      const float* p = a.ws + (size_t)row * ldp + n;
      f4 v = *(const f4*)p;
      for (uint32_t s = 1; s < splits; ++s) v += *(const f4*)(p + s * plane);
      return v;
    };
    if (a.epi == 3u) {
      const uint32_t n = col / 16 * 32 + col % 16;
      put_swiglu(a, row, col, sum(n), sum(n + 16));
    } else {
      put(a, row, col, sum(col));
    }
  }
}

namespace {
// fp32 outputs are computed in bf16 (above)
bool exact_sums(uint32_t epi) { return epi == 0u || epi == 2u; }
// The tiles, and what they take, in microseconds: a stage of 128 columns while a CU has one workgroup and while it has as many as
// fit, and what each workgroup takes besides. Measured with every CU busy, or nearly; {fp16 outputs, fp32 outputs}.
struct Variant {
  uint32_t bm, bn, fit;  // fit: workgroups of a CU
  float alone[2], full[2], besides;
};
constexpr Variant kVariants[] = {{256, 256, 1, {1.25f, 0.f}, {1.25f, 0.f}, 7.f},  // fp16 outputs only: the others' registers would not do
                                 {128, 128, 2, {0.60f, 0.87f}, {0.78f, 1.38f}, 3.f},
                                 {64, 128, 2, {0.42f, 0.65f}, {0.62f, 1.00f}, 2.f}};
constexpr int kVariantCount = sizeof(kVariants) / sizeof(kVariants[0]);
template <int BM, int BN, int WM, int WN, int NBUF>
void launch(const Fp8GemmArgs& a, uint32_t grid, hipStream_t s) {
  if (exact_sums(a.epi))
    hipLaunchKernelGGL((fp8_gemm_kernel<true, BM, BN, WM, WN, NBUF>), dim3(grid), dim3(WM * WN * 64), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_gemm_kernel<false, BM, BN, WM, WN, NBUF>), dim3(grid), dim3(WM * WN * 64), 0, s, a);
}
}  // namespace

int fp8_variant_count() { return kVariantCount; }

Fp8Plan fp8_gemm_plan_of(int v, uint32_t splits, uint32_t m, uint32_t n, uint32_t k) {
  auto parts = [](uint32_t x, uint32_t of) { return (uint32_t)(((uint64_t)x + of - 1) / of); };  // (x may end at 2^32 - 1)
  Fp8Plan p;
  p.variant = v;
  p.mtiles = parts(m, kVariants[v].bm);
  p.ntiles = parts(n, kVariants[v].bn);
  const uint32_t words = std::max(1u, parts(k, kFp8Word));  // no columns: one part, of none
  const uint32_t each = parts(words, splits);
  p.kps = each * kFp8Word;
  p.splits = parts(words, each);
  if (p.splits > 1) p.ws_bytes = (uint64_t)p.splits * m * (((uint64_t)n + 3) / 4 * 4) * sizeof(float);
  return p;
}

// The plan of the least estimated time: a launch, rounds of as many workgroups as fit, and where K is divided a second launch that
// reads the partial sums again. The estimates are 5 to 20 % high and rank as measured: 603 x 2,560 x 9,216 with fp32 outputs,
// tiles of 128 x 128 in 5 parts 37 us (43), in 2 parts 42 (46), of 64 x 128 in 2 parts 39 (43), undivided 49 (67).
Fp8Plan fp8_gemm_plan(uint32_t m, uint32_t n, uint32_t k, uint32_t epi, uint32_t cus) {
  const int exact = exact_sums(epi) ? 1 : 0;
  const uint32_t words = (k + kFp8Word - 1) / kFp8Word;
  Fp8Plan best;
  float least = INFINITY;
  for (int v = exact; v < kVariantCount; ++v) {
    const Variant& t = kVariants[v];
    for (uint32_t splits = 1; splits <= std::max(1u, std::min(words, kMostSplits)); ++splits) {
      const Fp8Plan p = fp8_gemm_plan_of(v, splits, m, n, k);
      const uint64_t groups = (uint64_t)p.mtiles * p.ntiles * p.splits;
      if (splits > 1 && (p.splits != splits || groups > (uint64_t)cus * t.fit)) continue;
      const float stage = groups <= cus ? t.alone[exact] : t.full[exact];
      const float rounds = groups <= cus ? 1.f : (float)((groups + cus * t.fit - 1) / (cus * t.fit));
      float time = 4.f + rounds * ((float)std::min(k, p.kps) / kStage * stage + t.besides);
      if (splits > 1) time += 4.f + (float)p.ws_bytes / 3e6f;  // bytes a microsecond, there and back
      if (time < least) least = time, best = p;
    }
  }
  return best;
}

hipError_t launch_fp8_gemm(const Fp8Plan& p, const Fp8& x, const Fp8& w, void* y, uint32_t ldy, uint32_t m, uint32_t n,
                           uint32_t k, uint32_t epi, float* ws, hipStream_t s) {
  if (m == 0 || n == 0) return hipSuccess;
  const Fp8GemmArgs a{x.codes, w.codes, x.scales, w.scales, y,     p.splits > 1 ? ws : nullptr, x.ld, w.ld, x.lds, w.lds, ldy,
                      m,       n,       k,        p.kps,    p.mtiles, p.ntiles, std::min(4u, p.ntiles), epi};
  const uint32_t grid = p.mtiles * p.ntiles * p.splits;
  if (p.variant == 0)
    hipLaunchKernelGGL((fp8_gemm_kernel<false, 256, 256, 2, 4, 2>), dim3(grid), dim3(512), 0, s, a);
  else if (p.variant == 1)
    launch<128, 128, 2, 2, 2>(a, grid, s);
  else
    launch<64, 128, 1, 4, 3>(a, grid, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const size_t total = (size_t)m * ((epi == 3u ? n / 2 : (n + 3) / 4 * 4) / 4);
  hipLaunchKernelGGL(fp8_reduce_kernel, dim3((uint32_t)std::min<size_t>((total + 255) / 256, 16384)), dim3(256), 0, s, a,
                     p.splits);
  return hipGetLastError();
}

}  // namespace dh
