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
//   * fp32 outputs: the codes times their scales as bf16, which holds them exactly, on v_mfma_f32_32x32x16_bf16 at half the
//     rate, whose sums are fp32's: 2e-7. (The 8-bit instruction without scales cuts just the same.)
//   * W is the first operand, so that a lane gets one row of y and four columns at a time, in four groups.
//   * K runs in slices of 64 columns through a ring of NBUF buffers in LDS, filled by DMA. Slice s is read into registers
//     while the products of slice s - 1 run; then its buffer is free for slice s + NBUF. One barrier a slice.
//   * A slice's row is 64 bytes, four 16-byte chunks; chunk c of row r lies at c ^ (r / 2 % 4), so that eight lanes that read
//     chunk c of eight rows at once read 128 different bytes' banks. Which of a slice's columns a lane takes as which operand
//     byte does not matter as long as both operands agree.
//   * The words of X's scales of 512 columns and the tile's rows lie in LDS, for up to kSegment columns at a time, and their
//     bytes are read with the slice.
#include <algorithm>

#include "fp8.h"
#include "tile_common.h"

namespace dh {

namespace {
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kSlice = 64;  // columns (bytes) of a slice
constexpr uint32_t kSegmentWords = 16;
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

// Eight codes times their scale, exactly.
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
}  // namespace

// A tile of BM of X's rows and BN of W's, waves WM x WN; EXACT: with sums in fp32 alone.
template <bool EXACT, int BM, int BN, int WM, int WN, int NBUF>
__global__ __launch_bounds__(WM * WN * 64, 1) void fp8_gemm_kernel(Fp8GemmArgs a) {
  constexpr int NW = WM * WN;
  constexpr int MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr uint32_t kXBytes = BM * kSlice, kBytes = (BM + BN) * kSlice;
  constexpr int kPieces = (BM + BN) / 16 / NW;  // DMAs of a wave for a slice
  static_assert((BM + BN) % (16 * NW) == 0 && BN / WN <= 128 && 128 % (BN / WN) == 0, "tile");
  constexpr uint32_t kWBlocks = (BN + 127) / 128;
  // [NBUF][X rows | W rows], X's scale words [kSegmentWords][BM], W's [kSegmentWords][kWBlocks]
  __shared__ __attribute__((aligned(1024))) char lds[NBUF * kBytes + kSegmentWords * 4 * (BM + kWBlocks)];
  uint32_t* const sx = (uint32_t*)(lds + NBUF * kBytes);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wm = wave / WN, wn = wave % WN, r = lane & 31, h = lane >> 5;

  uint32_t mt0, nt0, split;
  {
    const uint32_t tiles = a.mtiles * a.ntiles;
    uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
    split = id / tiles;
    id -= split * tiles;
    // stripes of `group` column tiles; within a stripe the columns fastest
    const uint32_t stripe = id / (a.mtiles * a.group), at = id - stripe * a.mtiles * a.group;
    const uint32_t wide = min(a.group, a.ntiles - stripe * a.group);
    mt0 = at / wide;
    nt0 = stripe * a.group + (at - mt0 * wide);
  }
  const uint32_t m0 = mt0 * BM, n0 = nt0 * BN;
  const uint32_t kbegin = split * a.kps, kend = min(a.k, kbegin + a.kps);

  // What a lane of each DMA fetches: 16 rows of 64 bytes; rows past the end are the last row again.
  uint32_t voff[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const uint32_t piece = i * NW + wave, row = piece * 16 + lane / 4;  // of the tile's X rows, then W rows
    const uint32_t chunk = (lane & 3) ^ (row >> 1 & 3);
    const bool of_x = piece < BM / 16;
    const uint32_t last = of_x ? a.m - 1 - m0 : a.n - 1 - n0;
    const uint32_t at = min(of_x ? row : row - BM, last);
    voff[i] = at * (of_x ? a.ldx : a.ldw) + chunk * 16;
  }
  const uint8_t* const xb = a.x + (size_t)m0 * a.ldx;
  const uint8_t* const wb = a.w + (size_t)n0 * a.ldw;

  f16v acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  struct Frags {
    i8v x[MT], w[NT];
    int ex[MT], ew;  // the scales' bytes
  };
  // chunks 2 h and 2 h + 1 of row r of each 32-row tile
  const uint32_t key = r >> 1 & 3, c0 = ((2 * h) ^ key) * 16, c1 = ((2 * h + 1) ^ key) * 16;
  const uint32_t xrow = (wm * (BM / WM) + r) * kSlice, wrow = kXBytes + (wn * (BN / WN) + r) * kSlice;
  const uint8_t* const xscale = (const uint8_t*)(sx + wm * (BM / WM) + r);
  const uint8_t* const wscale = (const uint8_t*)(sx + kSegmentWords * BM + wn * (BN / WN) / 128);
  auto read = [&](Frags& f, uint32_t s) {
    const char* const b = lds + s % NBUF * kBytes;
    auto two = [&](const char* p) {
      const u4 lo = *(const u4*)(p + c0), hi = *(const u4*)(p + c1);
      return i8v{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
#pragma unroll
    for (int i = 0; i < MT; ++i) f.x[i] = two(b + xrow + i * 32 * kSlice);
#pragma unroll
    for (int j = 0; j < NT; ++j) f.w[j] = two(b + wrow + j * 32 * kSlice);
    const uint32_t word = s / 8, byte = s / 2 % 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) f.ex[i] = xscale[(word * BM + 32 * i) * 4 + byte];
    f.ew = wscale[word * kWBlocks * 4 + byte];
  };

  for (uint32_t k0 = kbegin; k0 < kend; k0 += kSegment) {
    const uint32_t k1 = min(kend, k0 + kSegment), slices = (k1 - k0 + kSlice - 1) / kSlice;
    auto stage = [&](uint32_t s) {
      const uint32_t to = lds0 + (s % NBUF) * kBytes;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t piece = i * NW + wave;
        dma16(to + piece * 1024, voff[i], (piece < BM / 16 ? xb : wb) + k0 + s * kSlice);
      }
    };
    // the segment's scale words, four rows a lane
    const uint32_t words = (k1 - k0 + kFp8Word - 1) / kFp8Word, word0 = k0 / kFp8Word;
    uint32_t* const swords = sx + kSegmentWords * BM;
    for (uint32_t i = threadIdx.x; i < words * (BM / 4); i += NW * 64) {
      const uint32_t j = i / (BM / 4), g = min(i % (BM / 4) * 4, (a.m - 1 - m0) / 4 * 4);
      *(u4*)(sx + 4 * i) = *(const u4*)(a.sx + (size_t)(word0 + j) * a.ldsx + m0 + g);
    }
    for (uint32_t i = threadIdx.x; i < words * kWBlocks; i += NW * 64) {
      const uint32_t j = i / kWBlocks, b = min(n0 / kFp8Block + i % kWBlocks, (a.n - 1) / kFp8Block);
      swords[i] = a.sw[(size_t)(word0 + j) * a.ldsw + b];
    }
#pragma unroll
    for (uint32_t s = 0; s < NBUF; ++s)
      if (s < slices) stage(s);
    wait_vm<0>();
    __syncthreads();

    Frags f0, f1;
    read(f0, 0);
    auto step = [&](Frags& now, Frags& next, uint32_t s) {
      // slice s + 1 has landed, and everyone has read slice s
      if (s + NBUF - 1 < slices)
        wait_vm<(NBUF - 2) * kPieces>();
      else
        wait_vm<0>();
      wait_lgkm<0>();
      __syncthreads();
      if (s + NBUF < slices) stage(s + NBUF);
      if (s + 1 < slices) read(next, s + 1);
      if constexpr (EXACT) {
        auto factor = [](int byte) { return __uint_as_float((uint32_t)byte << 23); };
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          b8 w[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) w[j] = widened(now.w[j][2 * q], now.w[j][2 * q + 1], factor(now.ew));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const b8 x = widened(now.x[i][2 * q], now.x[i][2 * q + 1], factor(now.ex[i]));
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], x, acc[i][j], 0, 0, 0);
          }
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma_scaled(now.w[j], now.x[i], acc[i][j], now.ew, now.ex[i]);
    };
    for (uint32_t s = 0; s < slices; s += 2) {
      step(f0, f1, s);
      if (s + 1 < slices) step(f1, f0, s + 1);
    }
    __syncthreads();  // the next segment's scales and slices go where these lay
  }

  const uint32_t ldp = (a.n + 3) / 4 * 4;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const uint32_t row = m0 + wm * (BM / WM) + 32 * i + r;
    if (row >= a.m) continue;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t n = n0 + wn * (BN / WN) + 32 * j + 4 * h;
      auto four = [&](int q) { return f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]}; };
      if (a.ws) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + 8 * q < ldp) *(f4*)(a.ws + ((size_t)split * a.m + row) * ldp + n + 8 * q) = four(q);
      } else if (a.epi == 3u) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (n + 8 * q < a.n) put_swiglu(a, row, (n0 + wn * (BN / WN) + 32 * j) / 2 + 4 * h + 8 * q, four(q), four(q + 2));
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + 8 * q < a.n) put(a, row, n + 8 * q, four(q));
      }
    }
  }
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
struct Variant {
  uint32_t bm, bn;
};
// fp32 outputs are computed in bf16 (above)
bool exact_sums(uint32_t epi) { return epi == 0u || epi == 2u; }
constexpr Variant kVariants[] = {{256, 256}, {256, 128}, {128, 128}, {64, 128}};
template <int BM, int BN, int WM, int WN, int NBUF>
void launch(const Fp8GemmArgs& a, uint32_t grid, hipStream_t s) {
  if (exact_sums(a.epi))
    hipLaunchKernelGGL((fp8_gemm_kernel<true, BM, BN, WM, WN, NBUF>), dim3(grid), dim3(WM * WN * 64), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_gemm_kernel<false, BM, BN, WM, WN, NBUF>), dim3(grid), dim3(WM * WN * 64), 0, s, a);
}
}  // namespace

int fp8_variant_count() { return sizeof(kVariants) / sizeof(kVariants[0]); }

Fp8Plan fp8_gemm_plan_of(int v, uint32_t splits, uint32_t m, uint32_t n, uint32_t k) {
  Fp8Plan p;
  p.variant = v;
  p.mtiles = (m + kVariants[v].bm - 1) / kVariants[v].bm;
  p.ntiles = (n + kVariants[v].bn - 1) / kVariants[v].bn;
  const uint32_t words = (k + kFp8Word - 1) / kFp8Word;
  const uint32_t each = (words + splits - 1) / std::max(1u, splits);
  p.kps = std::max(1u, each) * kFp8Word;
  p.splits = std::max(1u, (words + each - 1) / std::max(1u, each));
  if (p.splits > 1) p.ws_bytes = (uint64_t)p.splits * m * ((n + 3) / 4 * 4) * sizeof(float);
  return p;
}

Fp8Plan fp8_gemm_plan(uint32_t m, uint32_t n, uint32_t k, uint32_t epi, uint32_t cus) {
  const int v = m > 1024 ? (exact_sums(epi) ? 1 : 0) : m > 64 ? 2 : 3;
  Fp8Plan p = fp8_gemm_plan_of(v, 1, m, n, k);
  const uint64_t tiles = (uint64_t)p.mtiles * p.ntiles;
  if (tiles * 2 <= cus) p = fp8_gemm_plan_of(v, (uint32_t)std::min<uint64_t>(16, cus / tiles), m, n, k);
  return p;
}

hipError_t launch_fp8_gemm(const Fp8Plan& p, const Fp8& x, const Fp8& w, void* y, uint32_t ldy, uint32_t m, uint32_t n,
                           uint32_t k, uint32_t epi, float* ws, hipStream_t s) {
  if (m == 0 || n == 0) return hipSuccess;
  const Fp8GemmArgs a{x.codes, w.codes, x.scales, w.scales, y,     p.splits > 1 ? ws : nullptr, x.ld, w.ld, x.lds, w.lds, ldy,
                      m,       n,       k,        p.kps,    p.mtiles, p.ntiles, std::min(4u, p.ntiles), epi};
  const uint32_t grid = p.mtiles * p.ntiles * p.splits;
  if (p.variant == 0)  // (never with exact sums: its registers would not do)
    hipLaunchKernelGGL((fp8_gemm_kernel<false, 256, 256, 2, 4, 4>), dim3(grid), dim3(512), 0, s, a);
  else if (p.variant == 1)
    launch<256, 128, 4, 2, 4>(a, grid, s);
  else if (p.variant == 2)
    launch<128, 128, 2, 2, 4>(a, grid, s);
  else
    launch<64, 128, 1, 4, 4>(a, grid, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const size_t total = (size_t)m * ((epi == 3u ? n / 2 : (n + 3) / 4 * 4) / 4);
  hipLaunchKernelGGL(fp8_reduce_kernel, dim3((uint32_t)std::min<size_t>((total + 255) / 256, 16384)), dim3(256), 0, s, a,
                     p.splits);
  return hipGetLastError();
}

}  // namespace dh
