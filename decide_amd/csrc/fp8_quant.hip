// Rows and weights into 8-bit floating point (OCP e4m3) with a power-of-two scale for each block of 128, for gfx950.
//
//   a = the block's largest finite magnitude, scale 2^e with the smallest e such that a <= 448 * 2^e (e >= -100),
//   code = e4m3(v / 2^e)
// Dividing by a power of two is exact (a quotient below fp32's normal range is below half of e4m3's smallest step, 2^-10,
// and its code 0 either way), so a code is a value rounded once. The exponent follows from the bits of a: 448 is
// 1.75 * 2^8, so a = f * 2^E with f in [1, 2) needs e = E - 8 where f <= 1.75 and E - 7 beyond.
//
// Four blocks of a row, 512 columns, are one wave's: eight columns a lane, 16 lanes a block, and the word that holds
// their four scales. Rows are coded from registers: each value is read once and its code written once, 8 bytes a lane.
// With the norm a workgroup takes a row, whose sum of squares and whose normed values are formed in 64 bits: a value is
// then one rounding to fp32 from exact, and which side of a scale's border it falls on does not depend on the order of a
// sum. Bound by memory: 16,383 x 9,216 fp16 values 78 us, 5.8 TB/s; eight normed rows of 2,560 4.2 us, a launch's time.
#include <algorithm>

#include "fp8.h"
#include "tile_common.h"

namespace dh {

namespace {
struct Half {};
struct Bf16 {};
struct QuantArgs {
  const void* x;
  const float* norm_w;
  uint8_t* codes;
  uint32_t* scales;
  uint32_t ldx, ldc, lds, rows, k;
  uint32_t add_one;
  float eps;
};

// Eight elements of T (float, Half, Bf16) as they lie in memory; those from `have` on are zero and are not read.
template <typename T>
struct Eight {
  static constexpr int kWords = std::is_same_v<T, float> ? 8 : 4;
  u4 v[kWords / 4];
  __device__ __forceinline__ void load(const void* x, size_t at, uint32_t have) {
    typedef std::conditional_t<std::is_same_v<T, float>, float, uint16_t> E;
    const E* const p = (const E*)x + at;
    if (have >= 8) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) v[i] = ((const u4*)p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) v[i] = u4{0, 0, 0, 0};
      uint32_t part[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) part[i] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < (int)have) {
          if constexpr (kWords == 8)
            part[i] = __float_as_uint(p[i]);
          else
            part[i / 2] |= (uint32_t)p[i] << 16 * (i % 2);
        }
      }
#pragma unroll
      for (int i = 0; i < kWords; ++i) v[i / 4][i % 4] = part[i];
    }
  }
  // Values that are wanted again are formed again: as floats they would take twice the registers.
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) asm volatile("" : "+v"(v[i]));
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (kWords == 8) {
      return __uint_as_float(v[i / 4][i % 4]);
    } else {
      const uint32_t w = v[0][i / 2];
      if constexpr (std::is_same_v<T, Half>)
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(i % 2 ? w >> 16 : w & 0xffff));
      else
        return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
    }
  }
};

// The bits of the largest finite magnitude among eight values.
__device__ __forceinline__ uint32_t top_of(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    top = max(top, b < 0x7f800000u ? b : 0u);
  }
  return top;
}
// The largest of each group of 16 lanes.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  auto with = [&](auto lanes) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(lanes)::value, 0xf, 0xf, false));
  };
  with(std::integral_constant<int, 0xb1>{});   // the neighbour's
  with(std::integral_constant<int, 0x4e>{});   // the neighbouring pair's
  with(std::integral_constant<int, 0x141>{});  // mirrored within 8 lanes: the other four's
  with(std::integral_constant<int, 0x140>{});  // within 16: the other eight's
  return v;
}
// The scale's byte (exponent + 127, at least 27) from the largest magnitude's bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const int b = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(b, 27);
}
// Eight codes. `b` is at most 248, so the factor 2^(127 - b) is a normal number.
__device__ __forceinline__ uint2 codes_of(const float* v, uint32_t b) {
  const float f = __uint_as_float((254 - b) << 23);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * f, v[4 * i + 1] * f, 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * f, v[4 * i + 3] * f, c, true);
  }
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) odd |= (__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u;
  if (__any(odd)) {  // what is not finite is the code of NaN
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u)
        w[i / 4] = (w[i / 4] & ~(0xffu << 8 * (i % 4))) | 0x7fu << 8 * (i % 4);
  }
  return uint2{w[0], w[1]};
}
// The word of the scales of a wave's four blocks, each held by a group of 16 lanes; 127 for those from `blocks` on.
__device__ __forceinline__ uint32_t word_of(uint32_t byte, uint32_t blocks) {
  uint32_t w = 0;
#pragma unroll
  for (uint32_t g = 0; g < 4; ++g)
    w |= (g < blocks ? (uint32_t)__builtin_amdgcn_readlane((int)byte, 16 * g) : 127u) << 8 * g;
  return w;
}

constexpr uint32_t kRowsEach = 4;  // rows of a wave of the kernel without the norm: their loads are in flight together
}  // namespace

// Four rows a wave, 16 a workgroup, 512 columns: without the norm blocks do not know of each other.
template <typename T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(QuantArgs a) {
  const uint32_t lane = threadIdx.x & 63, words = (a.k + kFp8Word - 1) / kFp8Word;
  const uint32_t word = blockIdx.x % words, row0 = (blockIdx.x / words * 4 + (threadIdx.x >> 6)) * kRowsEach;
  const uint32_t col = word * kFp8Word + 8 * lane, have = col < a.k ? a.k - col : 0;
  const uint32_t left = a.k - word * kFp8Word, blocks = (left + kFp8Block - 1) / kFp8Block;
  Eight<T> e[kRowsEach];
#pragma unroll
  for (uint32_t r = 0; r < kRowsEach; ++r) e[r].load(a.x, (size_t)(row0 + r) * a.ldx + col, row0 + r < a.rows ? have : 0);
#pragma unroll
  for (uint32_t r = 0; r < kRowsEach; ++r) {
    const uint32_t row = row0 + r;
    if (row >= a.rows) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e[r][i];
    const uint32_t b = scale_byte(max16(top_of(v)));
    if (lane / 16 < blocks) *(uint2*)(a.codes + (size_t)row * a.ldc + col) = codes_of(v, b);
    const uint32_t w = word_of(b, blocks);
    if (lane == 0) a.scales[(size_t)word * a.lds + row] = w;
  }
}

// A row a workgroup of four waves, wave w taking words w, w + 4, ...; the first CH of each stay in registers between the sum
// of squares and the codes, later ones are read again (from the caches: a row is at most some tens of KB).
template <typename T, int CH>
__global__ __launch_bounds__(256) void fp8_norm_rows_kernel(QuantArgs a) {
  __shared__ double sums[4];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
  const uint32_t words = (a.k + kFp8Word - 1) / kFp8Word;
  const size_t base = (size_t)row * a.ldx;
  Eight<T> e[CH];
  double sum = 0.0;
  auto add = [&](const Eight<T>& x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double d = x[i];
      sum = fma(d, d, sum);
    }
  };
  auto col_of = [&](uint32_t word) { return word * kFp8Word + 8 * lane; };
  auto have_of = [&](uint32_t word) { return col_of(word) < a.k ? a.k - col_of(word) : 0; };
#pragma unroll
  for (int c = 0; c < CH; ++c) e[c].load(a.x, base + col_of(wave + 4 * c), have_of(wave + 4 * c));
#pragma unroll
  for (int c = 0; c < CH; ++c) add(e[c]);
  for (uint32_t word = wave + 4 * CH; word < words; word += 4) {
    Eight<T> x;
    x.load(a.x, base + col_of(word), have_of(word));
    add(x);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  const double r = 1.0 / sqrt((sums[0] + sums[1] + sums[2] + sums[3]) / (double)a.k + (double)a.eps);
  auto code = [&](uint32_t word, const Eight<T>& x) {
    const uint32_t col = col_of(word), have = have_of(word);
    const uint32_t blocks = (a.k - word * kFp8Word + kFp8Block - 1) / kFp8Block;
    Eight<float> w;
    w.load(a.norm_w, col, have);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double g = a.add_one ? 1.0 + (double)w[i] : (double)w[i];
      v[i] = i < (int)have ? (float)((double)x[i] * r * g) : 0.f;  // (0 * inf would be NaN)
    }
    const uint32_t b = scale_byte(max16(top_of(v)));
    if (lane / 16 < blocks) *(uint2*)(a.codes + (size_t)row * a.ldc + col) = codes_of(v, b);
    const uint32_t word_value = word_of(b, blocks);
    if (lane == 0) a.scales[(size_t)word * a.lds + row] = word_value;
  };
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (wave + 4 * c < words) code(wave + 4 * c, e[c]);
  for (uint32_t word = wave + 4 * CH; word < words; word += 4) {
    Eight<T> x;
    x.load(a.x, base + col_of(word), have_of(word));
    code(word, x);
  }
}

// 128 rows and 512 columns a workgroup: 16 waves of eight rows, which stay in registers as they were read while the waves' largest
// values meet. 18,432 x 2,560 from bf16: 29.9 us, 4.7 TB/s, as a large copy's; eight waves of 16 rows 31.2, and 37.3 with the
// values kept as floats, whose registers leave a CU one workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void fp8_blocks_kernel(QuantArgs a) {
  constexpr uint32_t kWaves = 16, kRows = kFp8Block / kWaves;
  __shared__ uint32_t tops[kWaves][4];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (a.k + kFp8Word - 1) / kFp8Word;
  const uint32_t word = blockIdx.x % words, block = blockIdx.x / words, row0 = block * kFp8Block + wave * kRows;
  const uint32_t col = word * kFp8Word + 8 * lane, have = col < a.k ? a.k - col : 0;
  const uint32_t blocks = (a.k - word * kFp8Word + kFp8Block - 1) / kFp8Block;
  Eight<T> e[kRows];
#pragma unroll
  for (uint32_t r = 0; r < kRows; ++r) e[r].load(a.x, (size_t)(row0 + r) * a.ldx + col, row0 + r < a.rows ? have : 0);
  uint32_t top = 0;
#pragma unroll
  for (uint32_t r = 0; r < kRows; ++r) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e[r][i];
    top = max(top, top_of(v));
    e[r].keep();
  }
  top = max16(top);
  if (lane % 16 == 0) tops[wave][lane / 16] = top;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) top = max(top, tops[w][lane / 16]);
  const uint32_t b = scale_byte(top);
#pragma unroll
  for (uint32_t r = 0; r < kRows; ++r) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e[r][i];
    const uint2 c = codes_of(v, b);
    if (row0 + r < a.rows && lane / 16 < blocks) *(uint2*)(a.codes + (size_t)(row0 + r) * a.ldc + col) = c;
  }
  const uint32_t w = word_of(b, blocks);
  if (threadIdx.x == 0) a.scales[(size_t)word * a.lds + block] = w;
}

namespace {
template <typename T>
void rows_kernels(const QuantArgs& a, hipStream_t s) {
  const uint32_t words = (a.k + kFp8Word - 1) / kFp8Word;
  if (!a.norm_w)
    hipLaunchKernelGGL((fp8_rows_kernel<T>), dim3((a.rows + 4 * kRowsEach - 1) / (4 * kRowsEach) * words), dim3(256), 0, s, a);
  else if (words <= 8)
    hipLaunchKernelGGL((fp8_norm_rows_kernel<T, 2>), dim3(a.rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_norm_rows_kernel<T, 5>), dim3(a.rows), dim3(256), 0, s, a);
}
}  // namespace

hipError_t launch_fp8_quant_rows(const void* x, uint32_t ldx, uint32_t dtype, const float* norm_w, bool add_one, float eps,
                                 const Fp8& out, uint32_t rows, uint32_t k, hipStream_t s) {
  if (rows == 0 || k == 0) return hipSuccess;
  const QuantArgs a{x, norm_w, out.codes, out.scales, ldx, out.ld, out.lds, rows, k, add_one ? 1u : 0u, eps};
  if (dtype == 0)
    rows_kernels<Half>(a, s);
  else if (dtype == 1)
    rows_kernels<Bf16>(a, s);
  else
    rows_kernels<float>(a, s);
  return hipGetLastError();
}

hipError_t launch_fp8_quant_blocks(const void* w, uint32_t ldw, uint32_t dtype, const Fp8& out, uint32_t n, uint32_t k,
                                   hipStream_t s) {
  if (n == 0 || k == 0) return hipSuccess;
  const QuantArgs a{w, nullptr, out.codes, out.scales, ldw, out.ld, out.lds, n, k, 0, 0.f};
  const dim3 grid((n + kFp8Block - 1) / kFp8Block * ((k + kFp8Word - 1) / kFp8Word));
  if (dtype == 0)
    hipLaunchKernelGGL((fp8_blocks_kernel<Half>), grid, dim3(1024), 0, s, a);
  else if (dtype == 1)
    hipLaunchKernelGGL((fp8_blocks_kernel<Bf16>), grid, dim3(1024), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_blocks_kernel<float>), grid, dim3(1024), 0, s, a);
  return hipGetLastError();
}

}  // namespace dh
