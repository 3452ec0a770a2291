// Launch arguments and launchers of the 8-bit floating point codes and their matrix product (fp8_quant.hip,
// fp8_gemm.hip), shared by the kernels and the C ABI (api_fp8.cpp). Host-visible, no device code here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dh {

constexpr uint32_t kFp8Block = 128;  // columns (for weights: rows too) that share a scale
constexpr uint32_t kFp8Word = 512;   // columns whose four scales lie in one word

// A matrix of codes and its scales, as dh_fp8_matrix has them. Word j of row (or block of rows) r is at scales[j * lds + r].
struct Fp8 {
  uint8_t* codes;
  uint32_t* scales;
  uint32_t ld, lds;
};

// elements of x: 0 fp16, 1 bf16, 2 fp32; norm_w null: no norm
hipError_t launch_fp8_quant_rows(const void* x, uint32_t ldx, uint32_t dtype, const float* norm_w, bool add_one, float eps,
                                 const Fp8& out, uint32_t rows, uint32_t k, hipStream_t s);
hipError_t launch_fp8_quant_blocks(const void* w, uint32_t ldw, uint32_t dtype, const Fp8& out, uint32_t n, uint32_t k,
                                   hipStream_t s);

// How a product is computed: a tile variant, and K in `splits` parts of `kps` columns (a multiple of kFp8Word) whose partial
// sums [splits][m][n rounded up to 4] go through the workspace.
struct Fp8Plan {
  int variant = 0;
  uint32_t splits = 1, kps = 0;
  uint32_t mtiles = 0, ntiles = 0;
  uint64_t ws_bytes = 0;
};
Fp8Plan fp8_gemm_plan(uint32_t m, uint32_t n, uint32_t k, uint32_t epi, uint32_t cus);
int fp8_variant_count();
// The plan with variant v and so many splits (fewer where K has fewer words).
Fp8Plan fp8_gemm_plan_of(int v, uint32_t splits, uint32_t m, uint32_t n, uint32_t k);
hipError_t launch_fp8_gemm(const Fp8Plan& p, const Fp8& x, const Fp8& w, void* y, uint32_t ldy, uint32_t m, uint32_t n,
                           uint32_t k, uint32_t epi, float* ws, hipStream_t s);

}  // namespace dh
