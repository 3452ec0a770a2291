// C ABI of the 8-bit floating point codes and their product (include/decide_hip.h, "8-bit floating point").
// Contract violations return DH_EINVAL with a message; nothing is launched after a failed check.
#include <algorithm>
#include <cmath>

#include "api_internal.h"
#include "fp8.h"

using namespace dh_api;

namespace {
constexpr uint64_t kMaxThreads = UINT32_MAX;  // of a launch, in a dimension

int check_matrix(const char* op, const char* what, const dh_fp8_matrix* x, uint64_t scale_rows, uint32_t k) {
  if (!x) return fail(DH_EINVAL, "%s: null %s", op, what);
  const uint64_t wide = ((uint64_t)k + DH_FP8_BLOCK - 1) / DH_FP8_BLOCK * DH_FP8_BLOCK;
  if (x->ld < wide || x->ld % 16 != 0)
    return fail(DH_EINVAL, "%s: row stride %u of %s must be a multiple of 16 covering %llu columns (K = %u in whole blocks)",
                op, x->ld, what, (unsigned long long)wide, k);
  if (x->lds < scale_rows || x->lds % 4 != 0)
    return fail(DH_EINVAL, "%s: scale stride %u of %s must be a multiple of 4 covering its %llu rows or blocks of rows", op,
                x->lds, what, (unsigned long long)scale_rows);
  if ((x->codes && !aligned(x->codes, 16)) || (x->scales && !aligned(x->scales, 16)))
    return fail(DH_EINVAL, "%s: codes and scales of %s must be 16-byte aligned", op, what);
  if (x->ld > 1u << 23) return fail(DH_EINVAL, "%s: row stride %u of %s exceeds 2^23", op, x->ld, what);
  if (x->lds > 1u << 26) return fail(DH_EINVAL, "%s: scale stride %u of %s exceeds 2^26", op, x->lds, what);
  return DH_OK;
}

int check_source(const char* op, const void* x, uint32_t ldx, uint32_t dtype, uint32_t k) {
  if (dtype > 2) return fail(DH_EINVAL, "%s: dtype %u is not one of 0 (fp16), 1 (bf16), 2 (fp32)", op, dtype);
  if (ldx < k || ldx % 8 != 0)
    return fail(DH_EINVAL, "%s: row stride %u must be a multiple of 8 covering K = %u", op, ldx, k);
  if (x && !aligned(x, 16)) return fail(DH_EINVAL, "%s: the values must be 16-byte aligned", op);
  return DH_OK;
}

dh::Fp8 fp8(const dh_fp8_matrix* x) { return dh::Fp8{(uint8_t*)x->codes, (uint32_t*)x->scales, x->ld, x->lds}; }

int check_gemm(const char* op, const dh_fp8_matrix* x, const dh_fp8_matrix* w, uint32_t m, uint32_t n, uint32_t k) {
  int rc = check_matrix(op, "x", x, m, k);
  if (rc == DH_OK) rc = check_matrix(op, "w", w, ((uint64_t)n + DH_FP8_BLOCK - 1) / DH_FP8_BLOCK, k);
  return rc;
}

// What a plan takes must fit one launch. (Its partial sums are those of at most as many tiles as fit the device at once: they
// cannot reach the split-K workspace's ceiling.)
int plan_of(const char* op, const dh_ctx* ctx, uint32_t m, uint32_t n, uint32_t k, uint32_t epi, dh::Fp8Plan* p) {
  *p = dh::fp8_gemm_plan(m, n, k, epi, ctx->cus);
  if ((uint64_t)p->mtiles * p->ntiles * p->splits > kMaxThreads / 512)
    return fail(DH_EINVAL, "%s: %u x %u outputs exceed one launch; split the call along M or N", op, m, n);
  return DH_OK;
}
}  // namespace

extern "C" {

int dh_fp8_quant_rows(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, uint32_t dtype, const float* norm_w,
                      uint32_t add_one, float eps, const dh_fp8_matrix* out, uint32_t rows, uint32_t k) {
  int rc = check_source("fp8_quant_rows", x, ldx, dtype, k);
  if (rc == DH_OK) rc = check_matrix("fp8_quant_rows", "out", out, rows, k);
  if (rc != DH_OK) return rc;
  if (norm_w && !aligned(norm_w, 16)) return fail(DH_EINVAL, "fp8_quant_rows: norm_w must be 16-byte aligned");
  if (norm_w && (!(eps > 0.0f) || !std::isfinite(eps)))
    return fail(DH_EINVAL, "fp8_quant_rows: eps must be positive and finite");
  const uint64_t words = ((uint64_t)k + dh::kFp8Word - 1) / dh::kFp8Word;
  if (((uint64_t)rows + 15) / 16 * words > kMaxThreads / 256 || (norm_w && rows > kMaxThreads / 256))
    return fail(DH_EINVAL, "fp8_quant_rows: %u rows of %u columns exceed one launch; split the call", rows, k);
  if (!ctx) return fail(DH_EINVAL, "fp8_quant_rows: null context");
  if (rows == 0 || k == 0) return ok();
  if (!x || !out->codes || !out->scales) return fail(DH_EINVAL, "fp8_quant_rows: null pointer");
  mark(ctx, kKidFp8Rows);
  return hip_status(dh::launch_fp8_quant_rows(x, ldx, dtype, norm_w, add_one != 0, eps, fp8(out), rows, k,
                                              (hipStream_t)stream),
                    "fp8_quant_rows");
}

int dh_fp8_quant_blocks(dh_ctx* ctx, void* stream, const void* w, uint32_t ldw, uint32_t dtype, const dh_fp8_matrix* out,
                        uint32_t n, uint32_t k) {
  const uint64_t blocks = ((uint64_t)n + DH_FP8_BLOCK - 1) / DH_FP8_BLOCK;
  int rc = check_source("fp8_quant_blocks", w, ldw, dtype, k);
  if (rc == DH_OK) rc = check_matrix("fp8_quant_blocks", "out", out, blocks, k);
  if (rc != DH_OK) return rc;
  if (blocks * (((uint64_t)k + dh::kFp8Word - 1) / dh::kFp8Word) > kMaxThreads / 1024)
    return fail(DH_EINVAL, "fp8_quant_blocks: %u rows of %u columns exceed one launch; split the call", n, k);
  if (!ctx) return fail(DH_EINVAL, "fp8_quant_blocks: null context");
  if (n == 0 || k == 0) return ok();
  if (!w || !out->codes || !out->scales) return fail(DH_EINVAL, "fp8_quant_blocks: null pointer");
  mark(ctx, kKidFp8Blocks);
  return hip_status(dh::launch_fp8_quant_blocks(w, ldw, dtype, fp8(out), n, k, (hipStream_t)stream), "fp8_quant_blocks");
}

int dh_gemm_fp8(dh_ctx* ctx, void* stream, const dh_fp8_matrix* x, const dh_fp8_matrix* w, void* y, uint32_t ldy,
                uint32_t m, uint32_t n, uint32_t k, uint32_t epi) {
  if (epi > DH_EPI_SWIGLU_F16) return fail(DH_EINVAL, "gemm_fp8: epilogue %u is not one of 0..3", epi);
  if (epi == DH_EPI_SWIGLU_F16 && n % 32 != 0)
    return fail(DH_EINVAL, "gemm_fp8: N = %u must be a multiple of 32 with DH_EPI_SWIGLU_F16", n);
  int rc = check_gemm("gemm_fp8", x, w, m, n, k);
  if (rc != DH_OK) return rc;
  const uint32_t cols = epi == DH_EPI_SWIGLU_F16 ? n / 2 : n;
  const bool f32 = epi == DH_EPI_STORE_F32 || epi == DH_EPI_ADD_F32;
  if (ldy < cols || ldy % 4 != 0)
    return fail(DH_EINVAL, "gemm_fp8: row stride ldy = %u must be a multiple of 4 covering the %u output columns", ldy, cols);
  if (y && !aligned(y, f32 ? 16 : 8))
    return fail(DH_EINVAL, "gemm_fp8: y address %p must be a multiple of %d", y, f32 ? 16 : 8);
  if (!ctx) return fail(DH_EINVAL, "gemm_fp8: null context");
  if (m == 0 || n == 0) return ok();
  if (!y || (k && (!x->codes || !x->scales || !w->codes || !w->scales))) return fail(DH_EINVAL, "gemm_fp8: null pointer");
  dh::Fp8Plan p;
  rc = plan_of("gemm_fp8", ctx, m, n, k, epi, &p);
  if (rc != DH_OK) return rc;
  float* ws = nullptr;
  if (p.splits > 1) {
    rc = ensure_ws(ctx, (hipStream_t)stream, p.ws_bytes, &ws);
    if (rc != DH_OK) return rc;
    mark(ctx, kKidFp8Reduce);
  }
  mark(ctx, kKidFp8Gemm + p.variant);
  return hip_status(dh::launch_fp8_gemm(p, fp8(x), fp8(w), y, ldy, m, n, k, epi, ws, (hipStream_t)stream), "gemm_fp8");
}

int dh_gemm_fp8_ws(dh_ctx* ctx, void* stream, uint32_t max_m, uint32_t n, uint32_t k) {
  if (!ctx) return fail(DH_EINVAL, "gemm_fp8_ws: null context");
  if (max_m > DH_PLAN_MAX_ROWS)
    return fail(DH_EINVAL, "gemm_fp8_ws: max_m = %u exceeds %u (DH_PLAN_MAX_ROWS)", max_m, DH_PLAN_MAX_ROWS);
  uint64_t bytes = 0;
  for (uint32_t m = 1; m <= max_m && n; ++m)
    for (uint32_t epi : {DH_EPI_STORE_F32, DH_EPI_STORE_F16})
      bytes = std::max(bytes, dh::fp8_gemm_plan(m, n, k, epi, ctx->cus).ws_bytes);
  float* ws = nullptr;
  return bytes ? ensure_ws(ctx, (hipStream_t)stream, bytes, &ws) : ok();
}

}  // extern "C"

namespace dh_api {

size_t fp8_warm_bytes() { return 65536; }

int fp8_warm(dh_ctx* ctx, hipStream_t s, void* mem) {
  // one row of 1,024 values and its codes, as activations and as a weight; everything zeros
  char* const base = (char*)mem;
  float* const x = (float*)base;
  const dh_fp8_matrix rows{base + 4096, base + 8192, 1024, 4}, blocks{base + 12288, base + 16384, 1024, 4};
  float *const y = (float*)(base + 20480), *const ws = (float*)(base + 24576);
  int rc = dh_fp8_quant_rows(ctx, s, x, 1024, 2, nullptr, 0, 0.f, &rows, 1, 1024);
  if (rc == DH_OK) rc = dh_fp8_quant_rows(ctx, s, x, 1024, 2, x, 1, 1.f, &rows, 1, 1024);
  if (rc == DH_OK) rc = dh_fp8_quant_blocks(ctx, s, x, 1024, 2, &blocks, 1, 1024);
  for (int v = 0; v < dh::fp8_variant_count() && rc == DH_OK; ++v) {
    mark(ctx, kKidFp8Gemm + v);
    rc = hip_status(dh::launch_fp8_gemm(dh::fp8_gemm_plan_of(v, 1, 1, 4, 1024), fp8(&rows), fp8(&blocks), y, 4, 1, 1, 1024,
                                        DH_EPI_STORE_F16, nullptr, s),
                    "gemm_fp8");
  }
  if (rc == DH_OK) {
    mark(ctx, kKidFp8Reduce);
    rc = hip_status(dh::launch_fp8_gemm(dh::fp8_gemm_plan_of(dh::fp8_variant_count() - 1, 2, 1, 4, 1024), fp8(&rows),
                                        fp8(&blocks), y, 4, 1, 1, 1024, DH_EPI_STORE_F32, ws, s),
                    "gemm_fp8");
  }
  return rc;
}

}  // namespace dh_api
