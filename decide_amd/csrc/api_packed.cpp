// C ABI of attention over packed sequences (include/decide_hip.h, "Causal attention over packed sequences").
// Contract violations return DH_EINVAL with a message; nothing is launched after a failed check.
#include <algorithm>
#include <cmath>

#include "api_internal.h"
#include "packed.h"

using namespace dh_api;

namespace {
constexpr uint64_t kMaxThreads = UINT32_MAX;  // of a launch, in a dimension
constexpr uint32_t kMostStride = 1u << 24;    // elements of a row of k or v: a block of keys is addressed in 32 bits

int check_shape(const char* op, uint32_t q_rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(DH_EINVAL, "%s: head_dim = %u must be 64, 128 or 256", op, head_dim);
  if (kv_heads < 1 || kv_heads > 1024) return fail(DH_EINVAL, "%s: kv_heads = %u must be in 1..1024", op, kv_heads);
  if (heads < 1 || heads % kv_heads != 0 || heads / kv_heads > 1024)
    return fail(DH_EINVAL, "%s: heads = %u must be a multiple of the %u kv heads, at most 1024 for each", op, heads,
                kv_heads);
  const uint64_t tiles = (uint64_t)q_rows * (heads / kv_heads) / 32 + seqs;
  if ((uint64_t)q_rows * heads > UINT32_MAX || tiles * kv_heads > kMaxThreads / 512)
    return fail(DH_EINVAL, "%s: %u rows x %u heads over %u sequences exceed one launch; split the call", op, q_rows, heads,
                seqs);
  return DH_OK;
}

int check_rows(const char* op, const char* what, const void* p, uint32_t ld, uint32_t multiple, uint64_t wide,
               uintptr_t align) {
  if (ld < wide || ld % multiple != 0)
    return fail(DH_EINVAL, "%s: row stride %u of %s must be a multiple of %u covering its %llu columns", op, ld, what,
                multiple, (unsigned long long)wide);
  if (p && !aligned(p, align)) return fail(DH_EINVAL, "%s: %s must be %u-byte aligned", op, what, (unsigned)align);
  return DH_OK;
}
}  // namespace

extern "C" {

int dh_attention_packed(dh_ctx* ctx, void* stream, const dh_packed_batch* batch, const void* q, uint32_t ldq,
                        const void* k, uint32_t ldk, const void* v, uint32_t ldv, uint32_t dtype, uint32_t heads,
                        uint32_t kv_heads, uint32_t head_dim, float scale, const float* gate, uint32_t ldg, void* y,
                        uint32_t ldy) {
  const char* const op = "attention_packed";
  if (!batch) return fail(DH_EINVAL, "%s: null batch", op);
  int rc = check_shape(op, batch->q_rows, batch->seqs, heads, kv_heads, head_dim);
  if (rc != DH_OK) return rc;
  if (dtype > 1) return fail(DH_EINVAL, "%s: dtype %u is not one of 0 (fp16), 1 (bf16)", op, dtype);
  if (!(std::fabs(scale) <= 0x1p127f)) return fail(DH_EINVAL, "%s: scale must be finite and at most 2^127", op);
  const uint64_t wide = (uint64_t)heads * head_dim, narrow = (uint64_t)kv_heads * head_dim;
  rc = check_rows(op, "q", q, ldq, 8, wide, 16);
  if (rc == DH_OK) rc = check_rows(op, "k", k, ldk, 8, narrow, 16);
  if (rc == DH_OK) rc = check_rows(op, "v", v, ldv, 8, narrow, 16);
  if (rc == DH_OK) rc = check_rows(op, "y", y, ldy, 4, wide, 8);
  if (rc == DH_OK && gate) rc = check_rows(op, "gate", gate, ldg, 4, wide, 16);
  if (rc != DH_OK) return rc;
  if (ldk > kMostStride || ldv > kMostStride)
    return fail(DH_EINVAL, "%s: row strides %u and %u of k and v must be at most 2^24", op, ldk, ldv);
  if ((batch->q0 && !aligned(batch->q0, 4)) || (batch->k0 && !aligned(batch->k0, 4)))
    return fail(DH_EINVAL, "%s: q0 and k0 must be 4-byte aligned", op);
  if (!ctx) return fail(DH_EINVAL, "%s: null context", op);
  if (batch->q_rows == 0 || batch->seqs == 0) return ok();
  if (!batch->q0 || !batch->k0) return fail(DH_EINVAL, "%s: null pointer in the batch", op);
  if (!q || !y || (batch->k_rows && (!k || !v))) return fail(DH_EINVAL, "%s: null pointer", op);
  dh::PackArgs a{};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.gate = gate, a.y = (uint16_t*)y;
  a.q0 = batch->q0, a.k0 = batch->k0;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldg = ldg, a.ldy = ldy;
  a.seqs = batch->seqs, a.q_rows = batch->q_rows, a.k_rows = batch->k_rows;
  a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.group_inv = ((1u << 21) + a.group - 1) / a.group;
  a.scale = scale;
  const dh::PackPlan plan = dh::packed_plan(batch->q_rows, batch->seqs, heads, kv_heads, head_dim, batch->max_k, ctx->cus);
  a.slots = plan.slots, a.runs = plan.runs, a.min_run = plan.min_run;
  if (plan.ws_bytes) {
    rc = ensure_aux(ctx, (hipStream_t)stream, plan.ws_bytes, &a.ws);
    if (rc != DH_OK) return rc;
    mark(ctx, kKidPackedMerge);
  }
  mark(ctx, plan.wide ? kKidPackedWide : kKidPacked);
  return hip_status(plan.wide ? dh::launch_packed_wide(a, head_dim, dtype == 1, (hipStream_t)stream)
                              : dh::launch_packed_narrow(a, head_dim, dtype == 1, (hipStream_t)stream),
                    op);
}

int dh_attention_packed_ws(dh_ctx* ctx, void* stream, uint32_t q_rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads,
                           uint32_t head_dim) {
  int rc = check_shape("attention_packed_ws", q_rows, seqs, heads, kv_heads, head_dim);
  if (rc != DH_OK) return rc;
  if (!ctx) return fail(DH_EINVAL, "attention_packed_ws: null context");
  if (q_rows == 0 || seqs == 0) return ok();
  // Runs are as many whatever the call; there are at most kPackSlots tiles.
  const uint64_t bytes =
      dh::packed_run_bytes(std::max(1u, ctx->cus / kv_heads), dh::kPackSlots, kv_heads, head_dim);
  float* ws = nullptr;
  return ensure_aux(ctx, (hipStream_t)stream, bytes, &ws);
}

}  // extern "C"

namespace dh_api {

size_t packed_warm_bytes() { return dh::packed_run_bytes(1, 1, 1, 64) + 64; }

int packed_warm(dh_ctx* ctx, hipStream_t s, void* mem) {
  // one row that belongs to no sequence: every kernel ends at once
  dh::PackArgs a{};
  a.q = a.k = a.v = (const uint16_t*)mem;
  a.q0 = a.k0 = (const uint32_t*)mem;
  a.y = (uint16_t*)mem;
  a.ws = (float*)mem;
  a.ldq = a.ldk = a.ldv = a.ldy = 64;
  a.seqs = a.q_rows = a.k_rows = a.kv_heads = a.group = a.slots = a.runs = a.min_run = 1;
  a.group_inv = 1u << 21;
  mark(ctx, kKidPackedWide);
  mark(ctx, kKidPacked);
  mark(ctx, kKidPackedMerge);
  int rc = hip_status(dh::launch_packed_wide(a, 64, false, s), "attention_packed");
  if (rc == DH_OK) rc = hip_status(dh::launch_packed_narrow(a, 64, false, s), "attention_packed");
  return rc;
}

}  // namespace dh_api
