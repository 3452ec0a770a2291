// C ABI of the rotary embedding and the 8-bit paged cache (include/decide_hip.h, "The 8-bit paged key/value cache").
// Contract violations return DH_EINVAL with a message; nothing is launched after a failed check.
#include <algorithm>
#include <cmath>

#include "api_internal.h"
#include "kv8.h"

using namespace dh_api;

namespace {
bool misaligned(const void* p, uintptr_t a) { return p && !aligned(p, a); }
uint32_t size_of(uint32_t dtype) { return dtype == 2 ? 4 : 2; }

int check_dtype(const char* op, const char* what, uint32_t dtype) {
  if (dtype > 2) return fail(DH_EINVAL, "%s: %s %u is not one of 0 (fp16), 1 (bf16), 2 (fp32)", op, what, dtype);
  return DH_OK;
}

int check_rope(const char* op, const dh_rope_spec* p) {
  if (p->head_dim == 0 || p->head_dim % 4 != 0 || p->head_dim > 256)
    return fail(DH_EINVAL, "%s: head_dim = %u must be a multiple of 4 in 4..256", op, p->head_dim);
  if (p->rot < 2 || p->rot % 2 != 0 || p->rot > p->head_dim)
    return fail(DH_EINVAL, "%s: rot = %u must be even in 2..%u", op, p->rot, p->head_dim);
  if (p->layout > DH_ROPE_INTERLEAVED)
    return fail(DH_EINVAL, "%s: layout %u is not DH_ROPE_HALF or DH_ROPE_INTERLEAVED", op, p->layout);
  if (!p->inv_freq) return fail(DH_EINVAL, "%s: inv_freq is null", op);
  if (misaligned(p->inv_freq, 4) || misaligned(p->norm_w, 16))
    return fail(DH_EINVAL, "%s: inv_freq must be 4-byte and norm_w 16-byte aligned", op);
  if (!std::isfinite(p->amp)) return fail(DH_EINVAL, "%s: amp must be finite", op);
  if (p->norm_w && (!(p->eps > 0.0f) || !std::isfinite(p->eps)))
    return fail(DH_EINVAL, "%s: eps must be positive and finite", op);
  return DH_OK;
}

dh::RopeArgs rope_args(const dh_rope_spec* p) {
  if (!p) return dh::RopeArgs{};
  return dh::RopeArgs{p->inv_freq, p->norm_w, p->head_dim, p->rot, p->layout, p->add_one, p->eps, p->amp};
}

// Rows of `heads` heads at stride ld
int check_rows(const char* op, const char* what, const void* p, uint32_t ld, uint32_t dtype, uint64_t wide) {
  if (ld < wide || ld % 4 != 0)
    return fail(DH_EINVAL, "%s: row stride %u of %s must be a multiple of 4 covering its %llu columns", op, ld, what,
                (unsigned long long)wide);
  if (misaligned(p, 4 * size_of(dtype)))
    return fail(DH_EINVAL, "%s: %s must be %u-byte aligned", op, what, 4 * size_of(dtype));
  return DH_OK;
}

int check_cache(const char* op, const dh_kv8_cache* c) {
  if (!c) return fail(DH_EINVAL, "%s: null cache", op);
  if (c->kv_heads < 1 || c->kv_heads > 1024)
    return fail(DH_EINVAL, "%s: kv_heads = %u must be in 1..1024", op, c->kv_heads);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(DH_EINVAL, "%s: head_dim = %u must be 64, 128 or 256", op, c->head_dim);
  if (c->format > DH_KV8_INT8)
    return fail(DH_EINVAL, "%s: format %u is not DH_KV8_E4M3 or DH_KV8_INT8", op, c->format);
  if (c->pages < 1 || c->layers < 1) return fail(DH_EINVAL, "%s: a cache has at least one page and one layer", op);
  if (!c->pool) return fail(DH_EINVAL, "%s: the pool is null", op);
  if (misaligned(c->pool, 128)) return fail(DH_EINVAL, "%s: the pool must be 128-byte aligned", op);
  return DH_OK;
}

constexpr uint64_t kMaxThreads = UINT32_MAX;  // of a launch, in a dimension

int check_batch(const char* op, const dh_kv8_batch* b) {
  if (!b) return fail(DH_EINVAL, "%s: null batch", op);
  if (b->rows && b->seqs && (!b->table || !b->row0 || !b->qpos)) return fail(DH_EINVAL, "%s: null pointer in the batch", op);
  if (misaligned(b->table, 4) || misaligned(b->row0, 4) || misaligned(b->qpos, 4))
    return fail(DH_EINVAL, "%s: table, row0 and qpos must be 4-byte aligned", op);
  return DH_OK;
}

dh::KvArgs kv_args(const dh_kv8_cache* c, uint32_t layer, const dh_kv8_batch* b) {
  const uint64_t bytes = dh_kv8_page_bytes(c->kv_heads, c->head_dim);
  return dh::KvArgs{(uint8_t*)c->pool + (uint64_t)layer * c->pages * bytes, bytes, c->pages, c->kv_heads, b->table,
                    b->row0, b->qpos, b->ld_table, b->seqs, b->rows};
}

int check_heads(const char* op, const dh_kv8_cache* c, uint32_t heads) {
  if (heads < 1 || heads % c->kv_heads != 0 || heads / c->kv_heads > 1024)
    return fail(DH_EINVAL, "%s: heads = %u must be a multiple of the %u kv heads, at most 1024 for each", op, heads,
                c->kv_heads);
  return DH_OK;
}

// Work items are numbered in 32 bits; a tile's merge takes up to four workgroups.
int check_attention_size(const char* op, const dh_kv8_cache* c, uint32_t rows, uint32_t seqs, uint32_t heads) {
  const uint64_t tiles = ((uint64_t)rows * (heads / c->kv_heads)) / 16 + seqs;
  if ((uint64_t)rows * heads > UINT32_MAX || tiles * c->kv_heads * 4 > kMaxThreads / 512)
    return fail(DH_EINVAL, "%s: %u rows x %u heads over %u sequences exceed one launch; split the call", op, rows, heads,
                seqs);
  return DH_OK;
}
}  // namespace

extern "C" {

uint64_t dh_kv8_page_bytes(uint32_t kv_heads, uint32_t head_dim) {
  if (kv_heads < 1 || kv_heads > 1024 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  const uint64_t bytes = (uint64_t)kv_heads * (2 * DH_KV8_PAGE * head_dim + 2 * (DH_KV8_PAGE / DH_KV8_BLOCK) * 4);
  return (bytes + 127) / 128 * 128;
}

int dh_rope(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, uint32_t x_dtype, void* y, uint32_t ldy,
            uint32_t y_dtype, const uint32_t* pos, uint32_t rows, uint32_t heads, const dh_rope_spec* spec) {
  if (!spec) return fail(DH_EINVAL, "rope: null spec");
  int rc = check_rope("rope", spec);
  if (rc == DH_OK) rc = check_dtype("rope", "x_dtype", x_dtype);
  if (rc == DH_OK) rc = check_dtype("rope", "y_dtype", y_dtype);
  const uint64_t wide = (uint64_t)heads * spec->head_dim;
  if (rc == DH_OK) rc = check_rows("rope", "x", x, ldx, x_dtype, wide);
  if (rc == DH_OK) rc = check_rows("rope", "y", y, ldy, y_dtype, wide);
  if (rc != DH_OK) return rc;
  if (misaligned(pos, 4)) return fail(DH_EINVAL, "rope: pos must be 4-byte aligned");
  if (rows > kMaxThreads / 256) return fail(DH_EINVAL, "rope: %u rows exceed one launch; split the call", rows);
  if (x && x == y && (x_dtype != y_dtype || ldx != ldy))
    return fail(DH_EINVAL, "rope: y may be x only with its dtype and row stride");
  if (!ctx) return fail(DH_EINVAL, "rope: null context");
  if (rows && heads && (!x || !y || !pos)) return fail(DH_EINVAL, "rope: null pointer");
  if (rows && heads) mark(ctx, kKidRope);
  return hip_status(dh::launch_rope(x, ldx, x_dtype, y, ldy, y_dtype, pos, rows, heads, rope_args(spec),
                                    (hipStream_t)stream),
                    "rope");
}

int dh_rope_freqs(uint32_t rot, double base, uint32_t kind, double factor, double low, double high,
                  uint32_t trained_len, float* inv_freq, float* amp) {
  if (rot < 2 || rot % 2 != 0 || rot > 256) return fail(DH_EINVAL, "rope_freqs: rot = %u must be even in 2..256", rot);
  if (!(base > 0.0) || !std::isfinite(base)) return fail(DH_EINVAL, "rope_freqs: base must be positive and finite");
  if (kind > DH_ROPE_PARTS) return fail(DH_EINVAL, "rope_freqs: kind %u is not one of DH_ROPE_PLAIN..DH_ROPE_PARTS", kind);
  if (kind != DH_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
    return fail(DH_EINVAL, "rope_freqs: factor must be finite and at least 1");
  if (kind == DH_ROPE_BASE && rot < 4) return fail(DH_EINVAL, "rope_freqs: DH_ROPE_BASE needs rot > 2");
  if (kind == DH_ROPE_PARTS && (!(low >= 0.0) || !(high > low) || !std::isfinite(high) || trained_len < 1))
    return fail(DH_EINVAL, "rope_freqs: DH_ROPE_PARTS needs 0 <= low < high and a trained_len");
  if (!inv_freq || !amp) return fail(DH_EINVAL, "rope_freqs: null pointer");
  if (kind == DH_ROPE_BASE) base *= std::pow(factor, rot / (rot - 2.0));
  for (uint32_t i = 0; i < rot / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot);
    if (kind == DH_ROPE_LINEAR) f /= factor;
    if (kind == DH_ROPE_PARTS) {
      const double turns = trained_len * f / 6.283185307179586;
      const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
      f = f / factor * (1.0 - keep) + f * keep;
    }
    inv_freq[i] = (float)f;
  }
  *amp = kind == DH_ROPE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return ok();
}

int dh_kv8_append(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t layer, const dh_kv8_batch* batch,
                  const void* k, uint32_t ldk, const void* v, uint32_t ldv, uint32_t dtype, const dh_rope_spec* rope) {
  int rc = check_cache("kv8_append", cache);
  if (rc == DH_OK) rc = check_batch("kv8_append", batch);
  if (rc == DH_OK) rc = check_dtype("kv8_append", "dtype", dtype);
  if (rc == DH_OK && rope) rc = check_rope("kv8_append", rope);
  if (rc != DH_OK) return rc;
  if (layer >= cache->layers) return fail(DH_EINVAL, "kv8_append: layer %u of %u", layer, cache->layers);
  if (rope && rope->head_dim != cache->head_dim)
    return fail(DH_EINVAL, "kv8_append: the rotation's head_dim = %u is not the cache's %u", rope->head_dim,
                cache->head_dim);
  const uint64_t wide = (uint64_t)cache->kv_heads * cache->head_dim;
  rc = check_rows("kv8_append", "k", k, ldk, dtype, wide);
  if (rc == DH_OK) rc = check_rows("kv8_append", "v", v, ldv, dtype, wide);
  if (rc != DH_OK) return rc;
  if ((uint64_t)batch->rows / DH_KV8_BLOCK + 2 * (uint64_t)batch->seqs > kMaxThreads / 256)
    return fail(DH_EINVAL, "kv8_append: %u rows of %u sequences exceed one launch; split the call", batch->rows,
                batch->seqs);
  if (!ctx) return fail(DH_EINVAL, "kv8_append: null context");
  if (batch->rows && batch->seqs && (!k || !v)) return fail(DH_EINVAL, "kv8_append: null pointer");
  if (batch->rows && batch->seqs) mark(ctx, kKidKv8Append);
  return hip_status(dh::launch_kv8_append(kv_args(cache, layer, batch), cache->head_dim, cache->format == DH_KV8_INT8, k,
                                          ldk, v, ldv, dtype, rope_args(rope), ctx->cus, (hipStream_t)stream),
                    "kv8_append");
}

int dh_kv8_attention(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t layer, const dh_kv8_batch* batch,
                     const uint16_t* q, uint32_t ldq, uint32_t heads, float scale, const float* gate, uint32_t ldg,
                     uint16_t* y, uint32_t ldy, uint32_t max_tokens) {
  int rc = check_cache("kv8_attention", cache);
  if (rc == DH_OK) rc = check_batch("kv8_attention", batch);
  if (rc == DH_OK) rc = check_heads("kv8_attention", cache, heads);
  if (rc == DH_OK) rc = check_attention_size("kv8_attention", cache, batch->rows, batch->seqs, heads);
  if (rc != DH_OK) return rc;
  if (layer >= cache->layers) return fail(DH_EINVAL, "kv8_attention: layer %u of %u", layer, cache->layers);
  if (!std::isfinite(scale)) return fail(DH_EINVAL, "kv8_attention: scale must be finite");
  const uint64_t wide = (uint64_t)heads * cache->head_dim;
  if (ldq < wide || ldq % 8 != 0 || misaligned(q, 16))
    return fail(DH_EINVAL, "kv8_attention: q must be 16-byte aligned and ldq = %u a multiple of 8 covering %llu columns",
                ldq, (unsigned long long)wide);
  if (ldy < wide || ldy % 4 != 0 || misaligned(y, 8))
    return fail(DH_EINVAL, "kv8_attention: y must be 8-byte aligned and ldy = %u a multiple of 4 covering %llu columns",
                ldy, (unsigned long long)wide);
  if (gate && (ldg < wide || ldg % 4 != 0 || misaligned(gate, 16)))
    return fail(DH_EINVAL, "kv8_attention: gate must be 16-byte aligned and ldg = %u a multiple of 4 covering %llu columns",
                ldg, (unsigned long long)wide);
  if (!ctx) return fail(DH_EINVAL, "kv8_attention: null context");
  if (batch->rows == 0 || batch->seqs == 0) return ok();
  if (!q || !y) return fail(DH_EINVAL, "kv8_attention: null pointer");
  const dh::KvAttnPlan plan = dh::kv8_attention_plan(batch->rows, batch->seqs, heads, cache->kv_heads, cache->head_dim,
                                                     batch->ld_table, max_tokens, ctx->cus);
  float* aux = nullptr;
  if (plan.ws_bytes) {
    rc = ensure_aux(ctx, (hipStream_t)stream, plan.ws_bytes, &aux);
    if (rc != DH_OK) return rc;
    mark(ctx, kKidKv8Combine);
  }
  mark(ctx, kKidKv8Attn);
  return hip_status(dh::launch_kv8_attention(kv_args(cache, layer, batch), cache->head_dim,
                                             cache->format == DH_KV8_INT8, (const _Float16*)q, ldq, heads, scale, gate,
                                             ldg, (_Float16*)y, ldy, aux, plan, ctx->cus, (hipStream_t)stream),
                    "kv8_attention");
}

int dh_kv8_attention_ws(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t rows, uint32_t seqs,
                        uint32_t heads, uint32_t max_tokens) {
  int rc = check_cache("kv8_attention_ws", cache);
  if (rc == DH_OK) rc = check_heads("kv8_attention_ws", cache, heads);
  if (rc == DH_OK) rc = check_attention_size("kv8_attention_ws", cache, rows, seqs, heads);
  if (rc != DH_OK) return rc;
  if (!ctx) return fail(DH_EINVAL, "kv8_attention_ws: null context");
  if (rows == 0 || seqs == 0) return ok();
  const uint64_t bytes =
      dh::kv8_attention_ws_bytes(rows, heads, cache->kv_heads, cache->head_dim, max_tokens, ctx->cus);
  float* aux = nullptr;
  if (bytes) {
    rc = ensure_aux(ctx, (hipStream_t)stream, bytes, &aux);
    if (rc != DH_OK) return rc;
  }
  return ok();
}

int dh_kv8_copy_pages(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, const uint32_t* src, const uint32_t* dst,
                      uint32_t n) {
  int rc = check_cache("kv8_copy_pages", cache);
  if (rc != DH_OK) return rc;
  if (misaligned(src, 4) || misaligned(dst, 4))
    return fail(DH_EINVAL, "kv8_copy_pages: src and dst must be 4-byte aligned");
  const uint64_t bytes = dh_kv8_page_bytes(cache->kv_heads, cache->head_dim);
  if ((bytes / 16384 + 1) * (uint64_t)std::min(n, cache->pages) > kMaxThreads / 256 / cache->layers ||
      n > cache->pages)
    return fail(DH_EINVAL, "kv8_copy_pages: %u pairs for %u pages in %u layers exceed one launch", n, cache->pages,
                cache->layers);
  if (!ctx) return fail(DH_EINVAL, "kv8_copy_pages: null context");
  if (n && (!src || !dst)) return fail(DH_EINVAL, "kv8_copy_pages: null pointer");
  if (n) mark(ctx, kKidKv8Copy);
  return hip_status(dh::launch_kv8_copy_pages((uint8_t*)cache->pool, bytes, cache->pages, cache->layers, src, dst, n,
                                              (hipStream_t)stream),
                    "kv8_copy_pages");
}

}  // extern "C"

namespace dh_api {

size_t kv8_warm_bytes() { return 131072; }

int kv8_warm(dh_ctx* ctx, hipStream_t s, void* mem) {
  // one page of one head of 64 dims at 0 (a second one behind it), everything else zeros: one sequence, one row at
  // position 0, in page 0
  char* const base = (char*)mem;
  const dh_kv8_cache cache{base, 2, 1, 1, 64, DH_KV8_E4M3};
  static_assert(2 * 8320 <= 32768 && 2 * 16 * 66 * 4 + 4 * (dh::kKvMaxSlots + 1) <= 131072 - 49152, "what lies where");
  uint32_t* const u = (uint32_t*)(base + 32768);      // table, row0's 0, qpos, src: zeros
  float* const x = (float*)(base + 36864);
  uint16_t* const y = (uint16_t*)(base + 40960);
  const dh_rope_spec rope{x, nullptr, 64, 64, DH_ROPE_HALF, 0, 0.f, 1.f};
  const dh_kv8_batch batch{u, u, u, 1, 1, 1};  // row0 {0, 0}: the row belongs to no sequence, every kernel ends at once
  int rc = dh_rope(ctx, s, x, 64, 2, y, 64, 0, u, 1, 1, &rope);
  if (rc == DH_OK) rc = dh_kv8_append(ctx, s, &cache, 0, &batch, x, 64, x, 64, 2, &rope);
  if (rc == DH_OK) {
    mark(ctx, kKidKv8Attn);
    mark(ctx, kKidKv8Combine);
    // one run, with the combine; one wide tile
    for (const dh::KvAttnPlan& plan : {dh::KvAttnPlan{1, 1, 8, false, 0}, dh::KvAttnPlan{1, 0, 0, true, 0}})
      if (rc == DH_OK)
        rc = hip_status(dh::launch_kv8_attention(kv_args(&cache, 0, &batch), 64, false, (const _Float16*)x, 64, 1, 1.f,
                                                 nullptr, 0, (_Float16*)y, 64, (float*)(base + 49152), plan, ctx->cus, s),
                        "kv8_attention");
  }
  if (rc == DH_OK) rc = dh_kv8_copy_pages(ctx, s, &cache, u, u, 1);  // page 0 onto itself
  return rc;
}

}  // namespace dh_api
