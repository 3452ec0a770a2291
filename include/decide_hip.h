/*
 * decide_hip.h — C ABI of the MI355X (gfx950) prefill GEMM path of decide.
 *
 * Every entry point below replaces one method of decide-engine's Metal
 * backend; the reference interface each one stands in for is cited beside it
 * (paths relative to the decide source tree). All entry points:
 *   - take plain device pointers (already offset to the slice they address)
 *     and element counts, never host containers or framework types;
 *   - enqueue onto the caller's HIP stream (`stream`, a hipStream_t; NULL is
 *     the legacy default stream) and never synchronise, so stream order plays
 *     the part of decide's single serial compute encoder;
 *   - return DH_OK or a DH_E* status; on a status other than DH_OK the
 *     calling thread's dh_last_error() holds a one-line message. Contract
 *     violations are reported before anything is launched.
 * The library never allocates or frees caller memory. A context owns only its
 * launch plan and, per stream that uses it, two workspaces (device memory it
 * allocates itself): the split-K partials and the forward kernels' scratch
 * (attention's key pieces and the chunked recurrence's per-chunk matrices).
 * Threads and streams (decide: Gemm is Sync, its pipeline cache behind a
 * mutex, kernels/gemm.rs:46-55, 115-124):
 *   - a context may be shared by host threads and by streams. Its plan is
 *     fixed after dh_ctx_create (dh_gemm_force aside, which is atomic and
 *     meant for tuning), and each stream gets its own workspaces, allocated on
 *     that stream's first call that needs them and grown under an internal
 *     lock, so calls on different streams may overlap;
 *   - a workspace that grows is replaced, and the buffer it replaces stays
 *     allocated until dh_ctx_destroy, so a graph captured earlier
 *     (dh_model_capture) never reads freed memory; a graph keeps using the
 *     workspaces of the stream it was captured on, so its replays must not
 *     overlap other calls on that stream's workspaces;
 *   - a workspace never grows while its stream is being captured: such a call
 *     returns DH_EINVAL (size it first with dh_warm_up or an eager call of the
 *     same size on that stream);
 *   - a stream's workspaces stay with the context until dh_ctx_destroy, and a
 *     stream created later with the same handle reuses them: destroy a stream
 *     only after its work has finished;
 *   - dh_gemm_nt_noalloc's scratch is one array per GPU, shared by every
 *     context on it: its calls must not overlap on one GPU;
 *   - a dh_model (its activations, caches and request state) serves one
 *     request at a time: calls on one model must not overlap.
 */
#ifndef DECIDE_HIP_H
#define DECIDE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
#define DH_OK 0
#define DH_EINVAL 1   /* a contract violation (shape, stride, alignment, enum) */
#define DH_ELAUNCH 2  /* hipLaunchKernel / hipGetLastError reported an error */
#define DH_ENOMEM 3   /* the split-K workspace could not be allocated */
#define DH_EDEVICE 4  /* no usable gfx950 device, or a HIP runtime call failed */

/* Epilogues: exactly decide's `Epilogue` codes (crates/decide-engine/src/kernels/gemm.rs:15-26). */
#define DH_EPI_STORE_F32 0u  /* y fp32 [M, N] = acc */
#define DH_EPI_STORE_F16 1u  /* y fp16 [M, N] = half(acc) */
#define DH_EPI_ADD_F32 2u    /* y fp32 [M, N] += acc (residual add) */
#define DH_EPI_SWIGLU_F16 3u /* y fp16 [M, N/2] = silu(gate) * up over 16-column gate|up blocks */

/* The gate|up interleave block of DH_EPI_SWIGLU_F16 (decide's SWIGLU_BLOCK, config.rs:31). */
#define DH_SWIGLU_BLOCK 16u

/* dh_ctx_create flags. */
#define DH_GEMM_REFERENCE 1u /* every GEMM runs the simple M-independent kernel (decide's
                                DECIDE_GEMM=baseline, kernels/gemm.rs:56-65) */
#define DH_DELTA_CHUNKED 2u    /* dh_gated_delta always runs the chunked recurrence */
#define DH_DELTA_SEQUENTIAL 4u /* dh_gated_delta always runs the token-by-token kernel (with neither flag:
                                  chunked for t >= DH_DELTA_CHUNK_MIN_T; below that in blocks of 16 tokens, and
                                  token by token for t <= 36; the choice decide makes with DECIDE_DELTA,
                                  kernels/delta.rs:36-49) */
#define DH_DELTA_CHUNK_MIN_T 320u

typedef struct dh_ctx dh_ctx;

/* One member of a grouped GEMM: Y_i = X · W_iᵀ with its own epilogue. */
typedef struct dh_gemm_member {
  const void* w;   /* fp16 [n, k], row stride ldw (elements) */
  void* y;         /* output, row stride ldy in elements of its output type */
  uint32_t ldw;
  uint32_t ldy;
  uint32_t n;
  uint32_t epi;    /* DH_EPI_* */
} dh_gemm_member;

/* A launch plan as the planner chose it (for tests, tuning and reports). */
#define DH_GEMM_STREAM_VARIANT 64u /* dh_gemm_plan.variant of the small-M weight-streaming kernel (M <= 16,
                                      N <= 4096, K % 128 == 0; decide's gemm_nt_small, gemm_fast.metal:429-566): 16 × 32
                                      output tiles, 4 waves, W streamed from HBM straight into registers */
typedef struct dh_gemm_plan {
  uint32_t variant;     /* index into the compiled tile-kernel menu, or DH_GEMM_STREAM_VARIANT */
  uint32_t bm, bn;      /* output tile (rows, columns) */
  uint32_t waves;       /* wavefronts per workgroup */
  uint32_t splits;      /* split-K factor (1 = none) */
  uint32_t workgroups;  /* grid size of the tile kernel */
  uint64_t ws_bytes;    /* split-K workspace the launch needs */
  uint32_t order;       /* work order of the tile kernel: 0 = M tiles fastest; g > 0 = column stripes in groups of
                           g, each group's stripes fastest (chosen per launch so that each XCD's L2 sees a compact
                           block of X rows and W columns); the outputs are the same bits whatever the order. The
                           environment variable DH_GEMM_TILE_GROUP=<g> (0..64), read once per process, fixes it
                           for every launch (for measurements; the library reads no other variable) */
} dh_gemm_plan;

/* --- context (decide: Gemm::new / Gemm::with_impl, kernels/gemm.rs:56-83;
 *     Kernels::new, kernels/mod.rs:53-67) ---
 * Creates a context on the current device (which must be gfx950). Its first
 * creation on a device also takes that device's no-allocation scratch
 * (DH_NOALLOC_SCRATCH_BYTES, shared by every context on the device until the
 * process ends; see dh_gemm_nt_noalloc). Workspaces are per stream (above). */
int dh_ctx_create(uint32_t flags, dh_ctx** out);
void dh_ctx_destroy(dh_ctx* ctx);
/* The calling thread's message for its last failed call ("" if none). */
const char* dh_last_error(void);
/* Library version string. */
const char* dh_version(void);

/* Loads every kernel of the menu and runs each once on a tiny shape, and sizes
 * `stream`'s workspaces so that a timed forward of up to `max_m` rows on that
 * stream neither loads code nor allocates (decide: Gemm::warm_up,
 * gemm.rs:87-107): the split-K workspace for the largest split plan of decide's
 * engine shapes at any M up to max_m, and the forward kernels' workspace, whose
 * attention part is sized even for a GEMM-only context: 8.4 MB at max_m = 1,
 * growing with max_m to 84.5 MB (plus the chunked recurrence's, from
 * DH_DELTA_CHUNK_MIN_T rows). max_m must be in 1..DH_PLAN_MAX_ROWS. */
#define DH_PLAN_MAX_ROWS 65536u
int dh_warm_up(dh_ctx* ctx, void* stream, uint32_t max_m);
/* Distinct kernels launched through this context so far; after dh_warm_up it
 * must not grow (decide: Gemm::fast_pipelines, gemm.rs:109-113; engine.rs:163-172). */
uint32_t dh_variants_loaded(const dh_ctx* ctx);

/* --- the GEMM operator (decide: Gemm::gemm, kernels/gemm.rs:126-176) ---
 * y = epi(X · Wᵀ): X fp16 [m, k] row stride ldx, W fp16 [n, k] row stride ldw,
 * fp32 accumulation, ldy in elements of y's type. Contract (gemm.rs:140-163):
 * n % 32 == 0, k % 32 == 0, m >= 1, ldx >= k, ldw >= k, ldy >= n (n/2 for
 * SwiGLU), ldx % 8 == 0, ldw % 8 == 0, ldy even, x and w 16-byte aligned, y
 * 8-byte (fp32 outputs) or 4-byte (fp16 outputs) aligned, and X's and W's rows
 * each within 4 GiB of their base: ((m - 1)·ldx + k)·2 and ((n - 1)·ldw + k)·2
 * at most 2^32 - 1 bytes (no such limit in decide; its engine shapes are far
 * below it). A DH_GEMM_REFERENCE context checks only the first part, as
 * decide's baseline does (gemm.rs:140-156): shapes and strides, plus each
 * operand aligned to its own element size. */
int dh_gemm_nt(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, const void* w, uint32_t ldw, void* y,
               uint32_t ldy, uint32_t m, uint32_t n, uint32_t k, uint32_t epi);

/* The same GEMM without any allocation: no hipMalloc, hipFree or allocating
 * library call, for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid it). decide has no
 * counterpart. Split-K partials go to a device array of the library, file
 * scope, DH_NOALLOC_SCRATCH_BYTES on each GPU, which that GPU holds from the
 * first dh_ctx_create on it until the process ends. The planner picks among
 * plans whose partials fit it; a forced plan (dh_gemm_force) that needs more
 * is refused with DH_EINVAL. Same contract and arguments as dh_gemm_nt; the
 * context's device must be current. Every call on one GPU shares that array
 * and nothing in it needs clearing (each split-K launch writes every partial
 * it reads), but calls that overlap on one GPU (different streams, or
 * different contexts) race on it. */
#define DH_NOALLOC_SCRATCH_BYTES 50331648u /* 48 MiB */
int dh_gemm_nt_noalloc(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, const void* w, uint32_t ldw, void* y,
                       uint32_t ldy, uint32_t m, uint32_t n, uint32_t k, uint32_t epi);

/* Grouped form: every member shares X (m rows, k columns) and is computed in
 * ONE launch. decide has no grouped call; it fuses members by concatenating
 * their weight rows offline (convert.rs:204-245: qkv|z|b|a, q|gate|k|v,
 * gate|up) and calls Gemm::gemm once. This is that launch without the
 * concatenated copy. Same per-member contract as dh_gemm_nt; count in 1..8. */
int dh_gemm_nt_grouped(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, uint32_t m, uint32_t k,
                       const dh_gemm_member* members, uint32_t count);

/* The plan dh_gemm_nt would use (no launch, no device needed; decide:
 * gemm_configs::plan, crates/decide-metal/src/gemm_configs.rs:311-314). */
int dh_gemm_plan_for(const dh_ctx* ctx, uint32_t m, uint32_t n, uint32_t k, uint32_t epi, dh_gemm_plan* out);
/* The split-K workspace (bytes) that dh_gemm_nt's planner asks for at its
 * largest over every m in 1..max_m and every epilogue at (n, k), on this
 * context (no device needed; the planner runs once per m, so max_m is capped
 * at DH_PLAN_MAX_ROWS, about 0.15 s of host time per shape there). dh_warm_up
 * holds at least this for decide's engine shapes; a caller with other shapes
 * can size its own calls with it. */
int dh_gemm_ws_need(const dh_ctx* ctx, uint32_t max_m, uint32_t n, uint32_t k, uint64_t* out);
/* Forces the next GEMMs on this context, on every stream, to use `variant` and
 * `splits` (variant = UINT32_MAX restores the planner). For tuning sweeps
 * only: calls already running in other threads see the change at their next
 * plan. */
int dh_gemm_force(dh_ctx* ctx, uint32_t variant, uint32_t splits);
/* Number of compiled tile variants and the geometry of one of them: the tile's
 * rows and columns, its wavefronts (4, or 8 with two per SIMD) and the columns
 * of one wave position (with 8 waves, the two waves of a SIMD split it). */
uint32_t dh_gemm_variant_count(void);
int dh_gemm_variant_info(uint32_t variant, uint32_t* bm, uint32_t* bn, uint32_t* waves, uint32_t* wave_cols);

/* --- row gathers (decide: Head::gather_rows_f32 / gather_rows_f16,
 *     kernels/head.rs:28-46; kernels/head.metal:8-28) ---
 * out[i, :] = x[rowmap[i], :] for i < rows, h elements per row, bitwise. The
 * 2-byte form copies any 16-bit rows (fp16 activations, bf16 embedding rows). */
int dh_gather_rows_f32(dh_ctx* ctx, void* stream, const float* x, const uint32_t* rowmap, float* out,
                       uint32_t rows, uint32_t h);
int dh_gather_rows_f16(dh_ctx* ctx, void* stream, const uint16_t* x, const uint32_t* rowmap, uint16_t* out,
                       uint32_t rows, uint32_t h);

/* --- candidate-only LM head (decide: Head::final_head, kernels/head.rs:48-60;
 *     kernels/head.metal:30-59; cpu_ref::final_head, cpu_ref.rs:190-198) ---
 * For each of `rows` fp32 rows of x [rows, hidden]: zero-centred RMSNorm
 * (weight (1 + w), w fp32 [hidden], eps), then the fp32 dot product with the
 * bf16 rows of `table` [vocab, hidden] named by cand[r * max_cand + c] for
 * c < min(ncand[r], max_cand). Writes logits[r * max_cand + c]; entries past
 * ncand[r] are left untouched. decide fixes hidden = 2560 and max_cand = 62;
 * here both are parameters (hidden % 8 == 0, hidden <= 16384, 1 <= max_cand <= 524280).
 * Candidate ids >= vocab are a contract violation the kernel cannot see: the
 * caller validates ids (decide: forward.rs:1494-1537). */
int dh_final_head(dh_ctx* ctx, void* stream, const float* x, const float* w, const uint16_t* table,
                  const uint32_t* cand, const uint32_t* ncand, float* logits, uint32_t rows, uint32_t hidden,
                  uint32_t max_cand, float eps);

/* --- row RMSNorm, fp32 in, fp16 out (decide: Norm::rmsnorm, kernels/norm.rs:26-33;
 *     kernels/rmsnorm.metal:8-30) ---
 * y[r] = half(x[rowmap[r]] * rsqrt(mean(x^2) + eps) * (add_one ? 1 + w : w)).
 * Contract: h <= ld_in and h <= ld_out (norm.rs:27). */
int dh_rmsnorm_rows(dh_ctx* ctx, void* stream, const float* x, const float* w, uint16_t* y,
                    const uint32_t* rowmap, uint32_t rows, uint32_t h, uint32_t ld_in, uint32_t ld_out,
                    uint32_t add_one, float eps);

/* --- residual add fused with the norm that follows it (no single counterpart in decide: its forward runs
 *     the projection with the AddF32 epilogue, then rmsnorm over the same rows, forward.rs:1256-1282 with
 *     norm.rs:26-33) ---
 * y += X · Wᵀ (dh_gemm_nt with DH_EPI_ADD_F32, the same contract), then h[r] = half(y[r] * rsqrt(mean(y[r]^2)
 * + eps) * (add_one ? 1 + w : w)) for r < m (dh_rmsnorm_rows with rows r itself, h = n, ld_in = ldy,
 * ld_out = ldh). y and h are bitwise those of the two calls. Where the planner splits K, one kernel sums the
 * partials, adds the residual and norms each row, in place of the split-K reduce and the norm kernel.
 * Contract: as dh_gemm_nt, plus n >= 32 and n <= ldh. */
int dh_gemm_add_rmsnorm(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, const void* w, uint32_t ldw, float* y,
                        uint32_t ldy, uint32_t m, uint32_t n, uint32_t k, const float* norm_w, uint32_t add_one,
                        float eps, uint16_t* h, uint32_t ldh);

/* --- synthetic inputs (decide: the random-init role of testutil::uniform,
 *     testutil.rs:4-8, with the Gaussian shapes BASELINE asks for) ---
 * Fills n fp16 values with N(0, std) from a counter-based generator keyed by
 * seed: element i depends only on (seed, i), so fills are reproducible and
 * independent of launch shape. Used to random-initialise weights in place. */
int dh_fill_normal_f16(dh_ctx* ctx, void* stream, uint16_t* out, uint64_t n, uint64_t seed, float std);

/* --- weight layouts (decide: convert.rs:37-62, 74-90), host memory ---
 * Pure permutations / conversions of 16-bit row data, for building the fused
 * operands dh_gemm_nt consumes. */
/* gate, up: [n, k] each → out [2n, k] in blocks of `block` rows: g0 u0 g1 u1 …
 * (n % block == 0). */
int dh_interleave_gate_up(const uint16_t* gate, const uint16_t* up, uint16_t* out, uint32_t n, uint32_t k,
                          uint32_t block);
/* HF q_proj rows, per head [q_h (head_dim rows); gate_h (head_dim rows)] →
 * [all q rows | all gate rows]. src/out: [heads * 2 * head_dim, k]. */
int dh_deinterleave_q_gate(const uint16_t* src, uint16_t* out, uint32_t heads, uint32_t head_dim, uint32_t k);
/* bf16 bits → fp16 bits, round to nearest even. Returns DH_EINVAL if any finite
 * value overflows fp16 (decide aborts the conversion, convert.rs:168-173);
 * counts[0..3] = {values, subnormal, flushed to zero, overflow} if non-NULL. */
int dh_bf16_to_f16(const uint16_t* src, uint16_t* out, uint64_t n, uint64_t* counts);

/* ======================================================================
 * Forward kernels beside the GEMMs: the non-GEMM steps of decide's hybrid
 * decoder forward (forward.rs:1191-1254). Model constants are decide's
 * (config.rs:4-31): 16 key heads and 32 value heads of 128 dims in the
 * Gated-DeltaNet layers (CONV_DIM 8192 = q 2048 | k 2048 | v 4096), 16 query
 * heads over 4 kv heads of 256 dims in the attention layers.
 * ====================================================================== */

/* decide: Embed::embed (kernels/embed.rs:17; kernels/embed.metal). out fp32
 * [t, h] = the bf16 rows table[ids[i]] widened bitwise. h % 8 == 0, table and
 * out 16-byte aligned. ids < vocab is the caller's check (forward.rs:1494-1537). */
int dh_embed_bf16(dh_ctx* ctx, void* stream, const uint32_t* ids, const uint16_t* table, float* out, uint32_t t,
                  uint32_t h);

/* decide: Conv::conv_silu_l2 (kernels/conv.rs:20-35; cpu_ref::conv_silu_l2,
 * cpu_ref.rs:55-81). Reads the qkv columns 0..8192 of t rows of p (fp32, row
 * stride ldp) and prev, the 3 raw rows before them (fp32 [3, 8192], oldest
 * first); w is fp32 [8192, 4]. Writes fp32 q, k [t, 16, 128] (L2-normed, q also
 * scaled by 128^-1/2) and v [t, 32, 128]. ldp even and >= 8192; p, prev, q, k,
 * v 8-byte and w 16-byte aligned. */
int dh_conv_silu_l2(dh_ctx* ctx, void* stream, const float* p, const float* prev, const float* w, float* q, float* k,
                    float* v, uint32_t t, uint32_t ldp);
/* decide: Conv::conv_state_update (kernels/conv.rs:37-48; cpu_ref.rs:86-95).
 * prev_out [3, 8192] = the raw qkv rows t-3, t-2, t-1 (from prev_in where
 * negative). prev_out may be prev_in. */
int dh_conv_state_update(dh_ctx* ctx, void* stream, const float* p, const float* prev_in, float* prev_out, uint32_t t,
                         uint32_t ldp);

/* decide: Delta::gated_delta (kernels/delta.rs:53-80; cpu_ref::gated_delta,
 * cpu_ref.rs:101-129). fp32 throughout: q, k [t, 16, 128]; v, o [t, 32, 128];
 * a, b rows of stride ldab (value head h at column h); a_log, dt_bias [32];
 * state [32][128 dv][128 dk]. state_in may be state_out; with write_state 0
 * state_out is not written (and may be NULL). t >= 1, ldab >= 32; q, k and the
 * states 16-byte aligned. From t = DH_DELTA_CHUNK_MIN_T on (or always, in a
 * context created with DH_DELTA_CHUNKED) the recurrence runs 64 tokens at a
 * time as fp32 matrix products, in a context workspace that dh_warm_up sizes
 * for max_m tokens (a larger t grows it once). Below that it runs in blocks of
 * 16 tokens in one kernel, without a workspace, and for t <= 36 (or always,
 * with DH_DELTA_SEQUENTIAL) token by token. The three differ in rounding only;
 * a token whose inputs are not finite reaches only itself and later tokens
 * except in its own 64-token chunk of the chunked recurrence. */
int dh_gated_delta(dh_ctx* ctx, void* stream, const float* q, const float* k, const float* v, const float* a,
                   const float* b, const float* a_log, const float* dt_bias, const float* state_in, float* state_out,
                   float* o, uint32_t t, uint32_t ldab, uint32_t write_state);

/* decide: Conv::conv_silu_l2 then Delta::gated_delta on its outputs
 * (kernels/conv.rs:20-35, kernels/delta.rs:53-80; forward.rs:1203-1216), in one
 * call on the chunked recurrence: its prep kernel forms q, k and v from p, prev
 * and w itself, with dh_conv_silu_l2's arithmetic, so k and v never go through
 * memory. Results are bitwise those of dh_conv_silu_l2 followed by
 * dh_gated_delta on the chunked path, and q (the only conv output the rest of
 * the recurrence reads) is written as dh_conv_silu_l2 writes it. Arguments as
 * there: p's qkv columns 0..8192 of t rows (row stride ldp, even, >= 8192),
 * prev [3, 8192], w [8192, 4]; a, b rows of stride ldab; q [t, 16, 128] out.
 * Always the chunked path, whatever the context's DH_DELTA_* flags; p and prev
 * 8-byte, w, q and the states 16-byte aligned. */
int dh_conv_gated_delta_chunked(dh_ctx* ctx, void* stream, const float* p, const float* prev, const float* w, float* q,
                                const float* a, const float* b, const float* a_log, const float* dt_bias,
                                const float* state_in, float* state_out, float* o, uint32_t t, uint32_t ldp,
                                uint32_t ldab, uint32_t write_state);

/* decide: GNorm::gated_rmsnorm_silu (kernels/gnorm.rs:19-31; cpu_ref.rs:132-145).
 * y fp16 [t, 4096] = per (row, value head) RMSNorm of o over 128 dims with
 * weight w (fp32 [128], no +1), times silu(z); z rows of stride ldz. */
int dh_gated_rmsnorm_silu(dh_ctx* ctx, void* stream, const float* o, const float* z, const float* w, uint16_t* y,
                          uint32_t t, uint32_t ldz);

/* decide: Rope::q_norm_rope (kernels/rope.rs:25-37; cpu_ref::head_norm_rope,
 * cpu_ref.rs:149-162). For the 16 q heads (column 256 h) of rows of pq (fp32,
 * row stride ldq): zero-centred RMSNorm with qw (fp32 [256], applied as 1 + w),
 * RoPE on dims [0, 64) at position qpos[r] with inv_freq (fp32 [32]); writes
 * fp16 qo [rows, 16, 256]. ldq % 4 == 0; pq, qw 16-byte and qo 8-byte aligned. */
int dh_q_norm_rope(dh_ctx* ctx, void* stream, const float* pq, const float* qw, const float* inv_freq,
                   const uint32_t* qpos, uint16_t* qo, uint32_t rows, uint32_t ldq);
/* decide: Rope::kv_norm_rope (kernels/rope.rs:39-54). Row r at position
 * pos0 + r: the 4 k heads at column kcol, normed and rotated like q, into the
 * fp16 K cache kc [pos][4][256]; the 4 v heads at column vcol copied into the
 * V cache vc. pos0 + rows <= 8192 (decide's MAX_TOKENS cache rows). */
int dh_kv_norm_rope(dh_ctx* ctx, void* stream, const float* pkv, const float* kw, const float* inv_freq, uint16_t* kc,
                    uint16_t* vc, uint32_t rows, uint32_t ldkv, uint32_t kcol, uint32_t vcol, uint32_t pos0);

/* decide: Attn::attention (kernels/attn.rs:80-125; cpu_ref::attention,
 * cpu_ref.rs:167-188). q fp16 [rows, 16, 256]; row r at position qpos[r]
 * attends to cache rows 0..=qpos[r] of kc/vc (fp16 [pos][4][256]); the gate is
 * read from pq (fp32, row stride ldq) at column 4096 + 256 h + d. y fp16
 * [rows, 4096] = softmax(q·kᵀ/16)·v ⊙ σ(gate). rows >= 1, ldq >= 8192 and even;
 * q, kc, vc 16-byte, pq 8-byte, qpos and y 4-byte aligned. Cache rows
 * 0..=max(qpos) must hold finite values. Long query blocks' keys are split
 * across workgroups (cut points at fixed key offsets, sized as if the rows sat
 * at positions 0..rows-1) and merged through the context's forward-kernel
 * workspace, which dh_warm_up sizes. The cut length depends only on `rows`:
 * a row's bits depend on its own query, position and cache rows, and, when its
 * keys span a cut, on the call's row count (rounding only). */
int dh_attention(dh_ctx* ctx, void* stream, const uint16_t* q, const uint16_t* kc, const uint16_t* vc, const float* pq,
                 const uint32_t* qpos, uint16_t* y, uint32_t rows, uint32_t ldq);

/* Random-init fill for every parameter dtype (the role of decide's
 * testutil::uniform, testutil.rs:4-8, with the Gaussians BASELINE asks for):
 * n values N(mean, std) as fp16 (dtype 0), bf16 (1) or fp32 (2), element i a
 * function of (seed, i) only — the generator of dh_fill_normal_f16. */
int dh_fill_normal(dh_ctx* ctx, void* stream, void* out, uint64_t n, uint64_t seed, float mean, float std,
                   uint32_t dtype);

/* ======================================================================
 * The hybrid decoder forward (decide: Forward, crates/decide-engine/src/
 * forward.rs): the host that strings the kernels above into decide's layer
 * order with its buffers and fp16 rounding points, over one stream.
 * dh_model_forward runs the full route from position 0 as one chunk of all
 * T rows, and prunes the last layer (full attention) to the answer rows as
 * decide does (forward.rs:1133-1187); the request calls further down add
 * chunking, the prefix snapshot and the state cache. Weights live in device memory the model owns, named
 * as in decide's decide-weights-v1 index (convert.rs:158-245): "embed" (bf16
 * [vocab, 2560]), "final_norm", "L{l}.in_norm", "L{l}.w_in", "L{l}.w_out",
 * "L{l}.post_norm", "L{l}.w_gu", "L{l}.w_down", and per layer kind
 * "L{l}.conv_w", "L{l}.a_log", "L{l}.dt_bias", "L{l}.gnorm" (Gated-DeltaNet)
 * or "L{l}.q_norm", "L{l}.k_norm" (attention, layers with (l + 1) % 4 == 0).
 * ====================================================================== */
typedef struct dh_model dh_model;

typedef struct dh_model_config {
  uint32_t layers;       /* decoder layers (decide: 32: 36) */
  uint32_t vocab;        /* embedding rows (decide: 248,320; BASELINE: 151,936) */
  uint32_t max_tokens;   /* rows per forward, at most 8192 (decide's MAX_TOKENS) */
  uint32_t max_answers;  /* answer rows per forward (decide: MAX_ANSWERS 16) */
  uint32_t max_cand;     /* candidates per answer row (decide: MAX_CANDIDATES 62) */
} dh_model_config;

/* dh_model_forward flags */
#define DH_FORWARD_NO_PRUNE 1u /* run the last layer over every row (decide: set_prune(false)) */

/* Allocates the weights and activation buffers on the context's device. */
int dh_model_create(dh_ctx* ctx, const dh_model_config* cfg, dh_model** out);
void dh_model_destroy(dh_model* model);
/* Device address, element count and dtype (0 fp16, 1 bf16, 2 fp32) of a
 * weight by its decide-weights-v1 name. */
int dh_model_tensor(const dh_model* model, const char* name, void** ptr, uint64_t* elems, uint32_t* dtype);
/* Name of the model's i-th tensor (i from 0 until it returns NULL). */
const char* dh_model_tensor_name(const dh_model* model, uint32_t i);
/* Fills every tensor of the model from a decide-weights-v1 directory
 * (decide: Weights::open, weights.rs:105-183): `decide-index.json` plus the
 * blobs it lists, tensors at 16 KiB-aligned offsets. Checks decide's format
 * tag, dtypes, alignment and bounds, and that each tensor has the dtype and
 * element count the model holds. Blobs are memory-mapped and each tensor is
 * copied once into device memory. Synchronous. */
int dh_model_load(dh_model* model, const char* dir);
/* Random-initialises every weight on `stream` with dh_fill_normal (BASELINE
 * config 5: fp16 GEMM weights, bf16 embedding, fp32 small parameters). */
int dh_model_init_random(dh_model* model, void* stream, uint64_t seed);
/* One forward over t prompt tokens (device ids [t], each < vocab: the caller
 * validates ids, as decide's engine does, forward.rs:1494-1537), enqueued on
 * `stream`. For the n_ans answer rows (device u32 row indices, which are
 * also their positions) writes logits[r * max_cand + c] for the candidate ids
 * cand[r * max_cand + c], c < ncand[r] (decide: encode_final_head,
 * forward.rs:1296-1306). Does not synchronise. */
int dh_model_forward(dh_model* model, void* stream, const uint32_t* ids, uint32_t t, const uint32_t* ans_rows,
                     uint32_t n_ans, const uint32_t* cand, const uint32_t* ncand, float* logits, uint32_t flags);

/* Whole-forward HIP graph (decide has no counterpart: Metal encodes a command
 * buffer per run; this records the forward's launches once so a serving loop
 * replays them with one launch). Runs one eager forward on `stream` (so every
 * workspace is sized before capture), then captures a second into a graph.
 * Replays read and write the same buffers (ids, answer rows, candidates,
 * logits) with the same T and answer count; their contents may change between
 * replays. `stream` must be a created stream, not the legacy default stream. */
typedef struct dh_graph dh_graph;
int dh_model_capture(dh_model* model, void* stream, const uint32_t* ids, uint32_t t, const uint32_t* ans_rows,
                     uint32_t n_ans, const uint32_t* cand, const uint32_t* ncand, float* logits, uint32_t flags,
                     dh_graph** out);
int dh_graph_launch(dh_graph* graph, void* stream);
void dh_graph_destroy(dh_graph* graph);

/* ======================================================================
 * Requests (decide: Forward::logits, build_snapshot and the state cache,
 * crates/decide-engine/src/forward.rs:641-1116). Host ids and answers; each
 * call enqueues its work on `stream` and waits for it, as decide's do.
 *   - Chunks: a span runs in chunks of at most dh_model_chunk() rows, every
 *     layer of one chunk and then the next, state carried between chunks
 *     (forward.rs:887-915). Default: max_tokens (the whole span in one
 *     chunk); decide's default is CHUNK = 512 (config.rs:36).
 *   - Prefix snapshot: dh_model_build_snapshot runs the constant prompt
 *     prefix from zero state and keeps the state after it.
 *   - Tail truncation: rows after the last answer row never run.
 *   - State cache: an LRU of up to 4 states (default 2) at the end of
 *     prompts' state sections, which end with the state marker (default
 *     decide's STATE_MARKER, forward.rs:68). A request about a new state
 *     captures it on the way; one whose ids start with a cached state's ids
 *     runs from the end of that state.
 * ====================================================================== */
typedef struct dh_answer {
  uint32_t row;          /* absolute logit row (< the request's token count) */
  uint32_t ncand;        /* 1 .. max_cand */
  const uint32_t* cand;  /* host candidate token ids [ncand], each < vocab */
} dh_answer;

/* dh_model_logits flags */
#define DH_LOGITS_FULL 1u /* the full route whatever the ids (decide: logits_full, forward.rs:809-815) */

/* dh_model_last_route routes (decide: Route, forward.rs:196-207) */
#define DH_ROUTE_SNAPSHOT 0
#define DH_ROUTE_FULL 1
#define DH_ROUTE_STATE_CACHE 2

/* Logits of each answer's candidates into logits[i * max_cand + c] for the
 * caller's answer i and c < answers[i].ncand (other entries untouched).
 * Checks decide's contract with its messages (check_ids, sorted_answers,
 * forward.rs:1494-1541) and refuses non-finite logits (forward.rs:876-882).
 * Route: from the snapshot when the ids start with the prefix and every
 * answer row lies after it, from a cached state when the ids also start
 * with that state's ids (the longest such), else the full route
 * (decide: logits, forward.rs:696-735; run_answers, 817-885). */
int dh_model_logits(dh_model* model, void* stream, const uint32_t* ids, uint32_t len, const dh_answer* answers,
                    uint32_t n_answers, float* logits, uint32_t flags);
/* Runs `prefix_ids` (len < max_tokens) from position 0 with zero state and
 * keeps the state after it; replaces any earlier snapshot and empties the
 * state cache (decide: build_snapshot, forward.rs:641-675). */
int dh_model_build_snapshot(dh_model* model, void* stream, const uint32_t* prefix_ids, uint32_t len);
/* The snapshot's prefix length (*has_snapshot 0 before the first build;
 * decide: prefix_len, forward.rs:677-680). */
int dh_model_prefix_len(const dh_model* model, uint32_t* len, int* has_snapshot);
/* How the last dh_model_logits computed its request (DH_ROUTE_*, or -1
 * before the first) and the first position it computed (decide: last_route,
 * last_start, forward.rs:682-694). */
int dh_model_last_route(const dh_model* model, int32_t* route, int64_t* start);
/* Rows per chunk, 1 .. max_tokens (decide: set_chunk, forward.rs:560-566). */
int dh_model_set_chunk(dh_model* model, uint32_t rows);
uint32_t dh_model_chunk(const dh_model* model);
/* Prune the last layer to the answer rows (default on; decide: set_pruning, forward.rs:573-578). */
void dh_model_set_pruning(dh_model* model, int on);
int dh_model_pruning(const dh_model* model);
/* State cache capacity, 0 .. 4 (0 turns it off); shrinking evicts the least
 * recently used entries (decide: set_state_cache, forward.rs:732-743). */
int dh_model_set_state_cache(dh_model* model, uint32_t entries);
uint32_t dh_model_state_cache_capacity(const dh_model* model);
/* Forget every cached state, keeping the buffers for the next captures (forward.rs:745-750). */
void dh_model_forget_states(dh_model* model);
/* The token length of each cached state, most recently used first, into
 * lens[0 .. max); returns the number of entries (decide: cached_states, forward.rs:757-762). */
uint32_t dh_model_cached_states(const dh_model* model, uint32_t* lens, uint32_t max);
/* The ids that end a prompt's state; empties the cache (decide: set_state_marker, forward.rs:764-771). */
int dh_model_set_state_marker(dh_model* model, const uint32_t* marker, uint32_t len);
/* Where a prompt's state ends: one past the first `marker` in
 * ids[prefix .. min(limit, len)]; *found 0 if there is none (decide:
 * state_boundary, forward.rs:1503-1515). Host-only. */
int dh_state_boundary(const uint32_t* ids, uint32_t len, uint32_t prefix, const uint32_t* marker, uint32_t marker_len,
                      uint32_t limit, uint32_t* boundary, int* found);

/* ======================================================================
 * The 8-bit paged key/value cache: rotary positions, the append that codes
 * key and value rows into pages, the attention that reads them, and the
 * copying, sharing and moving of pages. decide has no counterpart: its caches
 * are fp16 and contiguous, one per request (kernels/rope.rs:39-54,
 * kernels/attn.rs:80-125), and a state is copied whole
 * (forward.rs:641-675). Here many sequences share the pages of the
 * prefix that they have in common, and a token takes half the bytes.
 *
 * A cache is a pool of pages, [layers][pages] records of dh_kv8_page_bytes()
 * each. A page holds DH_KV8_PAGE tokens of every kv head:
 *   K codes  [kv_heads][DH_KV8_PAGE][head_dim]   (one byte each)
 *   V codes  [kv_heads][head_dim][DH_KV8_PAGE]   (tokens innermost)
 *   scales   [kv_heads][2][4] float              (K's, V's; one for DH_KV8_BLOCK tokens)
 * and padding to a multiple of 128 bytes. A value is code x scale:
 *   DH_KV8_E4M3  the byte is an OCP e4m3 number (never its NaN), the scale the smallest power of two
 *                that brings the block's largest magnitude to at most 448;
 *   DH_KV8_INT8  the byte b stands for b - 128 (-127..127), the scale is the largest magnitude x 1/127 (in fp32).
 * Scales are at least 2^-100. A block (16 tokens of one head) that was given a
 * value that is not finite has a NaN scale: all of its values are NaN.
 * ====================================================================== */
#define DH_KV8_PAGE 64u
#define DH_KV8_BLOCK 16u
#define DH_KV8_E4M3 0u
#define DH_KV8_INT8 1u

typedef struct dh_kv8_cache {
  void* pool;         /* device memory, layers * pages * dh_kv8_page_bytes() bytes, 128-byte aligned */
  uint32_t pages;     /* pages of one layer */
  uint32_t layers;
  uint32_t kv_heads;  /* 1 .. 1024 */
  uint32_t head_dim;  /* 64, 128 or 256 */
  uint32_t format;    /* DH_KV8_E4M3 or DH_KV8_INT8 */
} dh_kv8_cache;

/* Bytes of one page of one layer (0 for a head_dim or kv_heads out of range). */
uint64_t dh_kv8_page_bytes(uint32_t kv_heads, uint32_t head_dim);

/* The rows of one call and the sequences they belong to; device arrays.
 * Rows row0[s] .. row0[s + 1] - 1 are sequence s's; row0 does not decrease,
 * and entries past `rows` count as `rows`. Rows before row0[0] or from
 * row0[seqs] on belong to none: nothing reads them or writes their outputs.
 * Token t of sequence s lies in page table[s * ld_table + t / DH_KV8_PAGE];
 * the same page may stand in several tables. */
#define DH_KV8_NO_POSITION 0xffffffffu
typedef struct dh_kv8_batch {
  const uint32_t* table; /* [seqs][ld_table] page ids */
  const uint32_t* row0;  /* [seqs + 1] */
  const uint32_t* qpos;  /* [rows] each row's position in its sequence, or DH_KV8_NO_POSITION */
  uint32_t ld_table;     /* entries of a table row */
  uint32_t seqs;
  uint32_t rows;         /* rows that the arrays and matrices hold (the launch is sized by it) */
} dh_kv8_batch;

/* A rotary embedding. Element pairs (i, i + rot / 2) (DH_ROPE_HALF) or
 * (2i, 2i + 1) (DH_ROPE_INTERLEAVED), i < rot / 2, turn by the angle
 * position * inv_freq[i], formed and reduced in 64 bits, with cos and sin
 * multiplied by `amp`; elements from rot on pass through. With norm_w, each
 * head is first RMS-normed over its head_dim elements and multiplied by w
 * (add_one 0) or 1 + w. */
#define DH_ROPE_HALF 0u
#define DH_ROPE_INTERLEAVED 1u
typedef struct dh_rope_spec {
  const float* inv_freq; /* device [rot / 2] */
  const float* norm_w;   /* device [head_dim], or NULL: no norm */
  uint32_t head_dim;     /* a multiple of 4, 4 .. 256 */
  uint32_t rot;          /* even, 2 .. head_dim */
  uint32_t layout;       /* DH_ROPE_* */
  uint32_t add_one;
  float eps;             /* > 0 with norm_w */
  float amp;             /* finite */
} dh_rope_spec;

/* y[r, h] = rope(norm(x[r, h]), pos[r]) for `heads` heads of spec->head_dim
 * elements, head h at column h * head_dim of rows of stride ldx and ldy
 * (elements). x_dtype and y_dtype: 0 fp16, 1 bf16, 2 fp32; arithmetic fp32.
 * y may be x where dtypes and strides agree. Contract: strides cover the heads
 * and are multiples of 4; x and y aligned to 4 of their elements; norm_w to
 * 16 bytes. pos: device u32 [rows], every value a position.
 * (dh_q_norm_rope is this with decide's layout: 16 heads of 256, 64 of them
 * rotated as halves, fp32 in, fp16 out, and its angle an fp32 product.) */
int dh_rope(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, uint32_t x_dtype, void* y, uint32_t ldy,
            uint32_t y_dtype, const uint32_t* pos, uint32_t rows, uint32_t heads, const dh_rope_spec* spec);

/* inv_freq[i] (host, [rot / 2]) and the amplitude for positions stretched by
 * `factor` (>= 1), from f_i = base^(-2i / rot):
 *   DH_ROPE_PLAIN   f_i (factor is not used);
 *   DH_ROPE_LINEAR  f_i / factor: positions squeezed into the trained range;
 *   DH_ROPE_BASE    base * factor^(rot / (rot - 2)) in place of base (rot > 2): the slowest pair squeezed by factor, the
 *                   fastest not at all;
 *   DH_ROPE_PARTS   f_i where pair i turns at least `high` times within trained_len positions, f_i / factor
 *                   where it turns at most `low` times, linear in the number of turns between; amplitude
 *                   0.1 ln(factor) + 1 (1 for the other kinds).
 * low, high and trained_len are read by DH_ROPE_PARTS only. Computed in 64 bits. */
#define DH_ROPE_PLAIN 0u
#define DH_ROPE_LINEAR 1u
#define DH_ROPE_BASE 2u
#define DH_ROPE_PARTS 3u
int dh_rope_freqs(uint32_t rot, double base, uint32_t kind, double factor, double low, double high,
                  uint32_t trained_len, float* inv_freq, float* amp);

/* Stores K and V rows at their sequences' ends: row r0 + i of sequence s, whose
 * first row in the batch is r0, becomes token qpos[r0] + i (the rows of a
 * sequence are consecutive tokens; later entries of qpos are not read). k and
 * v: kv_heads heads of head_dim elements, dtype as dh_rope's, row strides ldk
 * and ldv. With `rope` (head_dim as the cache's), each key is normed and
 * turned at its token's position, in 64 bits, and rounded to fp32 before it is
 * coded; without, keys are coded as they are. Values always are.
 * The call ends the sequence after its last row: a block that it starts within
 * keeps its earlier tokens (coded again where its scale grows; the scale never
 * shrinks while tokens stay), and whatever the block of the last row held
 * behind that row is cleared. A page that another sequence's table also holds
 * changes for that one too: copy it first (dh_kv8_copy_pages).
 * A token whose page id is not below cache->pages, or whose table entry would
 * lie past ld_table, is not stored; nor is a sequence whose first row has no
 * position. Contract: as dh_rope for k and v. */
int dh_kv8_append(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t layer, const dh_kv8_batch* batch,
                  const void* k, uint32_t ldk, const void* v, uint32_t ldv, uint32_t dtype, const dh_rope_spec* rope);

/* y[r, h] = softmax_t(scale * q[r, h] . K[t, g]) . V[t, g] (x sigmoid(gate[r, h])),
 * over tokens t = 0 ..= qpos[r] of row r's sequence, kv head g = h / (heads /
 * kv_heads); a row without a position sees no token and its y is zero,
 * whatever its q and gate hold. q fp16 [rows, heads * head_dim] row stride ldq,
 * y fp16 row stride ldy, gate (may be NULL) fp32 row stride ldg; scores and softmax fp32; the products of a weight
 * and its block's V scale, relative to the largest that the row meets, are
 * rounded to fp16 as the operand of their product with V's codes. max_tokens:
 * how many tokens the longest row sees, for the launch's division of long
 * sequences; a row may see more (slower) or all fewer. Rows in any order of
 * positions.
 * A row that sees a token whose page id is not below cache->pages, or whose
 * table entry would lie past ld_table, is NaN; so is one that sees a token of a
 * block with a NaN scale. Bytes behind a sequence's last seen token may hold
 * anything. Contract: heads % kv_heads == 0, at most 1,024 heads a kv head; scale finite;
 * ldq % 8 == 0, ldy % 4 == 0, ldg % 4 == 0; q and gate 16-byte, y 8-byte
 * aligned. Long sequences are divided across workgroups and merged through the
 * context's forward-kernel workspace (dh_kv8_attention_ws; an eager call of
 * the same sizes also grows it). The kernel and the cuts depend on the call's
 * sizes, the cuts also on how many pages its rows see, found on the device. For
 * given sizes a row's bits depend on its own query, gate, position and pages
 * and, where the call's sequences are cut, on the positions of the other rows
 * (rounding only). The same call gives the same bits. */
int dh_kv8_attention(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t layer, const dh_kv8_batch* batch,
                     const uint16_t* q, uint32_t ldq, uint32_t heads, float scale, const float* gate, uint32_t ldg,
                     uint16_t* y, uint32_t ldy, uint32_t max_tokens);
/* Grows `stream`'s forward-kernel workspace to what dh_kv8_attention needs for
 * these sizes and any smaller ones (before a capture on that stream, for
 * instance). */
int dh_kv8_attention_ws(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, uint32_t rows, uint32_t seqs,
                        uint32_t heads, uint32_t max_tokens);

/* Copies page src[i] to page dst[i] in every layer, i < n (device arrays):
 * what dh_pages_resize and dh_pages_compact ask for. A pair with an id not
 * below cache->pages is left out. No dst may be another pair's src or dst.
 * n <= cache->pages, pairs that are left out among them. */
int dh_kv8_copy_pages(dh_ctx* ctx, void* stream, const dh_kv8_cache* cache, const uint32_t* src, const uint32_t* dst,
                      uint32_t n);

/* Which pages which sequence holds: reference counts and tables in host memory,
 * no device involved. Sequences are numbered 0 .. max_seqs - 1 and start empty;
 * a new page is always the free one of the lowest id, so equal calls give
 * equal tables. One dh_pages serves one thread at a time. */
typedef struct dh_pages dh_pages;
int dh_pages_create(uint32_t pages, uint32_t max_seqs, dh_pages** out);
void dh_pages_destroy(dh_pages* p);
/* Makes sequence s hold `tokens` tokens: frees the pages past them or takes new
 * ones. Where tokens are added behind a page that is partly full and shared,
 * the sequence gets a page of its own in its place: copy_src / copy_dst name the
 * copy to make (dh_kv8_copy_pages) before the tokens are appended, and *copies
 * is 1 (else 0). If the free pages do not suffice nothing changes and the call
 * returns DH_ENOMEM. */
int dh_pages_resize(dh_pages* p, uint32_t seq, uint64_t tokens, uint32_t* copy_src, uint32_t* copy_dst,
                    uint32_t* copies);
/* Makes dst (empty before) share the pages of src's first `tokens` tokens. */
int dh_pages_fork(dh_pages* p, uint32_t src, uint32_t dst, uint64_t tokens);
/* Moves held pages to the lowest ids: src[i] -> dst[i], i < *moves (arrays of
 * max entries; as many pages as are held suffice). The tables name the new
 * pages at once; copy with dh_kv8_copy_pages before the next use. With more
 * than max moves to make nothing changes and the call returns DH_EINVAL. */
int dh_pages_compact(dh_pages* p, uint32_t* src, uint32_t* dst, uint32_t max, uint32_t* moves);
/* A sequence's tokens and pages, and the first min(max, *count) of its page ids. */
int dh_pages_table(const dh_pages* p, uint32_t seq, uint64_t* tokens, uint32_t* ids, uint32_t max, uint32_t* count);
/* Free pages, and the sequences that hold page `page`. */
uint32_t dh_pages_free(const dh_pages* p);
uint32_t dh_pages_refs(const dh_pages* p, uint32_t page);

/* ======================================================================
 * 8-bit floating point: rows and weights as e4m3 codes with a power-of-two
 * scale for each block of 128, and the matrix product of such codes. decide
 * has no counterpart: its GEMM path is fp16 (kernels/gemm.rs:126-176). Codes
 * take half of fp16's bytes and their products run at twice its rate.
 *
 * A matrix of K columns:
 *   codes   [rows][ld] bytes, OCP e4m3 numbers; columns from K to the next
 *           multiple of DH_FP8_BLOCK are zero
 *   scales  [ceil(K / 512)][lds][4] bytes: byte b of entry [j][r] is e + 127
 *           for the scale 2^e of columns 128 (4 j + b) .. + 127 of row r
 *           (activations) or of rows 128 r .. + 127 (weights); 1 .. 254. Bytes
 *           of blocks that lie wholly behind K count for nothing.
 * The value of a code is code x scale. The functions that code values choose
 * the smallest e >= -100 that brings the block's largest finite magnitude to
 * at most 448; each code is then one rounding (to nearest, ties to even) of
 * its value. A value that is not finite becomes the code 0x7f, NaN.
 * ====================================================================== */
#define DH_FP8_BLOCK 128u

typedef struct dh_fp8_matrix {
  void* codes;   /* device memory, 16-byte aligned */
  void* scales;  /* device memory, 16-byte aligned */
  uint32_t ld;   /* a multiple of 16 covering K in whole blocks, at most 2^23 */
  uint32_t lds;  /* a multiple of 4 covering the rows (activations) or blocks of rows (weights), at most 2^26 */
} dh_fp8_matrix;

/* Codes `rows` rows of k columns, x[r * ldx + c] with dtype 0 fp16, 1 bf16,
 * 2 fp32, with a scale for each row and block of columns. With norm_w (fp32
 * [k]) each row is first normed as dh_rmsnorm_rows does, x * (mean(x^2) +
 * eps)^-1/2 * (add_one ? 1 + w : w), in 64 bits and rounded to fp32. Writes the
 * codes of columns 0 .. k in whole blocks (zeros behind k) and the scale
 * entries of the rows (127 for blocks behind k). Contract: ldx covers k and is
 * a multiple of 8; x and norm_w 16-byte aligned; eps > 0 with norm_w. */
int dh_fp8_quant_rows(dh_ctx* ctx, void* stream, const void* x, uint32_t ldx, uint32_t dtype, const float* norm_w,
                      uint32_t add_one, float eps, const dh_fp8_matrix* out, uint32_t rows, uint32_t k);
/* The same for a weight of n rows, with a scale for each 128 rows x 128 columns. */
int dh_fp8_quant_blocks(dh_ctx* ctx, void* stream, const void* w, uint32_t ldw, uint32_t dtype, const dh_fp8_matrix* out,
                        uint32_t n, uint32_t k);

/* y = epi(X . W^T) of the values that codes and scales stand for: x of m rows
 * with a scale for each row, w of n rows with a scale for each 128 rows, k
 * columns each; epilogues and y as dh_gemm_nt's. Products are exact and sums
 * fp32; with fp16 outputs (SwiGLU among them) the products of each eight
 * neighbouring columns are first added by the matrix instruction, which cuts
 * what lies more than 13 bits below the largest of them (2^-13 of the largest
 * product a term at most; beside an fp16 rounding a fourteenth of its error on
 * normal data, a fifth where columns differ by factors of e).
 * With fp32 outputs values are held as bfloat16 first: exactly where the byte
 * of their scale is 3 .. 246, whatever the code; beyond, what is past
 * bfloat16's largest number counts as infinite and what is no multiple of its
 * smallest, 2^-133, is rounded to one. (The functions above bring only values
 * of 1.9375 x 2^127 and more there, whose code times scale is 2^128.)
 * Contract: any m, n and k (n % 32 == 0 for SwiGLU); ldy % 4 == 0; y 16-byte
 * (fp32 outputs) or 8-byte (fp16 outputs) aligned; a code of NaN makes its row
 * (of x) or column (of w's row) NaN. Where there are few tiles K is divided and
 * the parts are summed through `stream`'s split-K workspace (dh_gemm_fp8_ws, or
 * an eager call of the same size, grows it). A row's bits depend on the call's
 * m, n and k and on its own codes and scales alone. */
int dh_gemm_fp8(dh_ctx* ctx, void* stream, const dh_fp8_matrix* x, const dh_fp8_matrix* w, void* y, uint32_t ldy,
                uint32_t m, uint32_t n, uint32_t k, uint32_t epi);
/* Grows `stream`'s split-K workspace to what dh_gemm_fp8 needs for n, k and any
 * m up to max_m (at most DH_PLAN_MAX_ROWS). */
int dh_gemm_fp8_ws(dh_ctx* ctx, void* stream, uint32_t max_m, uint32_t n, uint32_t k);

/* ======================================================================
 * Causal attention over packed sequences: the rows of several requests one
 * behind another, each attending to its own sequence's keys. decide's attention
 * takes one request's 16 heads of 256 dims (dh_attention); here heads, sizes
 * and types are arguments, keys and values are read from the projections' rows
 * (or any other), and a sequence may bring one row or thousands.
 * ====================================================================== */
/* The sequences of a call; device arrays. Sequence s has the rows q0[s] ..
 * q0[s + 1] - 1 of q, gate and y and the rows k0[s] .. k0[s + 1] - 1 of k and v.
 * Neither decreases, and entries past q_rows (k_rows) count as q_rows (k_rows).
 * Rows of q that belong to no sequence are not read, and their y is left as it
 * was. */
typedef struct dh_packed_batch {
  const uint32_t* q0; /* [seqs + 1] */
  const uint32_t* k0; /* [seqs + 1]; may be q0: whole prompts */
  uint32_t seqs;
  uint32_t q_rows;    /* rows that q, gate and y hold (the launch is sized by it) */
  uint32_t k_rows;    /* rows that k and v hold */
  uint32_t max_k;     /* keys of the longest sequence, for the launch's division of long ones; a hint */
} dh_packed_batch;

/* y[r, h] = softmax_t(scale * q[r, h] . k[t, g]) . v[t, g] (x sigmoid(gate[r, h])),
 * kv head g = h / (heads / kv_heads). Row i (from 0) of a sequence of nq rows
 * and nk keys sees its keys 0 .. nk - nq + i: a whole prompt where nk = nq, the
 * last rows of a longer one, down to a single token, where nq < nk; where
 * nq > nk the first nq - nk rows see nothing and are zero, whatever their q and
 * gate hold. dtype, of q, k, v and y: 0 fp16, 1 bf16; gate (may be NULL) fp32.
 * Head h of a row at column h * head_dim; strides ldq, ldk, ldv, ldg, ldy in
 * elements. Scores and softmax fp32; a weight relative to its row's largest is
 * rounded to dtype as the operand of its product with v. A row does not depend
 * on keys and values that it does not see, whatever they hold; what it sees is
 * followed through softmax, infinities and NaN among it. Two limits: an infinite
 * value of a key whose weight is too small for dtype makes its column infinite
 * or NaN (zero times infinity), as the call's layout has it; and values are
 * summed in fp32 with weights of up to 2^8 before they are divided by the
 * weights' sum, so that bfloat16 values near 2^127 can give infinity.
 * Contract: head_dim 64, 128 or 256; heads % kv_heads == 0, at most 1,024 heads
 * a kv head; |scale| at most 2^127; ldq, ldk, ldv % 8 == 0, ldy, ldg % 4 == 0, each
 * covering its heads; q, k, v and gate 16-byte, y 8-byte aligned. Few rows over
 * many keys are divided across workgroups and merged through the context's
 * forward-kernel workspace (dh_attention_packed_ws; an eager call of the same
 * sizes also grows it). The same call gives the same bits. */
int dh_attention_packed(dh_ctx* ctx, void* stream, const dh_packed_batch* batch, const void* q, uint32_t ldq,
                        const void* k, uint32_t ldk, const void* v, uint32_t ldv, uint32_t dtype, uint32_t heads,
                        uint32_t kv_heads, uint32_t head_dim, float scale, const float* gate, uint32_t ldg, void* y,
                        uint32_t ldy);
/* Grows `stream`'s forward-kernel workspace to what dh_attention_packed needs
 * for calls of up to q_rows rows in up to `seqs` sequences (before a capture on
 * that stream, for instance). */
int dh_attention_packed_ws(dh_ctx* ctx, void* stream, uint32_t q_rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads,
                           uint32_t head_dim);

#ifdef __cplusplus
}
#endif

#endif /* DECIDE_HIP_H */
