// The 8-bit paged cache's launch arguments and launchers (kv8.hip, kv8_attention.hip), shared by the kernels and the
// C ABI (api_kv8.cpp). Host-visible, no device code here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dh {

constexpr uint32_t kKvPage = 64;   // tokens of a page
constexpr uint32_t kKvBlock = 16;  // tokens that share a scale

// A rotary embedding and the norm before it, as dh_rope_spec has them.
struct RopeArgs {
  const float* inv_freq;
  const float* norm_w;  // or null
  uint32_t head_dim, rot, interleaved, add_one;
  float eps, amp;
};

// One layer of a cache and the batch of a call.
struct KvArgs {
  uint8_t* pool;  // the layer's first page
  uint64_t page_bytes;
  uint32_t pages, kv_heads;
  const uint32_t* table;
  const uint32_t* row0;
  const uint32_t* qpos;
  uint32_t ld_table, seqs, rows;
};

// elements of x and y: 0 fp16, 1 bf16, 2 fp32
hipError_t launch_rope(const void* x, uint32_t ldx, uint32_t x_dtype, void* y, uint32_t ldy, uint32_t y_dtype,
                       const uint32_t* pos, uint32_t rows, uint32_t heads, const RopeArgs& rope, hipStream_t s);
// rope.inv_freq null: keys are coded as they are; cus: compute units of the device
hipError_t launch_kv8_append(const KvArgs& a, uint32_t head_dim, bool int8, const void* k, uint32_t ldk, const void* v,
                             uint32_t ldv, uint32_t dtype, const RopeArgs& rope, uint32_t cus, hipStream_t s);
hipError_t launch_kv8_copy_pages(uint8_t* pool, uint64_t page_bytes, uint32_t pages, uint32_t layers,
                                 const uint32_t* src, const uint32_t* dst, uint32_t n, hipStream_t s);

constexpr uint32_t kKvTile = 16;         // (row, head) pairs of a tile
constexpr uint32_t kKvMaxSlots = 2048;   // tiles that the runs are dealt over (their page counts lie in LDS)
constexpr uint32_t kKvWideTile = 128;    // the same for many rows
constexpr uint32_t kKvWideSlots = 1024;

// How an attention call is divided. runs > 0: the tiles' pages, one after another, in so many equal runs per kv head, a
// workgroup each, and their states in the workspace: [kv head][run][2] x (O [16][D], (largest score, sum) [16]), then
// the pages before each tile. runs = 0: a workgroup per tile and kv head, no workspace.
struct KvAttnPlan {
  uint32_t slots = 0;  // tiles of every kv head, an upper bound
  uint32_t runs = 0;
  uint32_t min_run = 1;  // pages of a run at least
  bool wide = false;
  uint64_t ws_bytes = 0;
};
KvAttnPlan kv8_attention_plan(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                              uint32_t ld_table, uint32_t max_tokens, uint32_t cus);
uint64_t kv8_attention_ws_bytes(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_tokens,
                                uint32_t cus);
hipError_t launch_kv8_attention(const KvArgs& a, uint32_t head_dim, bool int8, const _Float16* q, uint32_t ldq,
                                uint32_t heads, float scale, const float* gate, uint32_t ldg, _Float16* y,
                                uint32_t ldy, float* ws, const KvAttnPlan& plan, uint32_t cus, hipStream_t s);

}  // namespace dh
