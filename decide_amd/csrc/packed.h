// Launch arguments and launchers of attention over packed sequences (packed_wide.hip), shared by the kernels and the C ABI
// (api_packed.cpp). Host-visible, no device code here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dh {

struct PackArgs {
  const uint16_t *q, *k, *v;  // fp16 or bf16
  const float* gate;          // or null
  uint16_t* y;
  float* ws;  // the runs' states
  const uint32_t *q0, *k0;
  uint32_t ldq, ldk, ldv, ldg, ldy;
  uint32_t seqs, q_rows, k_rows;
  uint32_t kv_heads, group;  // query heads of a kv head
  uint32_t group_inv;        // 2^21 / group, rounded up
  uint32_t slots;            // tiles are numbered below it
  uint32_t runs;             // of each kv head; 0: a workgroup a tile
  uint32_t min_run;          // steps (of 128 keys) of a run at least
  float scale;
};

constexpr uint32_t kPackTile = 32;       // (row, head) pairs of a tile of the kernel for few rows
constexpr uint32_t kPackWideTile = 128;  // the same for many
constexpr uint32_t kPackSlots = 2048;    // tiles that runs are dealt over (their steps lie in LDS)
// Steps of 32 keys that a wave of the kernel for few rows holds in LDS: 32 KB at most.
constexpr int packed_ring(int head_dim) { return head_dim == 64 ? 3 : 256 / head_dim; }

// How a call is computed: wide tiles, or narrow ones, a workgroup each or dealt in runs with their states in the workspace.
struct PackPlan {
  bool wide = false;
  uint32_t slots = 0, runs = 0, min_run = 1;
  uint64_t ws_bytes = 0;
};
PackPlan packed_plan(uint32_t q_rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_k,
                     uint32_t cus);
uint64_t packed_run_bytes(uint32_t runs, uint32_t slots, uint32_t kv_heads, uint32_t head_dim);
hipError_t launch_packed_narrow(const PackArgs& a, uint32_t head_dim, bool bf16, hipStream_t s);
hipError_t launch_packed_wide(const PackArgs& a, uint32_t head_dim, bool bf16, hipStream_t s);

}  // namespace dh
