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
  float scale;
};

hipError_t launch_packed_wide(const PackArgs& a, uint32_t head_dim, bool bf16, hipStream_t s);

}  // namespace dh
