// Internal interface between the C-ABI layer and the planned-attention and rotation kernels.
#pragma once

#include "attn_kernels.cuh"
#include "plan.h"

namespace b200attn {

// q, q_small: (head_dim, head of the group, K/V head, token), boxes of tile_tokens and small_tokens tokens; the others:
// (head_dim, row, K/V head, 1)
struct PlanMaps {
  CUtensorMap q, q_small, k, v, k_prefix, v_prefix;
};

struct PlanParams {
  const int32_t* table;
  __nv_bfloat16* o;
  float* lse;  // [heads][lse_stride_h], or null
  int64_t o_stride_t, o_stride_h, lse_stride_h;
  float* part_o;    // [slot rows][128] fp32, normalised
  float* part_lse;  // [slot rows], natural log, -inf where no key was visible
  int32_t o_aligned;    // every row of o begins on a multiple of 32 bytes
  int32_t group;        // query heads per K/V head
  int32_t tile_tokens;  // floor(128 / group)
  int32_t tile_rows;    // tile_tokens * group
  int32_t small_tokens; // floor(32 / group): a piece of one Q tile with at most these is a small one; may be 0
  float scale_log2;
  int32_t* status;
  uint32_t wait_limit_ms;
};

cudaError_t prepare_plan_kernels();
cudaError_t launch_plan(const PlanMaps& maps, const PlanParams& p, int grid, bool wide, cudaStream_t stream);
cudaError_t launch_plan_join(const PlanParams& p, int grid, cudaStream_t stream);

}  // namespace b200attn
