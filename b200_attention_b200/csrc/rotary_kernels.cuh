// Internal interface between the C-ABI layer and the norm-and-rotation kernel.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace b200attn {

constexpr int kRotaryMaxAxes = 4;

struct RotaryOperand {
  const __nv_bfloat16* in;
  __nv_bfloat16* out;
  int64_t in_stride_b, in_stride_h, in_stride_t;     // in elements
  int64_t out_stride_b, out_stride_h, out_stride_t;
  const void* weight;  // [128], or null: no norm
};

struct RotaryParams {
  RotaryOperand q, k;
  int32_t batch, tokens, heads_q, heads_k;
  const void* positions;
  int64_t pos_stride_axis, pos_stride_batch, pos_stride_token;
  int32_t pos_type;     // 0 int32, 1 int64, 2 fp32
  int32_t weight_fp32;  // 0: weights are bf16
  const float* inv_freq;
  int32_t pairs;                              // rotated pairs, the first ones of a head
  int32_t section_end[kRotaryMaxAxes];        // pair j belongs to the first axis a with j < section_end[a]
  float eps;
  int32_t chunks, chunk_heads;                // set by the launcher: warps per token, heads of each
};

cudaError_t launch_qk_norm_rope(RotaryParams p, bool interleaved, int sm_count, cudaStream_t stream);

}  // namespace b200attn
