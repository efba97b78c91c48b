// Norm of queries and keys for each head, and their rotation by position, in one pass (sm_100a).
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (128 values of a head; only where a weight is given)
//   pair j of y:  (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position[axis(j)] * inv_freq[j]
//   pairs are (j, j + 64), or (2j, 2j + 1) when interleaved; pairs behind the last section stay as they are
//
// Bound by memory: 512 bytes per head and token, and not far from being bound by instructions: about 10 operations per
// value. A warp takes one token, a quarter of a warp one head: a lane holds values 8l .. 8l + 7 and 64 + 8l .. 64 + 8l + 7,
// which are eight whole pairs in either pairing, so the only exchange is the sum of squares over eight lanes. The
// angles depend on the token and the pair alone: each lane works out two, through shared memory they reach the lanes
// that need them, and they serve every head that the warp visits. The rotation is linear, so the norm's weight goes
// into the cosines and sines once per token and only the row's scale is left to apply per head; arithmetic is on
// packed pairs of 32-bit values.
// Measured at 16384 tokens, 32 + 8 heads: half a warp per head with every lane working out its own four angles ran
// 47.6 M warp instructions and was bound by them (71 us, 4.7 TB/s); this form takes 59.7 us, 5.6 TB/s, 87 % of what a
// plain copy reaches. Blocks of 4 warps against 8: 63.4 and 65.1 us.
// Statistics and rotation are in 32 bits and rounded to bf16 once. Angles are reduced to a fraction of a turn in
// 64 bits first: at position 10^6 a 32-bit product is already off by 0.03 radians.

#include "launch_overlap.cuh"
#include "ptx_sm100.cuh"
#include "rotary_kernels.cuh"

#include <cuda_bf16.h>

namespace b200attn {

namespace {

using ptx::f2;
using ptx::f2_fma;
using ptx::f2_make;
using ptx::f2_split;
using ptx::f2_splat;
using ptx::pack_bf16x2;

constexpr int kWarps = 4;
constexpr int kPairs = 64;
// Two numbers make a variant: the heads of a quarter warp that are on their way while one is worked on, and the blocks
// per SM that the registers are shared out for. Measured (us):
//                                               2 ahead, 6 blocks   1 ahead, 7 blocks   1 ahead, 6 blocks
//   16384 tokens x 40 heads (10 heads a quarter)      59.7                62.0                64.6
//   65536 tokens x 24 heads (6)                      155.2               147.6               155.7
//   1537 tokens x 24 heads, 2 warps a token (3)        6.8                 6.9                 6.2
//   32 tokens x 40 heads, 10 warps a token (1)         4.0                 3.7                 3.6
// One warp a token, 16384 and 65536 tokens, both pairings, 8 to 64 heads: the second is 3 to 20 % faster at 8, 12, 16, 20
// and 24 heads, the first 1 to 6 % at 26, 28, 30, 32, 36, 40, 48 and 64 (65536 tokens x 32 heads, half-split: level).
// ptxas spills 68, 48 and 8 bytes a thread in the three variants.
constexpr int kFewHeads = 24;  // of a token in one warp

__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}

__device__ __forceinline__ double position_of(const RotaryParams& p, int axis, int64_t b, int64_t t) {
  const int64_t at = axis * p.pos_stride_axis + b * p.pos_stride_batch + t * p.pos_stride_token;
  if (p.pos_type == 0) return double(static_cast<const int32_t*>(p.positions)[at]);
  if (p.pos_type == 1) return double(static_cast<const int64_t*>(p.positions)[at]);
  return double(static_cast<const float*>(p.positions)[at]);
}

// Nothing reads the result again before much else has gone through the L2: marked as such (3 % at 16384 tokens).
__device__ __forceinline__ void store16(char* p, uint4 v) { __stcs(reinterpret_cast<uint4*>(p), v); }

// Two bf16 of a word, in order and exchanged.
__device__ __forceinline__ f2 unpack2(uint32_t w) {
  return f2_make(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ f2 unpack2_swapped(uint32_t w) {
  return f2_make(__uint_as_float(w & 0xffff0000u), __uint_as_float(w << 16));
}
__device__ __forceinline__ uint32_t pack2(f2 v) {
  float lo, hi;
  f2_split(v, lo, hi);
  return pack_bf16x2(lo, hi);
}

__device__ __forceinline__ float weight_of(const void* w, int is_fp32, int i) {
  if (w == nullptr) return 1.0f;
  return is_fp32 ? static_cast<const float*>(w)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// Heads h0, h0 + 4, .. < end of one operand for the calling quarter warp (h0 already counts the quarter).
// `turn` holds (cos, sin) of the token's 64 pairs and is ready once `angles` has been called.
template <bool kInterleaved, int kDepth, class Angles>
__device__ __forceinline__ void rotate_heads(const RotaryOperand& x, const RotaryParams& p, int64_t b, int64_t t, int h0,
                                             int end, int l, const float2* turn, const float* w, Angles angles) {
  const char* src = reinterpret_cast<const char*>(x.in + b * x.in_stride_b + t * x.in_stride_t + h0 * x.in_stride_h + 8 * l);
  char* dst = reinterpret_cast<char*>(x.out + b * x.out_stride_b + t * x.out_stride_t + h0 * x.out_stride_h + 8 * l);
  const int64_t src_step = x.in_stride_h * 8, dst_step = x.out_stride_h * 8;  // four heads, in bytes
  uint4 raw[kDepth][2];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    raw[d][0] = raw[d][1] = make_uint4(0u, 0u, 0u, 0u);
    if (h0 + 4 * d < end) {
      raw[d][0] = *reinterpret_cast<const uint4*>(src + d * src_step);
      raw[d][1] = *reinterpret_cast<const uint4*>(src + d * src_step + 128);
    }
  }
  angles();
  // Packed coefficients. Pairs (j, j + 64): values (e0 e1)(e2 e3).. of the lower half with (f0 f1).. of the upper half,
  //   e' = e (w_e cos) + f (-w_f sin), f' = f (w_f cos) + e (w_e sin).
  // Pairs (2j, 2j + 1): the word (e f) itself, (e' f') = (e f)(w_e cos, w_f cos) + (f e)(-w_f sin, w_e sin).
  f2 cos_lo[4], cos_hi[4], sin_lo[4], sin_hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 w0 = *reinterpret_cast<const float2*>(w + 8 * l + 2 * i);
    const float2 w1 = *reinterpret_cast<const float2*>(w + 64 + 8 * l + 2 * i);
    if (kInterleaved) {
      const float2 c0 = turn[4 * l + i], c1 = turn[32 + 4 * l + i];
      cos_lo[i] = f2_make(w0.x * c0.x, w0.y * c0.x);
      sin_lo[i] = f2_make(-w0.y * c0.y, w0.x * c0.y);
      cos_hi[i] = f2_make(w1.x * c1.x, w1.y * c1.x);
      sin_hi[i] = f2_make(-w1.y * c1.y, w1.x * c1.y);
    } else {
      const float4 cs = *reinterpret_cast<const float4*>(turn + 8 * l + 2 * i);
      cos_lo[i] = f2_make(w0.x * cs.x, w0.y * cs.z);
      cos_hi[i] = f2_make(w1.x * cs.x, w1.y * cs.z);
      sin_lo[i] = f2_make(-w1.x * cs.y, -w1.y * cs.w);
      sin_hi[i] = f2_make(w0.x * cs.y, w0.y * cs.w);
    }
  }
  const bool norm = x.weight != nullptr;
  for (int h = h0; __any_sync(0xffffffffu, h < end); h += 4 * kDepth) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const uint32_t lo[4] = {raw[d][0].x, raw[d][0].y, raw[d][0].z, raw[d][0].w};
      const uint32_t hi[4] = {raw[d][1].x, raw[d][1].y, raw[d][1].z, raw[d][1].w};
      const bool live = h + 4 * d < end;
      if (h + 4 * (d + kDepth) < end) {
        raw[d][0] = *reinterpret_cast<const uint4*>(src + (d + kDepth) * src_step);
        raw[d][1] = *reinterpret_cast<const uint4*>(src + (d + kDepth) * src_step + 128);
      }
      f2 scale = f2_splat(1.0f);
      if (norm) {
        f2 sq0 = f2_splat(0.0f), sq1 = f2_splat(0.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f2 e = unpack2(lo[i]), f = unpack2(hi[i]);
          sq0 = f2_fma(e, e, sq0);
          sq1 = f2_fma(f, f, sq1);
        }
        float a, c;
        f2_split(ptx::f2_add(sq0, sq1), a, c);
        float sq = a + c;
        sq += __shfl_xor_sync(0xffffffffu, sq, 4);
        sq += __shfl_xor_sync(0xffffffffu, sq, 2);
        sq += __shfl_xor_sync(0xffffffffu, sq, 1);
        scale = f2_splat(rsqrtf(fmaf(sq, 1.0f / 128.0f, p.eps)));
      }
      uint32_t out_lo[4], out_hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f2 e = unpack2(lo[i]), f = unpack2(hi[i]);
        f2 a, c;
        if (kInterleaved) {
          a = f2_fma(e, cos_lo[i], f2_mul(unpack2_swapped(lo[i]), sin_lo[i]));
          c = f2_fma(f, cos_hi[i], f2_mul(unpack2_swapped(hi[i]), sin_hi[i]));
        } else {
          a = f2_fma(e, cos_lo[i], f2_mul(f, sin_lo[i]));
          c = f2_fma(f, cos_hi[i], f2_mul(e, sin_hi[i]));
        }
        if (norm) {
          a = f2_mul(a, scale);
          c = f2_mul(c, scale);
        }
        out_lo[i] = pack2(a);
        out_hi[i] = pack2(c);
      }
      if (live) {
        store16(dst + d * dst_step, make_uint4(out_lo[0], out_lo[1], out_lo[2], out_lo[3]));
        store16(dst + d * dst_step + 128, make_uint4(out_hi[0], out_hi[1], out_hi[2], out_hi[3]));
      }
    }
    src += kDepth * src_step;
    dst += kDepth * dst_step;
  }
}

template <bool kInterleaved, int kDepth, int kBlocksPerSm>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm) qk_norm_rope_kernel(const RotaryParams p) {
  __shared__ alignas(16) float2 turns_of[kWarps][kPairs];
  __shared__ alignas(16) float weights[2][128];  // 1 where there is none
  launch_dependents();
  wait_for_previous();
  for (int i = threadIdx.x; i < 256; i += kWarps * 32)
    weights[i >> 7][i & 127] = weight_of((i >> 7) ? p.k.weight : p.q.weight, p.weight_fp32, i & 127);
  __syncthreads();
  const int lane = threadIdx.x & 31, l = lane & 7, quarter = lane >> 3;
  // (64-bit divisions here cost as many instructions as two heads; there are fewer than 2^31 tokens, and chunks only
  // where there are few)
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t row = p.chunks == 1 ? unit : unit / uint32_t(p.chunks);
  const uint32_t b = p.batch == 1 ? 0 : row / uint32_t(p.tokens), t = row - b * uint32_t(p.tokens);
  if (b >= uint32_t(p.batch) || t >= uint32_t(p.tokens)) return;  // whole warps
  const int chunk = int(unit - row * uint32_t(p.chunks));
  float2* turn = turns_of[threadIdx.x >> 5];

  bool have = false;
  auto angles = [&]() {
    if (have) return;
    have = true;
#pragma unroll
    for (int i = 0; i < kPairs / 32; ++i) {
      const int j = lane + 32 * i;
      float2 cs = make_float2(1.0f, 0.0f);
      if (j < p.pairs) {
        int axis = 0;
#pragma unroll
        for (int a = 0; a < kRotaryMaxAxes - 1; ++a) axis += (j >= p.section_end[a]) ? 1 : 0;
        const double turns = position_of(p, axis, b, t) * (double(p.inv_freq[j]) * 0.15915494309189535);
        sincospif(2.0f * float(turns - rint(turns)), &cs.y, &cs.x);
      }
      turn[j] = cs;
    }
    __syncwarp();
  };
  // a warp's heads: some of q's, or of k's, or the last of q's and the first of k's
  const int first = chunk * p.chunk_heads, end = min(p.heads_q + p.heads_k, first + p.chunk_heads);
  if (first < p.heads_q)
    rotate_heads<kInterleaved, kDepth>(p.q, p, b, t, first + quarter, min(end, p.heads_q), l, turn, weights[0], angles);
  if (end > p.heads_q)
    rotate_heads<kInterleaved, kDepth>(p.k, p, b, t, max(first, p.heads_q) - p.heads_q + quarter, end - p.heads_q, l, turn, weights[1], angles);
}

}  // namespace

template <int kDepth, int kBlocksPerSm>
static cudaError_t launch_variant(const RotaryParams& p, bool interleaved, int64_t rows, cudaStream_t stream) {
  const int64_t blocks = (rows * p.chunks + kWarps - 1) / kWarps;
  return launch_overlapped(interleaved ? qk_norm_rope_kernel<true, kDepth, kBlocksPerSm>
                                       : qk_norm_rope_kernel<false, kDepth, kBlocksPerSm>,
                           unsigned(blocks), kWarps * 32, 0, stream, p);
}

cudaError_t launch_qk_norm_rope(RotaryParams p, bool interleaved, int sm_count, cudaStream_t stream) {
  const int64_t rows = int64_t(p.batch) * p.tokens;
  const int heads = p.heads_q + p.heads_k;
  // With few tokens a token's heads are spread over several warps (each works the angles out again), as far as all
  // warps are still resident at once.
  const int64_t resident = int64_t(sm_count) * 6 * kWarps, most = (heads + 3) / 4;
  int chunks = 1;
  if (rows * 2 <= resident) chunks = int(resident / rows < most ? resident / rows : most);
  p.chunk_heads = ((heads + chunks - 1) / chunks + 3) / 4 * 4;
  p.chunks = (heads + p.chunk_heads - 1) / p.chunk_heads;
  if (p.chunks > 1) return launch_variant<1, 6>(p, interleaved, rows, stream);
  if (heads <= kFewHeads) return launch_variant<1, 7>(p, interleaved, rows, stream);
  return launch_variant<2, 6>(p, interleaved, rows, stream);
}

}  // namespace b200attn
