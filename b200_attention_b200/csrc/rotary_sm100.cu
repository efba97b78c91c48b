// Norm of queries and keys for each head, and their rotation by position, in one pass (sm_100a).
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (128 values of a head; only where a weight is given)
//   pair j of y:  (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position[axis(j)] * inv_freq[j]
//   pairs are (j, j + 64), or (2j, 2j + 1) when interleaved; pairs behind the last section stay as they are
//
// Bound by memory: 512 bytes per head and token for about 10 operations per value. A warp takes one token, half a
// warp one head: a lane holds eight values of a head, which are four whole pairs in either pairing, so the only
// exchange is the sum of squares over 16 lanes. The angles depend on the token and the pair alone: a lane works
// its four out once and uses them for every head that the warp visits.
// Statistics and rotation are in 32 bits and rounded to bf16 once. Angles are reduced to a fraction of a turn in
// 64 bits first: at position 10^6 a 32-bit product is already off by 0.03 radians.

#include "rotary_kernels.cuh"

#include <cuda_bf16.h>

namespace b200attn {

namespace {

constexpr int kWarps = 8;
constexpr int kHeadsPerStep = 4;  // heads that a half warp has in flight

struct alignas(8) Half4 {
  __nv_bfloat162 lo, hi;
};

__device__ __forceinline__ double position_of(const RotaryParams& p, int axis, int64_t b, int64_t t) {
  const int64_t at = axis * p.pos_stride_axis + b * p.pos_stride_batch + t * p.pos_stride_token;
  if (p.pos_type == 0) return double(static_cast<const int32_t*>(p.positions)[at]);
  if (p.pos_type == 1) return double(static_cast<const int64_t*>(p.positions)[at]);
  return double(static_cast<const float*>(p.positions)[at]);
}

__device__ __forceinline__ void unpack4(uint2 raw, float (&v)[4]) {
  v[0] = __uint_as_float(raw.x << 16);
  v[1] = __uint_as_float(raw.x & 0xffff0000u);
  v[2] = __uint_as_float(raw.y << 16);
  v[3] = __uint_as_float(raw.y & 0xffff0000u);
}

__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
  union {
    Half4 h;
    uint2 u;
  } r;
  r.h.lo = __floats2bfloat162_rn(a, b);
  r.h.hi = __floats2bfloat162_rn(c, d);
  return r.u;
}

__device__ __forceinline__ float weight_of(const void* w, int is_fp32, int i) {
  return is_fp32 ? static_cast<const float*>(w)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// kInterleaved: values 8l .. 8l + 7 of a head in lane l of a half warp; otherwise 4l .. 4l + 3 and 64 + 4l .. + 3.
// Either way a[i], b[i] are the two values of pair 4l + i.
template <bool kInterleaved>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_rope_kernel(const RotaryParams p) {
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t row = unit / p.chunks;
  if (row >= int64_t(p.batch) * p.tokens) return;
  const int chunk = int(unit - row * p.chunks);
  const int64_t b = row / p.tokens, t = row - b * p.tokens;

  float cosv[4], sinv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = 4 * l + i;
    cosv[i] = 1.0f;
    sinv[i] = 0.0f;
    if (j < p.pairs) {
      int axis = 0;
#pragma unroll
      for (int a = 0; a < kRotaryMaxAxes - 1; ++a) axis += (j >= p.section_end[a]) ? 1 : 0;
      const double turns = position_of(p, axis, b, t) * (double(p.inv_freq[j]) * 0.15915494309189535);
      sincospif(2.0f * float(turns - rint(turns)), &sinv[i], &cosv[i]);
    }
  }

  const int heads = p.heads_q + p.heads_k;
  const int first = chunk * p.chunk_heads, end = min(heads, first + p.chunk_heads);
  for (int h0 = first; h0 < end; h0 += 2 * kHeadsPerStep) {
    uint2 raw[kHeadsPerStep][2];
#pragma unroll
    for (int s = 0; s < kHeadsPerStep; ++s) {
      const int h = h0 + 2 * s + half;
      if (h < end) {
        const bool is_k = h >= p.heads_q;
        const RotaryOperand& x = is_k ? p.k : p.q;
        const __nv_bfloat16* src = x.in + b * x.in_stride_b + int64_t(is_k ? h - p.heads_q : h) * x.in_stride_h + t * x.in_stride_t;
        if (kInterleaved) {
          const uint4 r = *reinterpret_cast<const uint4*>(src + 8 * l);
          raw[s][0] = make_uint2(r.x, r.y);
          raw[s][1] = make_uint2(r.z, r.w);
        } else {
          raw[s][0] = *reinterpret_cast<const uint2*>(src + 4 * l);
          raw[s][1] = *reinterpret_cast<const uint2*>(src + 64 + 4 * l);
        }
      } else {
        raw[s][0] = raw[s][1] = make_uint2(0u, 0u);
      }
    }
#pragma unroll
    for (int s = 0; s < kHeadsPerStep; ++s) {
      const int h = h0 + 2 * s + half;
      const bool is_k = h >= p.heads_q;
      const RotaryOperand& x = is_k ? p.k : p.q;
      float v[2][4];
      unpack4(raw[s][0], v[0]);
      unpack4(raw[s][1], v[1]);
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = fmaf(v[0][i], v[0][i], fmaf(v[1][i], v[1][i], sq));
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
      if (h >= end) continue;
      if (x.weight != nullptr) {
        const float scale = rsqrtf(sq * (1.0f / 128.0f) + p.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[0][i] *= scale * weight_of(x.weight, p.weight_fp32, kInterleaved ? 8 * l + i : 4 * l + i);
          v[1][i] *= scale * weight_of(x.weight, p.weight_fp32, kInterleaved ? 8 * l + 4 + i : 64 + 4 * l + i);
        }
      }
      float a[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = kInterleaved ? v[i >> 1][2 * (i & 1)] : v[0][i];
        const float f = kInterleaved ? v[i >> 1][2 * (i & 1) + 1] : v[1][i];
        a[i] = e * cosv[i] - f * sinv[i];
        c[i] = f * cosv[i] + e * sinv[i];
      }
      __nv_bfloat16* dst = x.out + b * x.out_stride_b + int64_t(is_k ? h - p.heads_q : h) * x.out_stride_h + t * x.out_stride_t;
      if (kInterleaved) {
        const uint2 lo = pack4(a[0], c[0], a[1], c[1]), hi = pack4(a[2], c[2], a[3], c[3]);
        *reinterpret_cast<uint4*>(dst + 8 * l) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        *reinterpret_cast<uint2*>(dst + 4 * l) = pack4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint2*>(dst + 64 + 4 * l) = pack4(c[0], c[1], c[2], c[3]);
      }
    }
  }
}

}  // namespace

cudaError_t launch_qk_norm_rope(RotaryParams p, bool interleaved, int sm_count, cudaStream_t stream) {
  const int64_t rows = int64_t(p.batch) * p.tokens;
  const int heads = p.heads_q + p.heads_k;
  // With few tokens a token's heads are spread over several warps (each works the angles out again).
  const int64_t wanted = int64_t(sm_count) * 32;
  int chunks = 1;
  if (rows < wanted) {
    const int64_t most = (heads + 1) / 2;
    chunks = int((wanted + rows - 1) / rows < most ? (wanted + rows - 1) / rows : most);
  }
  p.chunk_heads = ((heads + chunks - 1) / chunks + 1) / 2 * 2;
  p.chunks = (heads + p.chunk_heads - 1) / p.chunk_heads;
  const int64_t blocks = (rows * p.chunks + kWarps - 1) / kWarps;
  if (interleaved)
    qk_norm_rope_kernel<true><<<unsigned(blocks), kWarps * 32, 0, stream>>>(p);
  else
    qk_norm_rope_kernel<false><<<unsigned(blocks), kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace b200attn
