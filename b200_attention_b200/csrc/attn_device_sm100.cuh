// Device-side parts shared by the attention kernels: tile and descriptor constants, bounded waits,
// MMA issue helpers and the per-row softmax arithmetic.
#pragma once

#include "attn_kernels.cuh"
#include "ptx_sm100.cuh"

#include <cfloat>
#include <cmath>

namespace b200attn {

namespace {

using namespace ptx;

constexpr int kTileBytes = kBlockM * kHeadDim * 2;  // 32 KiB: one Q, K or V tile
constexpr int kBoxBytes = kTileBytes / 2;           // one 64-column TMA box
constexpr int kSwizzleGroupBytes = 1024;            // 8 rows x 128 bytes
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

constexpr uint32_t kIdescQK = umma_idesc_bf16(kBlockM, kBlockN, /*b_mn_major=*/false);
constexpr uint32_t kIdescPV = umma_idesc_bf16(kBlockM, kHeadDim, /*b_mn_major=*/true);

// ------------------------------------------------------------------------------------------
// Bounded waits
// ------------------------------------------------------------------------------------------
// Suspend-time hint of the polls in the slow path of a wait (see mbarrier.try_wait).
#ifndef B200ATTN_WAIT_HINT_NS
#define B200ATTN_WAIT_HINT_NS 1000
#endif

struct WaitCtx {
  uint32_t abort_addr;  // shared-memory word: non-zero once any thread of the CTA gave up
  int32_t* status;
  uint64_t limit_ns;
  int32_t item;
  int32_t tile;

  __device__ __forceinline__ bool aborted() const {
    uint32_t v;
    asm volatile("ld.volatile.shared::cta.u32 %0, [%1];\n" : "=r"(v) : "r"(abort_addr));
    return v != 0;
  }

  __device__ __forceinline__ void raise(int code, int site, uint32_t parity) const {
    asm volatile("st.volatile.shared::cta.u32 [%0], %1;\n" ::"r"(abort_addr), "r"(1u) : "memory");
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
      status[1] = site;
      status[2] = static_cast<int32_t>(blockIdx.x);
      status[3] = static_cast<int32_t>(threadIdx.x >> 5);
      status[4] = static_cast<int32_t>(parity);
      status[5] = item;
      status[6] = tile;
      __threadfence_system();
    }
  }

  __device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, int site) const {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t n = 1;; ++n) {
      if (mbar_try_wait(bar, parity, B200ATTN_WAIT_HINT_NS)) return true;
      if ((n & 7u) == 0) {
        if (aborted()) return false;
        if (global_timer_ns() - t0 > limit_ns) {
          raise(kDevWaitTimeout, site, parity);
          return false;
        }
      }
    }
  }

  // For roles run by a single thread.
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int site) const {
    if (mbar_try_wait(bar, parity, 0)) return true;
    return wait_slow(bar, parity, site);
  }

  // For the MMA and TMA roles, which whole warps run with uniform control flow.
  __device__ __forceinline__ bool wait_issue(uint32_t bar, uint32_t parity, int site) const {
    return wait_warp(bar, parity, site);
  }

  // For roles run by whole warps: every lane returns the same answer, so the warp stays
  // converged for the .sync.aligned TMEM instructions that follow.
  __device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int site) const {
    bool ok = mbar_try_wait(bar, parity, 0);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (!ok) ok = wait_slow(bar, parity, site);
    return __all_sync(0xffffffffu, ok);
  }
};

// ------------------------------------------------------------------------------------------
// MMA issue helpers (called by one thread)
// ------------------------------------------------------------------------------------------
// (No warp-level synchronisation in these helpers: the serial kernel calls them from one thread.)
// S[128 x 128] = Q_tile * K_tile^T, eight K=16 steps over head_dim. Called by a whole warp with
// uniform operands (so descriptors live in uniform registers); the lane with lead != 0 issues the
// eight MMAs inside one branch. Measured at B4 H16 L8192: whole-warp roles 1311 TFLOPS, the
// same roles run by a single lane 1080.
__device__ __forceinline__ void issue_qk(uint32_t lead, uint32_t s_tmem, uint32_t q_smem,
                                         uint32_t k_smem) {
  constexpr uint32_t hi = umma_desc_hi_sw128(kSwizzleGroupBytes);
  const uint32_t a0 = umma_desc_lo(q_smem, 0);
  const uint32_t b0 = umma_desc_lo(k_smem, 0);
  if (lead) {
#pragma unroll
    for (int kk = 0; kk < kHeadDim / 16; ++kk) {
      const uint32_t off = uint32_t(((kk >> 2) * kBoxBytes + (kk & 3) * 32) >> 4);
      umma_ss(s_tmem, a0 + off, hi, b0 + off, hi, kIdescQK, kk > 0 ? 1u : 0u);
    }
  }
}
// O[128 x 128] (+)= P[128 x 128 keys] * V_tile, eight K = 16 steps over the keys. P is bf16
// pairs in TMEM, 8 columns per K step starting at p_tmem.
__device__ __forceinline__ void issue_pv(uint32_t lead, uint32_t o_tmem, uint32_t p_tmem,
                                         uint32_t v_smem, bool accumulate) {
  constexpr uint32_t hi = umma_desc_hi_sw128(kSwizzleGroupBytes);
  const uint32_t b0 = umma_desc_lo(v_smem, kBoxBytes);
  if (lead) {
#pragma unroll
    for (int kk = 0; kk < kBlockN / 16; ++kk) {
      const uint32_t off = uint32_t((kk * 16 * 128) >> 4);
      umma_ts(o_tmem, p_tmem + kk * 8, b0 + off, hi, kIdescPV, (kk > 0 || accumulate) ? 1u : 0u);
    }
  }
}

// ------------------------------------------------------------------------------------------
// Softmax arithmetic: one query row per thread
// ------------------------------------------------------------------------------------------
// Keys at or beyond `valid` are masked: push their scores to -inf. Any `valid` will do: none of the tile's keys is left
// where it is 0 or less, all of them where it is 128 or more.
__device__ __forceinline__ void mask_tail(uint32_t (&s)[4][32], int valid) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (c * 32 + j >= valid) s[c][j] = __float_as_uint(kNegInf);
    }
  }
}

__device__ __forceinline__ float row_max(const uint32_t (&s)[4][32]) {
  float m0 = kNegInf, m1 = kNegInf, m2 = kNegInf, m3 = kNegInf;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      m0 = max3(m0, __uint_as_float(s[c][j + 0]), __uint_as_float(s[c][j + 1]));
      m1 = max3(m1, __uint_as_float(s[c][j + 2]), __uint_as_float(s[c][j + 3]));
      m2 = max3(m2, __uint_as_float(s[c][j + 4]), __uint_as_float(s[c][j + 5]));
      m3 = max3(m3, __uint_as_float(s[c][j + 6]), __uint_as_float(s[c][j + 7]));
    }
  }
  return fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
}

// A row keeps its reference maximum m until some score exceeds m by this many log2 units.
// With bf16 probabilities and fp32 sums nothing overflows or loses relative precision until the
// excess nears 2^100, so the bound can be generous; 32 makes a rebase a once-in-a-blue-moon event
// on real data while leaving 2^(127-32-20) of headroom for row sums over a million keys.
#ifndef B200ATTN_REBASE_LOG2
#define B200ATTN_REBASE_LOG2 32.0f
#endif

// 2^(s * c - m) for one 32-column chunk: 16 packed bf16 pairs out, row-sum pairs accumulated.
__device__ __forceinline__ void exp_chunk(const uint32_t (&s)[32], f2 scale2, f2 neg_m2,
                                          uint32_t (&packed)[16], f2& sum_a, f2& sum_b) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const f2 x = f2_fma(f2_make(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), scale2,
                        neg_m2);
    float x0, x1;
    f2_split(x, x0, x1);
    const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
    const f2 e = f2_make(e0, e1);
    if (j & 1) sum_b = f2_add(sum_b, e); else sum_a = f2_add(sum_a, e);
    packed[j] = pack_bf16x2(e0, e1);
  }
}

__device__ __forceinline__ float f2_hsum(f2 a, f2 b) {
  float lo, hi;
  f2_split(f2_add(a, b), lo, hi);
  return lo + hi;
}

}  // namespace
}  // namespace b200attn
