// C ABI of the planned attention calls and of the norm-and-rotation of queries and keys: argument checks, tensor
// maps and launches. See include/b200_attention.h.

#include "host_common.cuh"
#include "plan_kernels.cuh"
#include "rotary_kernels.cuh"

#include <cmath>
#include <cstring>
#include <new>

using namespace b200attn;
using namespace b200attn::host;

namespace {

constexpr uint64_t kSlotRowBytes = (kHeadDim + 1) * sizeof(float);

// A size-1 axis may come with any stride: it is never stepped along.
b200attn_operand with_extents(b200attn_operand t, int32_t heads, int32_t len) {
  t.stride_batch = 0;
  if (heads == 1) t.stride_head = 0;
  if (len == 1) t.stride_row = 0;
  return t;
}

int check_rotary_operand(const char* name, const b200attn_operand& t, const b200attn_qk_norm_rope_args& a, int heads) {
  if (t.ptr == nullptr) return fail(B200ATTN_ERR_INVALID_ARGUMENT, std::string(name) + ": null pointer");
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 15u) != 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, std::string(name) + ": pointer must be 16-byte aligned");
  const int64_t s[3] = {t.stride_batch, t.stride_head, t.stride_row};
  const int32_t ext[3] = {a.batch, heads, a.tokens};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && (s[i] % 8 != 0 || s[i] >= (int64_t(1) << 38) || s[i] <= -(int64_t(1) << 38)))
      return fail(B200ATTN_ERR_INVALID_ARGUMENT, std::string(name) + ": strides must be multiples of 8 elements and < 2^38");
  return B200ATTN_OK;
}

}  // namespace

extern "C" {

int b200attn_plan_create(const b200attn_plan_desc* d, b200attn_plan_info* info, void** out) {
  if (d == nullptr || info == nullptr || out == nullptr) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (d->struct_bytes != sizeof *d || info->struct_bytes != sizeof *info)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "struct_bytes does not match this library's structures");
  if (d->reserved != 0) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "reserved fields must be 0");
  if (d->len_q == nullptr || d->len_kv == nullptr)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "len_q and len_kv must be given");
  try {
    PlanInput in{};
    in.sequences = d->sequences;
    in.len_q = d->len_q;
    in.len_kv = d->len_kv;
    in.start_kv = d->start_kv;
    in.len_prefix = d->len_prefix;
    in.heads = d->heads;
    in.heads_kv = d->heads_kv;
    in.causal = d->causal != 0;
    in.sm_count = d->sm_count == 0 ? 148 : d->sm_count;
    Plan* plan = new Plan;
    std::string wrong;
    try {
      wrong = plan_build(in, plan);
    } catch (...) {
      delete plan;
      throw;
    }
    if (!wrong.empty()) {
      delete plan;
      return fail(B200ATTN_ERR_INVALID_ARGUMENT, wrong);
    }
    info->grid = plan->grid;
    info->pieces = plan->pieces;
    info->units = plan->units;
    info->wide_pieces = plan->wide_pieces;
    info->reserved = 0;
    info->rows_q = plan->rows_q;
    info->rows_kv = plan->rows_kv;
    info->slot_rows = plan->slot_rows;
    info->table_bytes = plan->table.size() * sizeof(int32_t);
    info->workspace_bytes = uint64_t(plan->slot_rows) * kSlotRowBytes;
    *out = plan;
    return B200ATTN_OK;
  } catch (const std::bad_alloc&) {
    return fail(B200ATTN_ERR_UNSUPPORTED, "out of host memory while planning");
  } catch (...) {
    return fail(B200ATTN_ERR_UNSUPPORTED, "planning failed");
  }
}

int b200attn_plan_table(const void* plan, void* table, uint64_t bytes) {
  if (plan == nullptr || table == nullptr) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "null argument");
  const Plan* p = static_cast<const Plan*>(plan);
  if (bytes < p->table.size() * sizeof(int32_t))
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "the buffer is smaller than the plan's table");
  memcpy(table, p->table.data(), p->table.size() * sizeof(int32_t));
  return B200ATTN_OK;
}

int b200attn_plan_destroy(void* plan) {
  delete static_cast<Plan*>(plan);
  return B200ATTN_OK;
}

int b200attn_forward_planned(const b200attn_planned_args* a) {
  if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "args is null");
  if (a->struct_bytes != sizeof *a)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "struct_bytes does not match this library's b200attn_planned_args");
  if (a->reserved != 0) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "reserved fields must be 0");
  if (a->head_dim != kHeadDim) return fail(B200ATTN_ERR_UNSUPPORTED, "head_dim must be 128");
  if (a->heads < 1 || a->heads_kv < 1 || a->heads % a->heads_kv != 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "heads must be a positive multiple of heads_kv");
  const int group = a->heads / a->heads_kv;
  if (group > kBlockM) return fail(B200ATTN_ERR_UNSUPPORTED, "more than 128 query heads per K/V head");
  if (a->rows_q < 1 || a->rows_kv < 0 || a->len_prefix < 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "rows_q must be positive, rows_kv and len_prefix not negative");
  if (a->grid < 0 || a->grid > kPlanMaxCtas || a->join_units < 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "grid must be 0 .. 160, join_units not negative");
  if (a->grid > 0 && a->rows_kv == 0 && a->len_prefix == 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "there are no keys to work on");
  if (a->table == nullptr || (reinterpret_cast<uintptr_t>(a->table) & 15u) != 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "table must be given, 16-byte aligned");
  if (a->slot_rows < 0 || (a->slot_rows > 0 && (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 31u) != 0)))
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "workspace must be given for slot_rows > 0, 32-byte aligned");
  if (a->lse != nullptr && a->lse_stride_head < a->rows_q && a->heads > 1)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "lse_stride_head must be at least rows_q");
  if (!std::isfinite(a->softmax_scale)) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "softmax_scale must be finite");
  const b200attn_operand q = with_extents(a->q, a->heads, a->rows_q), o = with_extents(a->o, a->heads, a->rows_q);
  const b200attn_operand k = with_extents(a->k, a->heads_kv, a->rows_kv), v = with_extents(a->v, a->heads_kv, a->rows_kv);
  const b200attn_operand kp = with_extents(a->k_prefix, a->heads_kv, a->len_prefix);
  const b200attn_operand vp = with_extents(a->v_prefix, a->heads_kv, a->len_prefix);
  int rc;
  if ((rc = check_operand("q", q, 1, a->heads, a->rows_q)) != 0) return rc;
  if ((rc = check_operand("o", o, 1, a->heads, a->rows_q)) != 0) return rc;
  if (a->rows_kv > 0) {
    if ((rc = check_operand("k", k, 1, a->heads_kv, a->rows_kv)) != 0) return rc;
    if ((rc = check_operand("v", v, 1, a->heads_kv, a->rows_kv)) != 0) return rc;
  }
  if (a->len_prefix > 0) {
    if ((rc = check_operand("k_prefix", kp, 1, a->heads_kv, a->len_prefix)) != 0) return rc;
    if ((rc = check_operand("v_prefix", vp, 1, a->heads_kv, a->len_prefix)) != 0) return rc;
  }

  int device = 0, sm_count = 0;
  PlanParams p;
  memset(&p, 0, sizeof p);
  if ((rc = current_device(&device, &sm_count, &p.status)) != 0) return rc;
  p.table = static_cast<const int32_t*>(a->table);
  p.o = static_cast<__nv_bfloat16*>(const_cast<void*>(o.ptr));
  p.lse = a->lse;
  p.o_stride_t = o.stride_row;
  p.o_stride_h = o.stride_head;
  p.lse_stride_h = a->lse_stride_head;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_lse = p.part_o == nullptr ? nullptr : p.part_o + a->slot_rows * kHeadDim;
  p.o_aligned = reinterpret_cast<uintptr_t>(o.ptr) % 32 == 0 && o.stride_row % 16 == 0 && o.stride_head % 16 == 0;
  p.group = group;
  p.tile_tokens = plan_tile_tokens(group);
  p.tile_rows = p.tile_tokens * group;
  p.small_tokens = plan_small_tokens(group);
  const float scale = a->softmax_scale > 0.0f ? a->softmax_scale : 1.0f / std::sqrt(float(kHeadDim));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.wait_limit_ms = g_wait_limit_ms.load(std::memory_order_relaxed);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);

  if (a->grid > 0) {
    PlanMaps maps;
    MapKey kq{q.ptr, 0, q.stride_head, q.stride_row, 1, a->heads_kv, a->rows_q, device};
    kq.group = group;
    kq.box_tokens = p.tile_tokens;
    if ((rc = make_tensor_map(kq, &maps.q)) != 0) return rc;
    maps.q_small = maps.q;
    kq.box_tokens = p.small_tokens;
    if (p.small_tokens > 0 && (rc = make_tensor_map(kq, &maps.q_small)) != 0) return rc;
    const b200attn_operand* src[4] = {&k, &v, &kp, &vp};
    CUtensorMap* dst[4] = {&maps.k, &maps.v, &maps.k_prefix, &maps.v_prefix};
    for (int i = 0; i < 4; ++i) {
      const int32_t rows = i < 2 ? a->rows_kv : a->len_prefix;
      if (rows == 0) continue;
      const MapKey key{src[i]->ptr, 0, src[i]->stride_head, src[i]->stride_row, 1, a->heads_kv, rows, device};
      if ((rc = make_tensor_map(key, dst[i])) != 0) return rc;
    }
    // a pair that has no rows is not read; its maps are the other pair's
    if (a->rows_kv == 0) maps.k = maps.k_prefix, maps.v = maps.v_prefix;
    if (a->len_prefix == 0) maps.k_prefix = maps.k, maps.v_prefix = maps.v;
    const cudaError_t e = launch_plan(maps, p, a->grid, a->wide_pieces > 0, stream);
    if (e != cudaSuccess) return fail_cuda("kernel launch", e);
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  if (a->join_units > 0) {
    const int most = sm_count * 8;  // blocks that are resident at once
    const cudaError_t e = launch_plan_join(p, a->join_units < most ? a->join_units : most, stream);
    if (e != cudaSuccess) return fail_cuda("kernel launch", e);
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  return B200ATTN_OK;
}

int b200attn_qk_norm_rope(const b200attn_qk_norm_rope_args* a) {
  if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "args is null");
  if (a->struct_bytes != sizeof *a)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "struct_bytes does not match this library's b200attn_qk_norm_rope_args");
  if (a->reserved != 0) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "reserved fields must be 0");
  if (a->head_dim != kHeadDim) return fail(B200ATTN_ERR_UNSUPPORTED, "head_dim must be 128");
  if (a->batch < 1 || a->tokens < 1 || a->heads_q < 1 || a->heads_k < 0)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "batch, tokens and heads_q must be positive, heads_k not negative");
  if (int64_t(a->heads_q) + a->heads_k > 65535) return fail(B200ATTN_ERR_UNSUPPORTED, "too many heads");
  if (int64_t(a->batch) * a->tokens >= (int64_t(1) << 31)) return fail(B200ATTN_ERR_UNSUPPORTED, "too many tokens");
  if (a->axes < 1 || a->axes > kRotaryMaxAxes) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "axes must be 1 .. 4");
  RotaryParams p;
  memset(&p, 0, sizeof p);
  int pairs = 0;
  for (int i = 0; i < kRotaryMaxAxes; ++i) {
    if (i < a->axes) {
      if (a->section[i] < 0 || a->section[i] > kHeadDim / 2)
        return fail(B200ATTN_ERR_INVALID_ARGUMENT, "sections must be 0 .. 64 pairs");
      pairs += a->section[i];
    }
    p.section_end[i] = pairs;
  }
  if (pairs < 1 || pairs > kHeadDim / 2)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "the sections must add up to 1 .. 64 pairs");
  if (a->weight_type < 0 || a->weight_type > 1 || a->position_type < 0 || a->position_type > 2)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "unknown weight_type or position_type");
  if (a->positions == nullptr || a->inv_freq == nullptr)
    return fail(B200ATTN_ERR_INVALID_ARGUMENT, "positions and inv_freq must be given");
  if (!(a->eps >= 0.0f) || std::isinf(a->eps)) return fail(B200ATTN_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  int rc;
  if ((rc = check_rotary_operand("q", a->q, *a, a->heads_q)) != 0) return rc;
  if ((rc = check_rotary_operand("q_out", a->q_out, *a, a->heads_q)) != 0) return rc;
  if (a->heads_k > 0) {
    if ((rc = check_rotary_operand("k", a->k, *a, a->heads_k)) != 0) return rc;
    if ((rc = check_rotary_operand("k_out", a->k_out, *a, a->heads_k)) != 0) return rc;
  }
  int device = 0, sm_count = 0;
  int32_t* status = nullptr;
  if ((rc = current_device(&device, &sm_count, &status)) != 0) return rc;

  auto operand = [](const b200attn_operand& in, const b200attn_operand& out, const void* weight) {
    RotaryOperand r;
    r.in = static_cast<const __nv_bfloat16*>(in.ptr);
    r.out = static_cast<__nv_bfloat16*>(const_cast<void*>(out.ptr));
    r.in_stride_b = in.stride_batch;
    r.in_stride_h = in.stride_head;
    r.in_stride_t = in.stride_row;
    r.out_stride_b = out.stride_batch;
    r.out_stride_h = out.stride_head;
    r.out_stride_t = out.stride_row;
    r.weight = weight;
    return r;
  };
  p.q = operand(a->q, a->q_out, a->q_weight);
  p.k = operand(a->k, a->k_out, a->k_weight);
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.heads_q = a->heads_q;
  p.heads_k = a->heads_k;
  p.positions = a->positions;
  p.pos_stride_axis = a->position_stride_axis;
  p.pos_stride_batch = a->position_stride_batch;
  p.pos_stride_token = a->position_stride_token;
  p.pos_type = a->position_type;
  p.weight_fp32 = a->weight_type;
  p.inv_freq = a->inv_freq;
  p.pairs = pairs;
  p.eps = a->eps;
  const cudaError_t e = launch_qk_norm_rope(p, a->interleaved != 0, sm_count, static_cast<cudaStream_t>(a->stream));
  if (e != cudaSuccess) return fail_cuda("kernel launch", e);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return B200ATTN_OK;
}

}  // extern "C"
