// Tensor-level bodies of the packed, shared-prefix and norm-and-rotation calls: argument rules, outputs, workspace, launch.
// Behind b200_attention_b200.packed and .rotary (direct.cpp).
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <atomic>
#include <limits>
#include <memory>
#include <optional>
#include <tuple>

#include "../../include/b200_attention.h"
#include "overlap.h"

namespace b200attn_torch {

inline void check_rc(int rc) {
  TORCH_CHECK(rc == B200ATTN_OK, "b200attn: ", b200attn_status_string(rc), ": ",
              b200attn_last_error());
}

// These calls record nothing: neither for a backward pass nor along a forward-mode one (level 0 is the only one).
inline void check_no_gradient(const char* name, const at::Tensor& t) {
  TORCH_CHECK(!(t.requires_grad() && c10::GradMode::is_enabled()), name,
              " requires grad: this library computes forward passes only");
  TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()), name,
              " carries a tangent: this library has no forward-mode gradients");
}

inline void check_bf16(const char* name, const at::Tensor& t) {
  check_no_gradient(name, t);
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (this library has no CPU path)");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
}

inline void check_rows(const char* name, const at::Tensor& t, int64_t heads, const at::Device& device) {
  check_bf16(name, t);
  TORCH_CHECK(t.dim() == 3 && t.size(2) == 128, name, " must be [rows, heads, 128], got ", t.sizes());
  TORCH_CHECK(t.stride(2) == 1, name, ": the head_dim axis must be contiguous");
  TORCH_CHECK(t.size(1) == heads, name, " has ", t.size(1), " heads, the plan ", heads);
  TORCH_CHECK(t.device() == device, name, " is on ", t.device(), ", the plan on ", device);
  TORCH_CHECK(t.size(0) < (int64_t(1) << 31) - 256, name, " has too many rows");
}

inline b200attn_operand row_operand(const at::Tensor& t) { return {t.data_ptr(), 0, t.stride(1), t.stride(0)}; }

// What a plan says to a call: heads, heads_kv, rows_q, rows_kv, len_prefix, grid, join units, slot rows; then grid, join
// units and slot rows for a call that is being captured, whose replays may find the table of other lengths; last, the
// stream that the table was allocated on, and the plan's wide pieces.
constexpr size_t kPlanInts = 13;

inline at::Tensor empty_on(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

inline bool capturing(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
  return status != cudaStreamCaptureStatusNone;
}

// A graph's replays read the table of the plan that its calls were captured with, whatever has become of the plan: the
// graph owns a reference to it (a user object, which its executable form takes over) and gives it up when it is destroyed
// and no replay runs any more. That happens on a thread of CUDA's, where neither CUDA nor Python may be called, so the
// reference only goes to a list there; the next plan or call frees what is on it.
struct GraphTable {
  at::Tensor table;
  GraphTable* next;
};

inline std::atomic<GraphTable*>& tables_given_up() {
  static std::atomic<GraphTable*> list{nullptr};
  return list;
}

inline void CUDART_CB give_up_table(void* held) {
  GraphTable* t = static_cast<GraphTable*>(held);
  t->next = tables_given_up().load(std::memory_order_relaxed);
  while (!tables_given_up().compare_exchange_weak(t->next, t, std::memory_order_release, std::memory_order_relaxed)) {
  }
}

// With the GIL held: the tensors may have Python's objects.
inline void free_tables() {
  if (tables_given_up().load(std::memory_order_relaxed) == nullptr) return;
  for (GraphTable* t = tables_given_up().exchange(nullptr, std::memory_order_acquire); t != nullptr;) {
    GraphTable* next = t->next;
    delete t;
    t = next;
  }
}

// Before the call is captured, so that no graph holds a call without its table.
inline void keep_for_graph(cudaStream_t stream, const at::Tensor& table) {
  static unsigned long long last_capture = 0;  // of a capture's calls of one plan (one for each layer) the first does it
  static const void* last_table = nullptr;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  cudaGraph_t graph = nullptr;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &capture, &graph));
  TORCH_CHECK(status == cudaStreamCaptureStatusActive && graph != nullptr, "the capture of this stream has failed");
  if (capture == last_capture && table.const_data_ptr() == last_table) return;
  cudaUserObject_t object = nullptr;
  std::unique_ptr<GraphTable> held(new GraphTable{table, nullptr});
  C10_CUDA_CHECK(cudaUserObjectCreate(&object, held.get(), give_up_table, 1, cudaUserObjectNoDestructorSync));
  held.release();  // the object's now
  const cudaError_t e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) (void)cudaUserObjectRelease(object, 1);
  C10_CUDA_CHECK(e);
  last_capture = capture;
  last_table = table.const_data_ptr();
}

// A tensor that the caller gave as output: a backward pass that saved it must see that it has changed.
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Returns O, LSE (or an undefined tensor), and whether the call was captured.
inline std::tuple<at::Tensor, at::Tensor, bool> attention_planned(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                     const std::optional<at::Tensor>& k_prefix,
                                                     const std::optional<at::Tensor>& v_prefix, const at::Tensor& table,
                                                     at::IntArrayRef plan, double scale, bool return_lse,
                                                     const std::optional<at::Tensor>& out) {
  TORCH_CHECK(plan.size() == kPlanInts, "malformed plan");
  const int64_t heads = plan[0], heads_kv = plan[1], rows_q = plan[2], rows_kv = plan[3], len_prefix = plan[4];
  const at::Device device = table.device();
  check_rows("q", q, heads, device);
  check_rows("k", k, heads_kv, device);
  check_rows("v", v, heads_kv, device);
  TORCH_CHECK(k.size(0) == v.size(0), "k has ", k.size(0), " rows, v ", v.size(0));
  TORCH_CHECK(q.size(0) >= rows_q, "q has ", q.size(0), " rows, the plan covers ", rows_q);
  TORCH_CHECK(k.size(0) >= rows_kv, "k and v have ", k.size(0), " rows, the plan reads up to row ", rows_kv);
  if (len_prefix > 0) {
    TORCH_CHECK(k_prefix.has_value() && v_prefix.has_value(), "the plan has a prefix");
    check_rows("k_prefix", *k_prefix, heads_kv, device);
    check_rows("v_prefix", *v_prefix, heads_kv, device);
    TORCH_CHECK(k_prefix->size(0) >= len_prefix && v_prefix->size(0) >= len_prefix,
                "k_prefix or v_prefix has fewer than the plan's ", len_prefix, " rows");
  }
  if (out.has_value()) {
    TORCH_CHECK(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->device() == device &&
                    out->stride(2) == 1,
                "out must match q in shape, dtype and device with a dense head_dim axis");
    check_bf16("out", *out);
    // A CTA stores rows while others still load theirs.
    check_place("out", *out, "q", &q, {{"k", &k}, {"v", &v}, {"k_prefix", len_prefix > 0 ? &*k_prefix : nullptr},
                                       {"v_prefix", len_prefix > 0 ? &*v_prefix : nullptr}});
  }

  c10::cuda::CUDAGuard guard(device);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  const bool captured = capturing(stream);
  if (captured)
    keep_for_graph(stream, table);
  else
    free_tables();
  int64_t grid = plan[captured ? 8 : 5];
  const int64_t units = plan[captured ? 9 : 6], slots = plan[captured ? 10 : 7];
  if (k.size(0) == 0 && len_prefix == 0) grid = 0;  // no key for any replay to work on
  const int64_t rows = q.size(0);
  at::Tensor o = out.has_value() ? *out : empty_on({rows, heads, 128}, at::kBFloat16, device);
  at::Tensor lse;
  if (return_lse) lse = empty_on({heads, rows}, at::kFloat, device);
  if (rows > rows_q) {
    if (!out.has_value()) o.narrow(0, rows_q, rows - rows_q).zero_();
    if (return_lse) lse.narrow(1, rows_q, rows - rows_q).fill_(-std::numeric_limits<float>::infinity());
  }
  if (rows == 0 || (grid == 0 && units == 0)) return {o, lse, captured};
  // From the caching allocator at every call: in stream order, and private to a graph that is being captured.
  at::Tensor workspace;
  if (slots > 0) workspace = empty_on({slots * 129}, at::kFloat, device);
  b200attn_planned_args a{};
  a.struct_bytes = sizeof a;
  a.heads = int32_t(heads);
  a.heads_kv = int32_t(heads_kv);
  a.head_dim = 128;
  a.rows_q = int32_t(rows);
  a.rows_kv = int32_t(k.size(0));
  a.len_prefix = int32_t(len_prefix);
  a.grid = int32_t(grid);
  a.join_units = int32_t(units);
  a.wide_pieces = int32_t(plan[12]);
  a.q = row_operand(q);
  a.k = row_operand(k);
  a.v = row_operand(v);
  if (len_prefix > 0) {
    a.k_prefix = row_operand(*k_prefix);
    a.v_prefix = row_operand(*v_prefix);
  }
  a.o = row_operand(o);
  if (return_lse) {
    a.lse = lse.data_ptr<float>();
    a.lse_stride_head = rows;
  }
  a.softmax_scale = float(scale);
  a.table = table.data_ptr();
  a.workspace = slots > 0 ? workspace.data_ptr() : nullptr;
  a.slot_rows = slots;
  a.stream = stream;
  check_rc(b200attn_forward_planned(&a));
  if (out.has_value()) written(o);
  // A plan may go, or take another table, while a call on another stream than the table's own still reads it. (The table
  // of a captured call stays.)
  if (!captured && reinterpret_cast<int64_t>(stream) != plan[11])
    c10::cuda::CUDACachingAllocator::recordStream(table.storage().data_ptr(),
                                                  c10::cuda::getCurrentCUDAStream(device.index()));
  return {o, lse, captured};
}

inline void check_tokens(const char* name, const at::Tensor& t, const at::Tensor* like) {
  check_bf16(name, t);
  TORCH_CHECK((t.dim() == 3 || t.dim() == 4) && t.size(-1) == 128, name,
              " must be [tokens, heads, 128] or [batch, tokens, heads, 128], got ", t.sizes());
  TORCH_CHECK(t.stride(-1) == 1, name, ": the head_dim axis must be contiguous");
  if (like != nullptr) {
    TORCH_CHECK(t.device() == like->device(), name, " is on ", t.device(), ", q on ", like->device());
    TORCH_CHECK(t.dim() == like->dim() && t.sizes().slice(0, t.dim() - 2) == like->sizes().slice(0, t.dim() - 2), name,
                " and q disagree on batch or tokens: ", t.sizes(), ", ", like->sizes());
  }
}

// (batch, head, token); an axis of one entry is never stepped along
inline b200attn_operand token_operand(const at::Tensor& t) {
  auto step = [&](int64_t d) { return t.size(d) == 1 ? int64_t(0) : t.stride(d); };
  return {t.data_ptr(), t.dim() == 4 ? step(0) : 0, step(-2), step(-3)};
}

inline std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                                const at::Tensor& positions, const at::Tensor& inv_freq,
                                                at::IntArrayRef sections, const std::optional<at::Tensor>& q_weight,
                                                const std::optional<at::Tensor>& k_weight, double eps, bool interleaved,
                                                const std::optional<at::Tensor>& q_out,
                                                const std::optional<at::Tensor>& k_out) {
  const int64_t axes = int64_t(sections.size());
  int64_t pairs = 0;
  for (const int64_t n : sections) {
    TORCH_CHECK_VALUE(n >= 0 && n <= 64, "sections must be counts of 0 .. 64 pairs");
    pairs += n;
  }
  TORCH_CHECK_VALUE(axes >= 1 && axes <= 4 && pairs >= 1 && pairs <= 64,
                    "sections must be 1 to 4 counts that add up to 1 .. 64, got ", sections);
  TORCH_CHECK_VALUE(inv_freq.numel() == pairs, "inv_freq holds ", inv_freq.numel(), " frequencies, sections add up to ",
                    pairs);
  check_tokens("q", q, nullptr);
  if (k.has_value()) check_tokens("k", *k, &q);
  TORCH_CHECK(k.has_value() || !k_weight.has_value(), "k_weight is given without k");
  TORCH_CHECK(q.size(-2) > 0 || !k.has_value() || k->size(-2) == 0, "q has no heads, k has ", k.has_value() ? k->size(-2) : 0);
  const int64_t batch = q.dim() == 4 ? q.size(0) : 1, tokens = q.size(-3);
  TORCH_CHECK(positions.device() == q.device() && inv_freq.device() == q.device(),
              "positions and inv_freq must be on q's device");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous(),
              "inv_freq must be a contiguous fp32 vector");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong ||
                  positions.scalar_type() == at::kFloat,
              "positions must be int32, int64 or float32, got ", positions.scalar_type());
  const at::Tensor pos = positions.dim() == 1 ? positions.unsqueeze(0) : positions;
  TORCH_CHECK((pos.dim() == 2 && pos.size(0) == axes && pos.size(1) == tokens) ||
                  (pos.dim() == 3 && pos.size(0) == axes && pos.size(1) == batch && pos.size(2) == tokens),
              "positions must be [", axes, ", ", tokens, "] or [", axes, ", ", batch, ", ", tokens, "], got ",
              positions.sizes());
  check_no_gradient("positions", positions);
  check_no_gradient("inv_freq", inv_freq);
  const at::Tensor* weight[2] = {q_weight.has_value() ? &*q_weight : nullptr, k_weight.has_value() ? &*k_weight : nullptr};
  for (const at::Tensor* w : weight) {
    if (w == nullptr) continue;
    TORCH_CHECK(w->device() == q.device() && w->dim() == 1 && w->size(0) == 128 && w->is_contiguous() &&
                    (w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat),
                "a weight must be a contiguous bf16 or fp32 vector of 128 on q's device");
    check_no_gradient("a weight", *w);
  }
  TORCH_CHECK(weight[0] == nullptr || weight[1] == nullptr || weight[0]->scalar_type() == weight[1]->scalar_type(),
              "q_weight and k_weight must have the same type");
  const at::Tensor* given[2] = {q_out.has_value() ? &*q_out : nullptr, k_out.has_value() ? &*k_out : nullptr};
  if (given[0] != nullptr) {
    check_tokens("out of q", *given[0], &q);
    TORCH_CHECK(given[0]->sizes() == q.sizes(), "out of q must match q in shape");
  }
  if (given[1] != nullptr && k.has_value()) {
    check_tokens("out of k", *given[1], &q);
    TORCH_CHECK(given[1]->sizes() == k->sizes(), "out of k must match k in shape");
  }
  // q and k among one another: rotary.py
  for (const at::Tensor* out : given) {
    if (out == nullptr) continue;
    for (const at::Tensor* read : {&positions, &inv_freq, weight[0], weight[1]})
      TORCH_CHECK(read == nullptr || !may_overlap(*out, *read), "an output overlaps positions, inv_freq or a weight");
  }

  c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor qo = given[0] != nullptr ? *given[0] : empty_on(q.sizes(), at::kBFloat16, q.device());
  at::Tensor ko;
  if (k.has_value()) ko = given[1] != nullptr ? *given[1] : empty_on(k->sizes(), at::kBFloat16, k->device());
  if (batch * tokens == 0 || q.size(-2) == 0) return {qo, ko};
  TORCH_CHECK(batch * tokens < (int64_t(1) << 31) && q.size(-2) < (1 << 16) && (!k.has_value() || k->size(-2) < (1 << 16)),
              "too many tokens or heads");
  b200attn_qk_norm_rope_args a{};
  a.struct_bytes = sizeof a;
  a.batch = int32_t(batch);
  a.tokens = int32_t(tokens);
  a.heads_q = int32_t(q.size(-2));
  a.head_dim = 128;
  a.q = token_operand(q);
  a.q_out = token_operand(qo);
  if (k.has_value() && k->size(-2) > 0) {
    a.heads_k = int32_t(k->size(-2));
    a.k = token_operand(*k);
    a.k_out = token_operand(ko);
  }
  a.q_weight = weight[0] != nullptr ? weight[0]->data_ptr() : nullptr;
  a.k_weight = weight[1] != nullptr ? weight[1]->data_ptr() : nullptr;
  const at::Tensor* any_weight = weight[0] != nullptr ? weight[0] : weight[1];
  a.weight_type = any_weight != nullptr && any_weight->scalar_type() == at::kFloat ? 1 : 0;
  a.position_type = pos.scalar_type() == at::kInt ? 0 : pos.scalar_type() == at::kLong ? 1 : 2;
  a.positions = pos.data_ptr();
  a.position_stride_axis = pos.stride(0);
  a.position_stride_batch = pos.dim() == 3 ? pos.stride(1) : 0;
  a.position_stride_token = pos.stride(-1);
  a.inv_freq = inv_freq.data_ptr<float>();
  a.axes = int32_t(axes);
  for (int64_t i = 0; i < axes; ++i) a.section[i] = int32_t(sections[size_t(i)]);
  a.eps = float(eps);
  a.interleaved = interleaved ? 1 : 0;
  a.stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  check_rc(b200attn_qk_norm_rope(&a));
  if (given[0] != nullptr) written(qo);
  if (given[1] != nullptr && a.heads_k > 0) written(ko);
  return {qo, ko};
}

}  // namespace b200attn_torch
