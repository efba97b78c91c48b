// Whether strided tensors can share memory: arithmetic on addresses, sizes and strides, for the rules on outputs that a
// caller brings. No device.
#pragma once

#include <ATen/ATen.h>

#include <algorithm>
#include <array>
#include <cstdint>

namespace b200attn_torch {

// A tensor as runs of bytes: the first run's address, a run's length, and the axes along which runs repeat.
struct Runs {
  static constexpr int kMaxAxes = 8;
  struct Axis {
    int64_t step, count;  // bytes, entries (> 1)
  };
  int64_t first = 0, length = 0, last = 0;  // last: address behind the last byte
  int axes = 0;
  std::array<Axis, kMaxAxes> axis;
  bool empty = false, known = true;  // known: few enough axes

  explicit Runs(const at::Tensor& t) : first(int64_t(reinterpret_cast<uintptr_t>(t.const_data_ptr()))), length(t.element_size()) {
    const int64_t item = t.element_size();
    empty = t.numel() == 0;
    if (empty) return;
    for (int64_t d = t.dim() - 1; d >= 0; --d) {
      const int64_t n = t.size(d), step = t.stride(d) * item;
      if (n == 1) continue;
      if (step == length && axes == 0) {
        length *= n;
      } else if (axes < kMaxAxes) {
        axis[size_t(axes++)] = {step, n};
      } else {
        known = false;
      }
    }
    last = first + length;
    for (int i = 0; i < axes; ++i) last += axis[size_t(i)].step * (axis[size_t(i)].count - 1);
    std::sort(axis.begin(), axis.begin() + axes, [](const Axis& x, const Axis& y) { return x.step > y.step; });
  }
};

// True where the tensors share a byte, or where that would take long to find out.
inline bool may_overlap(const at::Tensor& a, const at::Tensor& b) {
  const Runs x(a), y(b);
  if (x.empty || y.empty) return false;
  if (!x.known || !y.known) return true;
  if (x.last <= y.first || y.last <= x.first) return false;
  // Runs i of x and j of y meet iff  x.first - y.first + sum i_d step_d - sum j_d step_d  lies in
  // [-(x.length - 1), y.length - 1]: a sum of whole multiples of steps, each multiple of a limited range (one range for
  // the two tensors' axes of the same step), that has to fall into an interval. Largest step first; where steps nest,
  // as in any real layout, one or two multiples of each are left to look at.
  struct Term {
    int64_t step, low, high;
  };
  std::array<Term, 2 * Runs::kMaxAxes + 1> term;
  int terms = 0;
  for (int i = 0, j = 0; i < x.axes || j < y.axes;) {
    const int64_t sx = i < x.axes ? x.axis[size_t(i)].step : -1, sy = j < y.axes ? y.axis[size_t(j)].step : -1;
    Term t{std::max(sx, sy), 0, 0};
    if (sx == t.step) t.high = x.axis[size_t(i++)].count - 1;
    if (sy == t.step) t.low = -(y.axis[size_t(j++)].count - 1);
    term[size_t(terms++)] = t;
  }
  // what the terms from k on can add
  std::array<int64_t, 2 * Runs::kMaxAxes + 2> least, most;
  least[size_t(terms)] = most[size_t(terms)] = 0;
  for (int k = terms - 1; k >= 0; --k) {
    least[size_t(k)] = least[size_t(k + 1)] + term[size_t(k)].step * term[size_t(k)].low;
    most[size_t(k)] = most[size_t(k + 1)] + term[size_t(k)].step * term[size_t(k)].high;
  }
  int budget = 4096;
  auto reach = [&](auto&& self, int k, int64_t from, int64_t to) -> bool {  // can the terms from k on fall into [from, to]?
    if (most[size_t(k)] < from || least[size_t(k)] > to) return false;
    if (k == terms) return true;
    const Term& t = term[size_t(k)];
    if (t.step == 0) return self(self, k + 1, from, to);
    auto floor_div = [](int64_t n, int64_t d) { return n >= 0 ? n / d : -((-n + d - 1) / d); };
    const int64_t low = std::max(t.low, floor_div(from - most[size_t(k + 1)] + t.step - 1, t.step));
    const int64_t high = std::min(t.high, floor_div(to - least[size_t(k + 1)], t.step));
    for (int64_t c = low; c <= high; ++c) {
      if (--budget < 0) return true;
      if (self(self, k + 1, from - c * t.step, to - c * t.step)) return true;
    }
    return false;
  };
  const int64_t apart = x.first - y.first;
  return reach(reach, 0, -(x.length - 1) - apart, y.length - 1 - apart);
}

// True where every element of the one is the element of the same index of the other.
inline bool same_place(const at::Tensor& a, const at::Tensor& b) {
  if (a.const_data_ptr() != b.const_data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// True where no two elements share memory: each axis steps over all that the smaller ones cover.
inline bool dense_apart(const at::Tensor& t) {
  const Runs r(t);
  if (r.empty) return true;
  if (!r.known) return false;
  int64_t covered = r.length;
  for (int i = r.axes - 1; i >= 0; --i) {
    const Runs::Axis& a = r.axis[size_t(i)];
    if (a.step < covered) return false;
    covered += a.step * (a.count - 1);
  }
  return true;
}

// An output of the caller's: no element twice, apart from what other parts of the call read, and apart from its own
// input or exactly that.
inline void check_place(const char* name, const at::Tensor& out, const char* own_name, const at::Tensor* own,
                        std::initializer_list<std::pair<const char*, const at::Tensor*>> others) {
  TORCH_CHECK(dense_apart(out), name, ": elements share memory");
  TORCH_CHECK(own == nullptr || same_place(out, *own) || !may_overlap(out, *own), name, " overlaps ", own_name,
              " without being it");
  for (const auto& [other, t] : others)
    TORCH_CHECK(t == nullptr || !may_overlap(out, *t), name, " overlaps ", other);
}

}  // namespace b200attn_torch
