// Whether two operands share memory: blocks of a kernel that writes one while others still
// read the other would depend on which comes first.
#pragma once

#include <torch/extension.h>

#include <algorithm>

// An operand that a kernel has written: what autograd saved of it is not it any more
inline void written(const torch::Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// a, b: rows of adjacent numbers (N, W) that may lie apart, or contiguous tensors.  Exact:
// rows of one between those of the other, columns beside its columns, do not overlap.
inline bool rows_overlap(const torch::Tensor& a, const torch::Tensor& b) {
  struct Rows {
    long at, n, pitch, width;               // in bytes
    explicit Rows(const torch::Tensor& t)
        : at((long)t.data_ptr()), n(1), pitch(0), width(t.numel() * t.element_size()) {
      if (t.dim() != 2 || t.numel() == 0 || t.size(0) == 1) return;
      n = t.size(0), pitch = t.stride(0) * t.element_size();
      width = t.size(1) * t.element_size();
    }
    long end() const { return at + (n - 1) * pitch + width; }
  };
  const Rows p(a), q(b);
  if (p.width == 0 || q.width == 0 || p.end() <= q.at || q.end() <= p.at) return false;
  if (p.pitch == 0 && q.pitch == 0) return true;
  const Rows& one = q.pitch == 0 ? q : p;   // whose rows are gone through
  const Rows& other = q.pitch == 0 ? p : q;
  // Row i of one lies on those rows j of other that have
  //   d - other.width < j * pitch < d + one.width,   d = one.at + i * one.pitch - other.at;
  // of rows equally far apart j - i decides, which is any number of a range
  const bool same = one.pitch == other.pitch;
  const long least = same ? -(one.n - 1) : 0;
  auto floor_div = [](long x, long y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  for (long i = 0; i < (same ? 1 : one.n); ++i) {
    const long d = one.at + i * one.pitch - other.at;
    const long low = floor_div(d - other.width, other.pitch) + 1;
    const long high = -floor_div(-(d + one.width), other.pitch) - 1;
    if (std::max(low, least) <= std::min(high, other.n - 1)) return true;
  }
  return false;
}
