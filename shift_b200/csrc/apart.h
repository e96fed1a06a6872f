// Whether two matrices (inner stride 1, rows that do not overlap) share a byte.
#pragma once
#include <torch/extension.h>

namespace sb {

inline bool share_memory(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  struct Span {
    int64_t begin, end, row, step;   // bytes
  };
  auto span = [](const at::Tensor& t) {
    const int64_t size = t.element_size(), row = t.size(1) * size, step = t.size(0) > 1 ? t.stride(0) * size : row;
    const int64_t begin = reinterpret_cast<intptr_t>(t.data_ptr());
    return Span{begin, begin + (t.size(0) - 1) * step + row, row, step};
  };
  const Span a = span(x), b = span(y);
  if (a.end <= b.begin || b.end <= a.begin) return false;
  if (a.step != b.step) return true;                        // or at least not shown to lie apart
  const int64_t shift = ((b.begin - a.begin) % a.step + a.step) % a.step;      // columns of one buffer, side by side?
  return !(shift >= a.row && shift + b.row <= a.step);
}

}  // namespace sb
