// Host side: whether two strided tensors share memory. at::assert_no_overlap says nothing about tensors that are not dense,
// and views into one fused buffer never are.
#pragma once
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <initializer_list>
#include <utility>

namespace br {

// The bytes of a tensor: runs of `width` at every sum of multiples (below `count`) of the steps, largest step first.
struct Footprint {
  struct Dim {
    int64_t count, step;
  };
  const char* base = nullptr;
  std::array<Dim, 4> dims{};
  int n = 0;
  int64_t width = 0;  // 0: no elements

  explicit Footprint(const torch::Tensor& t) : base(static_cast<const char*>(t.data_ptr())), width(t.element_size()) {
    TORCH_CHECK(t.dim() <= 4, "at most four dimensions");
    if (t.numel() == 0) {
      width = 0;
      return;
    }
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1) dims[n++] = {t.size(d), t.stride(d) * (int64_t)t.element_size()};
    std::sort(dims.begin(), dims.begin() + n, [](const Dim& a, const Dim& b) { return a.step > b.step; });
    while (n > 0 && dims[n - 1].step == width) width *= dims[--n].count;
  }
};

inline int64_t bytes_spanned(const Footprint::Dim* d, int n, int64_t width) {
  for (int i = 0; i < n; ++i) width += (d[i].count - 1) * d[i].step;
  return width;
}

// b starts delta bytes behind a. With the larger of the outer steps as a period, both are slots at multiples of it (a
// tensor without that step is one slot), and only the slots' distances at which their spans meet are looked into: one
// or two of them unless a tensor's rows overlap each other. More than 2^16 are taken as shared.
inline bool share(const Footprint::Dim* a, int na, int64_t wa, const Footprint::Dim* b, int nb, int64_t wb, int64_t delta) {
  const int64_t ea = bytes_spanned(a, na, wa), eb = bytes_spanned(b, nb, wb);
  if (delta >= ea || -delta >= eb) return false;
  if (na == 0 && nb == 0) return true;
  const int64_t step = std::max(na ? a[0].step : 0, nb ? b[0].step : 0);
  if (step == 0) return true;
  const bool pa = na && a[0].step == step, pb = nb && b[0].step == step;
  const int64_t ia = bytes_spanned(a + pa, na - pa, wa), ib = bytes_spanned(b + pb, nb - pb, wb);
  auto floor_div = [&](int64_t x) { return x >= 0 ? x / step : -((-x + step - 1) / step); };
  // distances m of the slots with -ib < delta + m step < ia
  const int64_t lo = std::max(floor_div(-ib - delta) + 1, pa ? 1 - a[0].count : 0);
  const int64_t hi = std::min(floor_div(ia - 1 - delta), pb ? b[0].count - 1 : 0);
  if (hi - lo >= 1 << 16) return true;
  for (int64_t m = lo; m <= hi; ++m)
    if (share(a + pa, na - pa, wa, b + pb, nb - pb, wb, delta + m * step)) return true;
  return false;
}

using Named = std::pair<const char*, const torch::Tensor*>;

// An output must not share memory with any of the others, nor its elements with each other.
inline void check_output(const char* what, Named out, std::initializer_list<Named> others) {
  const Footprint o(*out.second);
  if (o.width == 0) return;
  int64_t inner = o.width;
  for (int d = o.n - 1; d >= 0; --d) {
    TORCH_CHECK(o.dims[d].step >= inner, what, ": elements of ", out.first, " share memory");
    inner += (o.dims[d].count - 1) * o.dims[d].step;
  }
  for (const Named& other : others) {
    const Footprint x(*other.second);
    TORCH_CHECK(x.width == 0 || other.second->device() != out.second->device() ||
                    !share(o.dims.data(), o.n, o.width, x.dims.data(), x.n, x.width, x.base - o.base),
                what, ": ", out.first, " shares memory with ", other.first);
  }
}

}  // namespace br
