// Whether strided views share memory: what an operator writes must not overlap what it reads or writes besides.
#pragma once

#include <ATen/ATen.h>

#include <cstdint>
#include <optional>

namespace pla_ops {

// A view in bytes: equally long runs of contiguous bytes, repeated along axes of falling stride.
struct Runs {
  static constexpr int MOST = 4;
  int64_t at = 0, run = 0, size[MOST], stride[MOST];      // of the first `axes`
  int axes = 0;
  bool empty = false;

  Runs() = default;
  explicit Runs(const at::Tensor& t) {
    const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
    const int64_t bytes = static_cast<int64_t>(t.element_size());
    at = static_cast<int64_t>(reinterpret_cast<intptr_t>(t.const_data_ptr()));
    empty = t.numel() == 0;
    run = bytes;
    for (size_t d = sizes.size(); d-- > 0;) add(sizes[d], strides[d] * bytes);
    fold();
  }
  // One more axis, kept in order of stride; views have few, and come innermost axis first.
  void add(int64_t n, int64_t step) {
    if (n <= 1) return;
    if (axes == MOST) TORCH_CHECK(false, "views of more than ", MOST, " axes are not supported");
    if (axes == 0 && step == run) {        // the usual innermost axis
      run *= n;
      return;
    }
    int i = axes++;
    for (; i > 0 && stride[i - 1] < step; --i) size[i] = size[i - 1], stride[i] = stride[i - 1];
    size[i] = n, stride[i] = step;
  }
  // Axes that continue the run become part of it.
  void fold() {
    while (axes > 0 && stride[axes - 1] == run) run *= size[--axes];
  }
  int64_t extent(int from = 0) const {
    int64_t n = run;
    for (int i = from; i < axes; ++i) n += (size[i] - 1) * stride[i];
    return n;
  }
  // Every axis steps over all that the later ones reach. Broadcast axes (stride 0) never do.
  bool separate() const {
    for (int i = 0; i < axes; ++i)
      if (!empty && stride[i] < extent(i + 1)) return false;
    return true;
  }
  bool same(const Runs& y) const {
    if (at != y.at || run != y.run || axes != y.axes) return false;
    for (int i = 0; i < axes; ++i)
      if (size[i] != y.size[i] || stride[i] != y.stride[i]) return false;
    return true;
  }
};

// True when a's axes from `i` on and b's from `j` on, b beginning `delta` bytes behind a, certainly share no byte: they end before
// one another, or step together and every step leaves the other's place free (halves of one cache, parts of one packed row).
inline bool apart(const Runs& a, int i, const Runs& b, int j, int64_t delta) {
  if (delta >= a.extent(i) || delta + b.extent(j) <= 0) return true;
  if (i == a.axes || j == b.axes || a.stride[i] != b.stride[j]) return false;
  const int64_t step = a.stride[i];
  if (step < a.extent(i + 1) || step < b.extent(j + 1)) return false;
  const int64_t rest = (delta % step + step) % step;
  return apart(a, i + 1, b, j + 1, rest) && apart(a, i + 1, b, j + 1, rest - step);
}
inline bool apart(const Runs& a, const Runs& b) { return a.empty || b.empty || apart(a, 0, b, 0, b.at - a.at); }

// What one call reads and writes, tensor by tensor (about 0.1 us for a call with caches).
class Arguments {
 public:
  // Each returns the argument's number, -1 for one that is not given.
  int read(const at::Tensor& t) { return add(Runs(t)); }
  int read(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined() ? read(*t) : -1; }
  // A tensor of the caller's that is written: its elements must not overlap each other, nor anything added so far. It may be argument
  // `in_place`, element for element, where every row is read before it is written.
  int write(const at::Tensor& t, const char* name, int in_place = -1) {
    const Runs mine(t);
    TORCH_CHECK(mine.separate(), name, " has elements that overlap (an expanded tensor?)");
    for (int i = 0; i < count_; ++i)
      TORCH_CHECK(apart(mine, seen_[i]) || (i == in_place && mine.same(seen_[i])), name, " overlaps another argument",
                  in_place >= 0 ? " (it may be its own input, element for element)" : "");
    return add(mine);
  }

 private:
  int add(const Runs& r) {
    TORCH_CHECK(count_ < MOST, "too many arguments");
    seen_[count_] = r;
    return count_++;
  }
  static constexpr int MOST = 12;
  Runs seen_[MOST];
  int count_ = 0;
};

}  // namespace pla_ops
