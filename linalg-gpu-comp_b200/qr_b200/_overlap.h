// Whether two strided tensors share memory, exactly, for the checks of what a call may write into.
//
// A tensor is a set of equally long dense runs of bytes, as few as its strides allow.  Ranges that lie apart,
// or runs that alternate at one pitch (column slices of one buffer), are told from sizes and strides; only
// what is left walks over the runs of both.
#pragma once

#include <ATen/ATen.h>

#include <algorithm>
#include <optional>
#include <vector>

namespace qrb_entry {

class Runs {
 public:
  explicit Runs(const at::Tensor& t) : base_(reinterpret_cast<intptr_t>(t.const_data_ptr())), length_(t.element_size()) {
    empty_ = t.numel() == 0;
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) <= 1) continue;
      if (t.stride(i) == 0) repeated_ = true;
      else dims_.push_back({t.size(i), t.stride(i) * static_cast<int64_t>(t.element_size())});
    }
    std::sort(dims_.begin(), dims_.end(), [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    // dimensions that only lengthen the run, then those that only continue the one before
    size_t inner = 0;
    while (inner < dims_.size() && dims_[inner].stride == length_) length_ *= dims_[inner++].size;
    dims_.erase(dims_.begin(), dims_.begin() + inner);
    std::vector<Dim> merged;
    for (const Dim& d : dims_) {
      if (!merged.empty() && d.stride == merged.back().size * merged.back().stride) merged.back().size *= d.size;
      else merged.push_back(d);
    }
    dims_ = std::move(merged);
    extent_ = length_;
    for (const Dim& d : dims_) extent_ += (d.size - 1) * d.stride;
  }

  bool meets(const Runs& o) const {
    if (empty_ || o.empty_ || base_ + extent_ <= o.base_ || o.base_ + o.extent_ <= base_) return false;
    if (dims_.empty() && o.dims_.empty()) return true;
    if (dims_.size() <= 1 && o.dims_.size() <= 1) {   // one pitch, or a single run beside rows of one
      const int64_t pitch = dims_.empty() ? o.dims_[0].stride : dims_[0].stride;
      const bool same = dims_.empty() || o.dims_.empty() || o.dims_[0].stride == pitch;
      const int64_t at = ((o.base_ - base_) % pitch + pitch) % pitch;
      if (same && at >= length_ && at + o.length_ <= pitch) return false;
    }
    const std::vector<intptr_t> a = starts(), b = o.starts();
    for (size_t i = 0, j = 0; i < a.size() && j < b.size();) {
      if (a[i] + length_ <= b[j]) ++i;
      else if (b[j] + o.length_ <= a[i]) ++j;
      else return true;
    }
    return false;
  }

  // Whether some byte belongs to two elements.
  bool meets_itself() const {
    if (empty_) return false;
    if (repeated_) return true;
    int64_t reach = length_;   // every dimension steps over all that the smaller ones cover
    bool nested = true;
    for (const Dim& d : dims_) {
      nested &= d.stride >= reach;
      reach += (d.size - 1) * d.stride;
    }
    if (nested) return false;
    const std::vector<intptr_t> a = starts();
    for (size_t i = 1; i < a.size(); ++i)
      if (a[i] < a[i - 1] + length_) return true;
    return false;
  }

 private:
  struct Dim {
    int64_t size, stride;   // stride in bytes
  };
  intptr_t base_;
  int64_t length_, extent_;
  bool empty_, repeated_ = false;   // repeated_: a dimension without a stride
  std::vector<Dim> dims_;   // beyond the run, smallest stride first

  std::vector<intptr_t> starts() const {
    std::vector<intptr_t> all{base_};
    for (const Dim& d : dims_) {
      const size_t n = all.size();
      for (int64_t i = 1; i < d.size; ++i)
        for (size_t j = 0; j < n; ++j) all.push_back(all[j] + i * d.stride);
    }
    std::sort(all.begin(), all.end());
    return all;
  }
};

// A tensor and the bytes from its first element to behind its last, taken once for several comparisons.
struct Range {
  const at::Tensor* t = nullptr;
  intptr_t lo = 0, hi = 0;
  Range(const at::Tensor& x) : t(&x) {
    const auto sizes = x.sizes(), strides = x.strides();
    int64_t n = 1;
    for (size_t i = 0; i < sizes.size(); ++i) {
      if (sizes[i] == 0) return;
      n += (sizes[i] - 1) * strides[i];
    }
    lo = reinterpret_cast<intptr_t>(x.const_data_ptr());
    hi = lo + n * static_cast<int64_t>(x.element_size());
  }
  Range(const std::optional<at::Tensor>& x) {
    if (x.has_value()) *this = Range(*x);
  }
};

inline bool overlap(const Range& a, const Range& b) {
  return a.lo < b.hi && b.lo < a.hi && Runs(*a.t).meets(Runs(*b.t));
}

// Both name the same elements at the same places.
inline bool same_place(const at::Tensor& a, const at::Tensor& b) {
  if (a.const_data_ptr() != b.const_data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

}  // namespace qrb_entry
