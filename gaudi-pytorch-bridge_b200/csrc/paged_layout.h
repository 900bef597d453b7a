// Whether the slots of a paged cache lie apart in memory.  Plain C++: the C ABI and the torch extension both ask before they let
// a kernel write.
#pragma once

#include <cstdint>

namespace b200q {

// A cache [pages][slots][heads] of `dim` contiguous elements each, strides in elements; everything below is in bytes.
class CacheLayout {
 public:
  CacheLayout(const void* base, int64_t elt, int64_t dim, const int64_t (&sizes)[3], const int64_t (&strides)[3])
      : at_(reinterpret_cast<intptr_t>(base)) {
    extent_[0] = dim * elt;
    for (int i = 0; i < 3; ++i) {
      if (sizes[i] == 0) empty_ = true;
      if (sizes[i] <= 1) continue;  // (a stride that no index uses)
      int64_t step = strides[i] * elt;
      if (step < 0) {
        at_ += (sizes[i] - 1) * step;
        step = -step;
      }
      int j = levels_++;
      for (; j > 0 && stride_[j - 1] > step; --j) {
        stride_[j] = stride_[j - 1];
        size_[j] = size_[j - 1];
      }
      stride_[j] = step;
      size_[j] = sizes[i];
    }
    for (int i = 0; i < levels_; ++i) extent_[i + 1] = extent_[i] + (size_[i] - 1) * stride_[i];
  }

  // Each stride steps over all that lies inside it.
  bool apart() const {
    if (empty_) return true;
    for (int i = 0; i < levels_; ++i)
      if (stride_[i] < extent_[i]) return false;
    return true;
  }
  // For two that are apart in themselves: no byte belongs to both.  Exact where their strides are the same from the outermost one
  // on, as far in as their memory meets (two caches in one allocation); else such memory counts as shared.
  bool apart_from(const CacheLayout& other) const { return empty_ || other.empty_ || apart_from(other, levels_, other.levels_, other.at_ - at_); }

 private:
  // of the blocks of `mine` and `theirs` levels, theirs `delta` bytes behind mine
  bool apart_from(const CacheLayout& other, int mine, int theirs, int64_t delta) const {
    if (delta >= extent_[mine] || -delta >= other.extent_[theirs]) return true;
    if (mine == 0 || theirs == 0 || stride_[mine - 1] != other.stride_[theirs - 1]) return false;
    // blocks whose numbers differ by d are delta + d * step apart; the step is longer than a block, so that only the nearest can meet
    const int64_t step = stride_[mine - 1], nearest = -delta / step;
    for (int64_t d = nearest - 1; d <= nearest + 1; ++d)
      if (d > -size_[mine - 1] && d < other.size_[theirs - 1] && !apart_from(other, mine - 1, theirs - 1, delta + d * step)) return false;
    return true;
  }

  intptr_t at_;
  int64_t size_[3], stride_[3], extent_[4];
  int levels_ = 0;
  bool empty_ = false;
};

}  // namespace b200q
