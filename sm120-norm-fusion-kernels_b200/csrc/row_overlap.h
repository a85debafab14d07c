// row_overlap.h -- whether two sets of equally spaced rows share a byte. Views of
// one buffer (the columns of a projection's output) interleave without sharing
// any, so spans alone do not decide it.
#pragma once

#include <cstdint>

namespace sm120n {

// `count` rows of `width` bytes, `stride` >= width bytes apart.
struct RowSet {
  const void* data;
  int64_t count;
  int64_t stride;
  int64_t width;
};

inline RowSet row_set(const void* data, int64_t count, int64_t stride, int64_t width, int64_t elem) {
  return RowSet{data, count, stride * elem, width * elem};
}

inline bool rows_overlap(const RowSet& a, const RowSet& b) {
  using Wide = __int128;
  if (a.data == nullptr || b.data == nullptr || a.count < 1 || b.count < 1 || a.width < 1 ||
      b.width < 1) {
    return false;
  }
  const Wide apart = Wide{static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.data) -
                                               reinterpret_cast<uintptr_t>(a.data))};
  const Wide step_a = a.count > 1 ? a.stride : b.stride;  // one row has no stride of its own
  const Wide step_b = b.count > 1 ? b.stride : step_a;
  const Wide end_a = (a.count - 1) * step_a + a.width;
  const Wide end_b = apart + (b.count - 1) * step_b + b.width;
  if (end_a <= apart || end_b <= 0) return false;
  if (a.count == 1 && b.count == 1) return true;
  // first multiple `k` of `step` with apart + k * step > -b.width, at least `least`
  auto first = [&](Wide from, Wide step, Wide least) {
    const Wide room = -from - b.width;
    Wide k = room / step;
    if (k * step > room) --k;  // rounded down
    return k + 1 < least ? least : k + 1;
  };
  if (step_a == step_b) {  // row j of b lies k = j - i strides behind row i of a
    const Wide k = first(apart, step_a, -(Wide{a.count} - 1));
    return k <= b.count - 1 && apart + k * step_a < a.width;
  }
  for (int64_t i = 0; i < a.count; ++i) {
    const Wide from = apart - i * step_a;
    const Wide j = first(from, step_b, 0);
    if (j <= b.count - 1 && from + j * step_b < a.width) return true;
  }
  return false;
}

}  // namespace sm120n
