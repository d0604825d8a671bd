// Host checks of which tensors may share memory.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace ferret {

// The bytes that a tensor spans; none where there is no tensor.
struct Range {
  const void* at;
  uint64_t bytes;
};

inline bool overlap(const Range& a, const Range& b) {
  const uint64_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at != nullptr && b.at != nullptr && x < y + b.bytes && y < x + a.bytes;
}

// A tensor that is written overlaps another that is written, or one that is read.
inline bool clash(std::initializer_list<Range> written, std::initializer_list<Range> read) {
  for (auto w = written.begin(); w != written.end(); ++w) {
    for (auto other = written.begin(); other != w; ++other)
      if (overlap(*w, *other)) return true;
    for (const Range& r : read)
      if (overlap(*w, r)) return true;
  }
  return false;
}

// bf16 [rows, heads, width] with these strides in elements.
inline Range bf16_range(const void* at, uint64_t rows, uint64_t row_stride, uint64_t heads, uint64_t head_stride,
                        uint64_t width) {
  return {at, 2 * ((rows - 1) * row_stride + (heads - 1) * head_stride + width)};
}

// Whether a packed output at `out` stands on exactly these rows: in place.
inline bool in_place(const void* out, const void* in, long long rows, long long row_stride, long long heads,
                     long long head_stride, long long width) {
  return out == in && (rows == 1 || row_stride == heads * width) && (heads == 1 || head_stride == width);
}

}  // namespace ferret
