// nq8_overlap.h -- whether the rows of two states share memory.
#pragma once

#include <stdint.h>

namespace nq {

// `rows` rows of `bytes` bytes, `stride` apart.
struct RowSpan {
  const void *ptr;
  int64_t bytes, stride;
};
// States whose rows interleave (columns of one tensor) do not overlap; of
// different strides they count as overlapping where their ranges do.
inline bool overlap(const RowSpan &a, const RowSpan &b, int64_t rows) {
  const int64_t pa = reinterpret_cast<intptr_t>(a.ptr), pb = reinterpret_cast<intptr_t>(b.ptr);
  if (pa + (rows - 1) * a.stride + a.bytes <= pb || pb + (rows - 1) * b.stride + b.bytes <= pa) return false;
  if (rows == 1 || a.stride != b.stride) return true;
  const int64_t d = ((pb - pa) % a.stride + a.stride) % a.stride;  // from a row of a to the next of b
  return d < a.bytes || d + b.bytes > a.stride;
}
// Whether a reordering of n states would write what it also reads or writes
// for another state; dst may be src with the same stride.
inline bool reorder_overlaps(const void *const *src, void *const *dst, const int64_t *bytes, const int64_t *src_stride,
                             const int64_t *dst_stride, int n, int64_t rows) {
  for (int i = 0; i < n; ++i) {
    const RowSpan to{dst[i], bytes[i], dst_stride[i]};
    for (int j = 0; j < n; ++j) {
      const bool in_place = i == j && src[i] == dst[i] && (rows == 1 || src_stride[i] == dst_stride[i]);
      if (!in_place && overlap(to, RowSpan{src[j], bytes[j], src_stride[j]}, rows)) return true;
      if (j < i && overlap(to, RowSpan{dst[j], bytes[j], dst_stride[j]}, rows)) return true;
    }
  }
  return false;
}

}  // namespace nq
