// Index arithmetic of the norm's row kernels, apart from them so that the host
// can enumerate it.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define I8_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define I8_HOST_DEVICE inline
#endif

namespace i8moe {

// Rows whose width no pack divides (kShift in the kernels): where every tensor
// starts on 16 bytes and its stride leaves the same remainder as the width, row
// r begins shift_of(r, k) elements behind a 16-byte boundary in all of them, so
// that packs counted from that boundary are aligned everywhere; the first and
// the last one reach over the row's ends.  Only the weight is off by the shift.
// 4096 x 2047 bf16 with a residual: 23 us instead of 31 element by element,
// with its gradients 55 instead of 74.
template <int kVec>
I8_HOST_DEVICE int shift_of(int64_t r, int k) {
  return static_cast<int>((static_cast<uint32_t>(r) * static_cast<uint32_t>(k)) % kVec);
}

// Columns that the threads of a row have to cover.
template <int kVec, bool kShift>
constexpr int covered(int k) {
  return k + (kShift ? kVec - 1 : 0);
}

// A CTA of the forward kernel: x threads for each of y rows, kPer packs a
// thread.  Several rows share a CTA where a row takes less than a warp, and
// those of the last CTA may lie past the tensor's end.
struct RowBlock {
  int x, y;
};
template <int kVec, int kPer, bool kShift>
I8_HOST_DEVICE RowBlock row_block(int k) {
  const int need = (covered<kVec, kShift>(k) + kVec * kPer - 1) / (kVec * kPer);
  int x = 1;
  while (x < 32 && x < need) x *= 2;
  if (need > 32) x = (need + 31) / 32 * 32;
  return {x, x <= 32 ? 128 / x : 1};
}

// What a thread of row r covers: elements first + p * stride + [0, kVec) as far
// as they lie in [0, k).  Rows past the last have no columns and no shift: with
// one, their first thread would stand before the row and find a column there.
struct RowPart {
  int first, k;
};
template <int kVec, bool kShift>
I8_HOST_DEVICE RowPart row_part(int64_t r, int64_t rows, int k, int tid) {
  if (r >= rows) return {tid * kVec, 0};
  return {tid * kVec - (kShift ? shift_of<kVec>(r, k) : 0), k};
}

// The element of a row of k >= 1 that is read in place of element i where that
// lies outside.
I8_HOST_DEVICE int nearest_element(int i, int k) {
  const int j = i < 0 ? 0 : i;
  return j < k ? j : k - 1;
}

}  // namespace i8moe
