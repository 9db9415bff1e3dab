// Whether strided blocks of memory share a byte: plain C++ for the host, so that
// it is tested as it stands.
//
// A block is a base and up to four axes of (count, bytes between two of them, not
// negative) of whole elements.  Two blocks meet where
//   base_a + sum_i x_i s_i = base_b + sum_j y_j t_j,  0 <= x_i < n_i, 0 <= y_j < m_j
// has a solution; with m_j - 1 - y_j in place of y_j every term is positive, and the
// axes, longest stride first, are searched for the value that is left: in views of
// one tensor, whose strides contain each other, an axis has one or two candidates.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace fpx {

struct MemoryAxis {
  int64_t count, stride;
};

struct MemoryBlock {
  uintptr_t base = 0;
  bool empty = true;
  int axes = 0;
  MemoryAxis axis[5] = {};
  __int128 span = 0;  // bytes from the first to the last

  MemoryBlock() = default;
  template <typename... Axes>
  MemoryBlock(const void* p, int64_t element, Axes... a)
      : base(reinterpret_cast<uintptr_t>(p)), empty(p == nullptr) {
    // (a stride past every memory stays one)
    constexpr int64_t far = int64_t(1) << 58;
    for (const MemoryAxis x : {MemoryAxis{element, 1},
                               MemoryAxis{a.count, (a.stride < far ? a.stride : far) * element}...}) {
      if (x.count < 1) empty = true;
      if (x.count <= 1) continue;
      span += (__int128)(x.count - 1) * x.stride;
      axis[axes++] = x;
    }
  }
};

namespace overlap {

constexpr int kSteps = 20000;  // a search of more is given up: taken to overlap

// sum_i x_i stride_i = target with 0 <= x_i < count_i, axes from i on.
inline bool solve(const MemoryAxis* axis, const __int128* rest, int axes, int i, __int128 target,
                  int& steps) {
  if (target < 0 || target > rest[i]) return false;
  if (target == 0) return true;
  if (i == axes) return false;
  if (--steps < 0) return true;
  const __int128 s = axis[i].stride;
  const __int128 most = target / s;
  int64_t x = (int64_t)(most < axis[i].count - 1 ? most : axis[i].count - 1);
  for (; x >= 0 && target - x * s <= rest[i + 1]; --x)
    if (solve(axis, rest, axes, i + 1, target - x * s, steps)) return true;
  return false;
}

// The same for axes in any order, of counts of 1 and strides of 0 among them.
inline bool reachable(const MemoryAxis* given, int count, __int128 target) {
  MemoryAxis axis[10];
  int axes = 0;
  for (int i = 0; i < count; ++i) {
    if (given[i].count <= 1 || given[i].stride == 0) continue;
    int at = 0;
    while (at < axes && axis[at].stride > given[i].stride) ++at;
    if (at < axes && axis[at].stride == given[i].stride) {
      axis[at].count += given[i].count - 1;
      continue;
    }
    for (int j = axes++; j > at; --j) axis[j] = axis[j - 1];
    axis[at] = given[i];
  }
  __int128 rest[11];
  rest[axes] = 0;
  for (int i = axes - 1; i >= 0; --i)
    rest[i] = rest[i + 1] + (__int128)(axis[i].count - 1) * axis[i].stride;
  int steps = kSteps;
  return solve(axis, rest, axes, 0, target, steps);
}

}  // namespace overlap

// Whether a and b have a byte in common.
inline bool blocks_meet(const MemoryBlock& a, const MemoryBlock& b) {
  if (a.empty || b.empty) return false;
  const __int128 apart = (__int128)b.base - (__int128)a.base;
  if (apart > a.span || -apart > b.span) return false;
  MemoryAxis axis[10];
  int axes = 0;
  for (int i = 0; i < a.axes; ++i) axis[axes++] = a.axis[i];
  for (int i = 0; i < b.axes; ++i) axis[axes++] = b.axis[i];
  return overlap::reachable(axis, axes, apart + b.span);
}

// Whether two elements of a block, of different places, have a byte in common.
inline bool block_meets_itself(const MemoryBlock& a) {
  if (a.empty) return false;
  // (each axis steps over all that the shorter strides reach: the ordinary case)
  bool nested = true;
  for (int i = 0; i < a.axes && nested; ++i) {
    __int128 below = 0;
    for (int j = 0; j < a.axes; ++j)
      if (j != i && (a.axis[j].stride < a.axis[i].stride ||
                     (a.axis[j].stride == a.axis[i].stride && j < i)))
        below += (__int128)(a.axis[j].count - 1) * a.axis[j].stride;
    nested = a.axis[i].stride > below;
  }
  if (nested) return false;
  // a difference of places whose first axis, k, is at least one step apart, the axes
  // after it any number either way
  for (int k = 0; k < a.axes; ++k) {
    MemoryAxis axis[5];
    int axes = 0;
    __int128 target = -(__int128)a.axis[k].stride;
    axis[axes++] = {a.axis[k].count - 1, a.axis[k].stride};
    for (int i = k + 1; i < a.axes; ++i) {
      axis[axes++] = {2 * a.axis[i].count - 1, a.axis[i].stride};
      target += (__int128)(a.axis[i].count - 1) * a.axis[i].stride;
    }
    if (a.axis[k].stride == 0 || overlap::reachable(axis, axes, target)) return true;
  }
  return false;
}

}  // namespace fpx
