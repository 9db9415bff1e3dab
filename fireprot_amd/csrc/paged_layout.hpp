// Index rules of the paged key-value cache, shared by its kernels and by the
// host: plain C++ with no device types, so they are tested on the CPU as they
// stand.
//
// A cache holds `pages` pages of 2^page_shift slots.  k and v each are
// [pages][heads][slots of a page][head_dim], the scales of an 8-bit cache
// [pages][heads][slots of a page]: one head's keys of a page are contiguous,
// which is what an attention work-group reads.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define FPX_HD __host__ __device__ __forceinline__
#else
#define FPX_HD inline
#endif

namespace fpx {

constexpr int64_t kSlotNone = -1;     // a negative slot: no token
constexpr int64_t kSlotOutside = -2;  // a slot past the cache's end

// Row (of head_dim channels, and of the scales) of a slot and head, or
// kSlotNone / kSlotOutside.
FPX_HD int64_t cache_row(int64_t slot, int head, int64_t pages, int heads, int page_shift) {
  if (slot < 0) return kSlotNone;
  const int64_t page = slot >> page_shift;
  if (page >= pages) return kSlotOutside;
  return ((page * heads + head) << page_shift) + (slot & ((int64_t(1) << page_shift) - 1));
}

// Keys [first, end) that a sequence of `length` tokens attends to, or invalid
// where the length does not fit the call (negative, or above max_length).
struct KeyRange {
  int first, end, valid;
};

FPX_HD KeyRange key_range(int length, int max_length, int window) {
  if (length < 0 || length > max_length) return {0, 0, 0};
  return {window > 0 && length > window ? length - window : 0, length, 1};
}

// The work on a range is counted in units of `unit` keys, the first begun at a
// multiple of 32; a sequence without keys is one unit (somebody writes its
// rows).
constexpr int kKeyAlign = 32;

FPX_HD int first_key(const KeyRange& r) { return r.first & ~(kKeyAlign - 1); }

FPX_HD int unit_count(const KeyRange& r, int unit) {
  return r.end <= r.first ? 1 : (r.end - first_key(r) - 1) / unit + 1;
}

// Most units a sequence of this call can have: the longest range, begun at the
// last key of an aligned group (a window begins anywhere in one).
FPX_HD int64_t unit_limit(int64_t max_length, int64_t window, int unit) {
  int64_t span = max_length;
  if (window > 0 && window + kKeyAlign - 1 < span) span = window + kKeyAlign - 1;
  return span < 1 ? 1 : (span - 1) / unit + 1;
}

// `total` units in equal shares for `groups` work-groups, one more for the first
// few: the first unit of a share, and the share that a unit is in.
struct Shares {
  int size, larger;  // units of a share; the first `larger` shares have one more
};

FPX_HD Shares make_shares(int total, int groups) { return {total / groups, total % groups}; }

FPX_HD int share_start(const Shares& s, int group) {
  return group * s.size + (group < s.larger ? group : s.larger);
}

FPX_HD int share_of(const Shares& s, int unit) {
  const int wide = s.larger * (s.size + 1);
  return unit < wide ? unit / (s.size + 1) : s.larger + (unit - wide) / s.size;
}

// Work-groups of the attention's kernel that a CU's registers hold at once, at least:
// a work-group has a wave on each SIMD.  `split`: queries that enter the products as
// several terms (FP32 and FP16 over an 8-bit cache).
FPX_HD int resident_groups(bool split, int head_dim, int query_tiles) {
  return head_dim > 128 || query_tiles > 1 || (split && head_dim == 128) ? 2 : 3;
}

// Entry of the block table that serves a group of keys from `key` on: that of
// the nearest key of the range, so that a group wholly outside it (its keys
// are masked) names no page the sequence does not hold.
FPX_HD int table_entry(int key, const KeyRange& r, int page_shift) {
  const int k = key < r.first ? r.first : key >= r.end ? r.end - 1 : key;
  return k >> page_shift;
}

// Whether a block-table entry names a page of the cache.
FPX_HD bool page_valid(int page, int64_t pages) {
  return page >= 0 && (int64_t)page < pages;
}

}  // namespace fpx
