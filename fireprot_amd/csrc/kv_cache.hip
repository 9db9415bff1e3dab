// The paged key-value cache (fpx_cache_write, fpx_cache_read): rows of keys
// and values put at their slots, as they are or in 8 bits with a scale per
// row (in 4 bits: of 32 channels), and read back (cache_rows.hpp has the formats).
//
// Both kernels only move rows.  head_dim / 8 threads take a row, 8 channels
// each (16 bytes of BF16), so the row's maximum is a reduction of at most 32
// neighbouring lanes with no LDS; kRows rows of k and of v are in flight per
// thread.  Memory bounds the large ones: 64 098 tokens of 8 heads of 128 read
// back from FP8 as BF16, 403 MB, take 64 us, 6.3 TB/s, past the 5.3 of a plain
// copy, as most of it is writes.  7685 tokens of 16 heads of 64, FP16 and INT8,
// are written in 13 us and read back in 12, of which 3 to 4 are a launch.
#include "cache_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

constexpr int kCacheThreads = 256;

// tokens x heads rows of S into a cache of C.  kVec: the source rows are
// 16-byte aligned.
template <typename S, typename C, int kDim, bool kVec, bool kStream>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheArgs a) {
  constexpr int kGroup = kDim / 8;                  // threads of a row
  constexpr int kPass = kCacheThreads / kGroup;     // rows of a pass
  constexpr int kRows = 2;
  const int c = (threadIdx.x & (kGroup - 1)) * 8;
  const int64_t rows = a.tokens * a.heads;
  for (int64_t base = (int64_t)blockIdx.x * kPass * kRows + threadIdx.x / kGroup; base < rows;
       base += (int64_t)gridDim.x * kPass * kRows) {
    Eight<S> x[kRows][2];
    int64_t at[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = base + r * kPass;
      at[r] = kSlotNone;
      if (row >= rows) continue;
      const uint32_t t = (uint32_t)row / (uint32_t)a.heads;
      const int h = (int)((uint32_t)row - t * (uint32_t)a.heads);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const S* src = static_cast<const S*>(a.rows[w]) + t * a.stride_t[w] + h * a.stride_h[w] + c;
        if constexpr (kVec)
          x[r][w].template load<kStream>(src);
        else
          x[r][w].load_each(src);
      }
      at[r] = cache_row(a.slots[t], h, a.pages, a.heads, a.page_shift);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      // the row's threads share its slot, so a reduction below runs in all of
      // them or in none
      if (at[r] < 0) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if constexpr (kCoded<C>) {
          float v[1][8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[0][i] = x[r][w].value(i);
          put_codes<C, kDim, 1>(v, a.cache[w], a.scale[w], at[r], c);
        } else {
          Eight<C> y;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (__is_same(S, C))
              y.x[i] = x[r][w].x[i];
            else
              y.set(i, x[r][w].value(i));
          }
          y.store(held_at<C, kDim>(a.cache[w], at[r], c));
        }
      }
    }
  }
}

// Spans of eight channels of a row that a thread reads, half a row apart: of 4-bit rows
// two, so that what leads to a row serves as many bytes as in 8 bits.  And tokens of one
// head that are read one after another, before the next head's: 4-bit rows are parts of a
// line of the cache, and so are their scales, of which the next slot's row has the rest.
// 64098 tokens of 8 heads of 128 to BF16, 332 MB: 78 us with one span, 84 with two, 70 with
// tokens in runs of 16, 63 with one row of each tensor in flight in a thread and not four.
template <typename C>
constexpr int kReadSpans = __is_same(C, Fp4) ? 2 : 1;
template <typename C>
constexpr int kReadTokens = __is_same(C, Fp4) ? 16 : 1;
template <typename C>
constexpr int kReadRows = __is_same(C, Fp4) ? 1 : 4;

// The rows of `slots` back as S: zeros where there is no slot, NaN for a slot
// past the cache's end.
template <typename S, typename C, int kDim, bool kVec, bool kStream>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(CacheArgs a) {
  constexpr int kSpans = kReadSpans<C>;
  constexpr int kGroup = kDim / 8 / kSpans;
  constexpr int kPass = kCacheThreads / kGroup;
  constexpr int kRows = kReadRows<C>;
  constexpr uint32_t kRun = kReadTokens<C>;
  const int c = (threadIdx.x & (kGroup - 1)) * 8;
  const int64_t rows = round_up(a.tokens, kRun) * a.heads;
  for (int64_t base = (int64_t)blockIdx.x * kPass * kRows + threadIdx.x / kGroup; base < rows;
       base += (int64_t)gridDim.x * kPass * kRows) {
    uint32_t t[kRows];
    int h[kRows];
    int64_t at[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = base + r * kPass;
      at[r] = kSlotNone;
      if (row >= rows) continue;
      const uint32_t run = (uint32_t)row / kRun, first = run / (uint32_t)a.heads;
      t[r] = first * kRun + (uint32_t)row % kRun;
      h[r] = (int)(run - first * (uint32_t)a.heads);
      // (a look at t where no run passes the end would part the loads of the slots)
      if (kRun == 1 || t[r] < a.tokens)
        at[r] = cache_row(a.slots[t[r]], h[r], a.pages, a.heads, a.page_shift);
    }
    Held<C> held[kRows][2][kSpans];
    float scale[kRows][2][kSpans];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (at[r] < 0) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int s = 0; s < kSpans; ++s) {
          const int d = c + s * (kDim / kSpans);
          held[r][w][s].template load<kStream>(
              held_at<C, kDim>(static_cast<const void*>(a.cache[w]), at[r], d));
          if constexpr (kCoded<C>) scale[r][w][s] = scale_at<C, kDim>(a.scale[w], at[r], d);
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (base + r * kPass >= rows || (kRun > 1 && t[r] >= a.tokens)) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int s = 0; s < kSpans; ++s) {
          Eight<S> y;
          const float fill = at[r] == kSlotOutside ? __builtin_nanf("") : 0.0f;
          if constexpr (kCoded<C>) {
            float v[8];
            decode<C>(held[r][w][s].x, scale[r][w][s], v);
#pragma unroll
            for (int i = 0; i < 8; ++i) y.set(i, at[r] < 0 ? fill : v[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if constexpr (__is_same(S, C))
                y.x[i] = at[r] < 0 ? (S)fill : held[r][w][s].x[i];
              else
                y.set(i, at[r] < 0 ? fill : held[r][w][s].value(i));
            }
          }
          S* dst = const_cast<S*>(static_cast<const S*>(a.rows[w])) + t[r] * a.stride_t[w] +
                   h[r] * a.stride_h[w] + c + s * (kDim / kSpans);
          if constexpr (kVec)
            y.store(dst);
          else
            y.store_each(dst);
        }
    }
  }
}

template <typename S, typename C, int kDim>
hipError_t launch_dim(const CacheArgs& a, bool read, hipStream_t stream) {
  constexpr int kPass = kCacheThreads / (kDim / 8);
  const int64_t per = kPass * (read ? kReadRows<C> * kReadSpans<C> : 2);
  const int64_t rows = (read ? round_up(a.tokens, kReadTokens<C>) : a.tokens) * a.heads;
  const int64_t blocks = (rows + per - 1) / per;
  // (the kernels walk on in strides of the grid)
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
  uint64_t bytes = 0;
  for (int w = 0; w < 2; ++w)
    bytes |= reinterpret_cast<uintptr_t>(a.rows[w]) |
             (uint64_t)(a.stride_t[w] | a.stride_h[w]) * sizeof(S);
  const bool vec = bytes % 16 == 0;
  // what is read and no cache holds anyway is streamed past them
  const int64_t row = read ? held_bytes<C>(kDim) : kDim * (int64_t)sizeof(S);
  const bool once = 2 * a.tokens * a.heads * row >= kStreamBytes;
  if (read) {
    if (!vec)
      cache_read_kernel<S, C, kDim, false, false><<<grid, kCacheThreads, 0, stream>>>(a);
    else if (once)
      cache_read_kernel<S, C, kDim, true, true><<<grid, kCacheThreads, 0, stream>>>(a);
    else
      cache_read_kernel<S, C, kDim, true, false><<<grid, kCacheThreads, 0, stream>>>(a);
  } else {
    if (!vec)
      cache_write_kernel<S, C, kDim, false, false><<<grid, kCacheThreads, 0, stream>>>(a);
    else if (once)
      cache_write_kernel<S, C, kDim, true, true><<<grid, kCacheThreads, 0, stream>>>(a);
    else
      cache_write_kernel<S, C, kDim, true, false><<<grid, kCacheThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename S, typename C>
hipError_t launch_cache_type(const CacheArgs& a, bool read, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: return launch_dim<S, C, 32>(a, read, stream);
    case 64: return launch_dim<S, C, 64>(a, read, stream);
    case 128: return launch_dim<S, C, 128>(a, read, stream);
    default: return launch_dim<S, C, 256>(a, read, stream);
  }
}

template <typename S>
hipError_t launch_source(const CacheArgs& a, bool read, hipStream_t stream) {
  switch (a.cache_dtype) {
    case 0: return launch_cache_type<S, float>(a, read, stream);
    case 1: return launch_cache_type<S, __bf16>(a, read, stream);
    case 2: return launch_cache_type<S, _Float16>(a, read, stream);
    case 3: return launch_cache_type<S, Fp8>(a, read, stream);
    case 4: return launch_cache_type<S, Int8>(a, read, stream);
    default: return launch_cache_type<S, Fp4>(a, read, stream);
  }
}

}  // namespace

hipError_t launch_cache(const CacheArgs& a, bool read, hipStream_t stream) {
  switch (a.row_dtype) {
    case 0: return launch_source<float>(a, read, stream);
    case 1: return launch_source<__bf16>(a, read, stream);
    default: return launch_source<_Float16>(a, read, stream);
  }
}

}  // namespace fpx
