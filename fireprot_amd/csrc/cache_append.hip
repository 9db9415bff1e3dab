// New tokens' keys and values into the paged cache, the keys (and the queries, which
// go back to the caller) turned by their positions on the way (fpx_cache_append): in
// one pass what fpx_rotary, the look-up of slots in a block table and fpx_cache_write
// do in three and more launches with the turned keys written out in between.
//
//   q_out = rotate(q),  cache[slot] = format(rotate(k)), format(v)
//
// rotate as rotary.hip has it, in FP32; format as cache_rows.hpp has it, from the FP32
// values: a turned key is rounded once, into the cache's type.
//
// Memory bounds a prompt (each row is read once and written once), a launch's start a
// step.  A work-group takes `tt` tokens: their factors (cos, sin) go into LDS once and
// serve all heads, their slots are looked up meanwhile.  head_dim / 8 neighbouring lanes
// take a row, 8 channels each, so that a row's maximum needs no LDS; where the whole head
// is turned, half as many take two eights half a row apart, which are each other's pairs
// in the half layout.  Otherwise (a part turned) the other half of a pair is loaded a
// second time by the lane that needs it.
//
// 16384 tokens of 32 query and 8 cache heads of 128 BF16 channels into 4 bits, 354 MB:
// 67 to 70 us, 5.2 TB/s, a plain copy's rate (one eight to a lane, not streamed: 83).
// 1665 tokens of 16 and 16 heads of 64 FP16 channels into INT8: 8.6 us.  64 tokens of 32
// and 8 heads into BF16: 4.6 us, of which a launch is 3 to 4.
#include "cache_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"
#include "rotary.hpp"

namespace fpx {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendBatch = 3;            // vectors in flight per thread, about
constexpr int kAppendTokens = 16;          // at most, per work-group
constexpr int kAppendMaxGroups = 1 << 22;  // work-groups of a launch
constexpr int kAppendAngles = 2048;        // (token, pair) factors held in LDS: 16 KB

// How a thread takes a row's channels: eight one by one from any address; eight as a
// vector, those of the other halves of their pairs read besides (rows 16-byte aligned, and
// the halves of the turned part); or two vectors, between which pairs are complete.
enum AppendMode { kAppendEach, kAppendVector, kAppendPairs };

template <typename S, typename C, int kDim, int kMode, bool kStream>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(AppendArgs a) {
  constexpr bool kVec = kMode != kAppendEach;
  constexpr int kSpans = kMode == kAppendPairs ? 2 : 1;
  constexpr int kApart = kDim / kSpans;
  constexpr int kGroup = kDim / 8 / kSpans;  // threads of a row
  constexpr int kBatch = kAppendBatch - kSpans + 1;
  __shared__ float2 factor[kAppendAngles];
  __shared__ const S* row_in[kAppendTokens][3];  // of q, k and v
  __shared__ S* row_out[kAppendTokens];
  __shared__ int64_t first_row[kAppendTokens];   // of the cache: head 0's

  const int half = a.rot >> 1;
  const int64_t first = a.first + (int64_t)blockIdx.x * a.tt;
  const int tokens = (int)(a.total - first < a.tt ? a.total - first : a.tt);
  auto place = [&](int tl, int64_t& b, int64_t& n) {
    const uint32_t t = (uint32_t)(first + tl);
    b = t / (uint32_t)a.tokens;
    n = t - b * a.tokens;
  };
  auto position = [&](int64_t b, int64_t n) -> int64_t {
    const int64_t at = b * a.pos_b + n * a.pos_n;
    return a.pos64 ? static_cast<const int64_t*>(a.pos)[at]
                   : (int64_t) static_cast<const int32_t*>(a.pos)[at];
  };
  // (the last threads, which have fewest angles)
  const int back = kAppendThreads - 1 - (int)threadIdx.x;
  if (back < 4 * tokens) {
    const int tl = back >> 2, w = back & 3;
    int64_t b, n;
    place(tl, b, n);
    if (w < 3) {
      row_in[tl][w] = static_cast<const S*>(a.in[w]) + b * a.in_b[w] + n * a.in_n[w];
    } else {
      row_out[tl] = static_cast<S*>(a.q_out) + b * a.out_b + n * a.out_n;
      int64_t row = kSlotNone;
      if (a.slots) {
        row = cache_row(a.slots[first + tl], 0, a.pages, a.heads, a.page_shift);
      } else {
        const int64_t pos = position(b, n);
        const int64_t entry = pos >> a.page_shift;
        if (pos >= 0 && entry < a.table_pages) {
          const int page = a.table[b * a.table_b + entry];
          if (page_valid(page, a.pages))
            row = (((int64_t)page * a.heads) << a.page_shift) +
                  (pos & ((int64_t(1) << a.page_shift) - 1));
        }
      }
      first_row[tl] = row;
    }
  }
  for (int i = threadIdx.x; i < tokens * half; i += kAppendThreads) {
    const int tl = i / half, p = i - tl * half;
    int64_t b, n;
    place(tl, b, n);
    const float2 cs = turn((double)position(b, n), a.freq[p]);
    factor[i] = {cs.x * a.scale, cs.y * a.scale};
  }
  __syncthreads();

  const int rows = a.q_heads + 2 * a.heads;  // of a token
  const int items = tokens * rows * kGroup;
  const int c = (threadIdx.x & (kGroup - 1)) * 8;
  for (int base = threadIdx.x; base < items; base += kAppendThreads * kBatch) {
    Eight<S> x[kBatch][kSpans], y[kBatch];
    int token[kBatch], head[kBatch], which[kBatch];
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      const int item = base + r * kAppendThreads;
      which[r] = -1;
      if (item >= items) continue;
      const int row = item / kGroup;
      const int tl = divide(row, rows, a.rows_magic);
      int h = row - tl * rows;
      const int w = h < a.q_heads ? 0 : h < a.q_heads + a.heads ? 1 : 2;
      h -= w == 0 ? 0 : w == 1 ? a.q_heads : a.q_heads + a.heads;
      token[r] = tl;
      head[r] = h;
      which[r] = w;
      const S* src = row_in[tl][w] + h * (w == 0 ? a.in_h[0] : w == 1 ? a.in_h[1] : a.in_h[2]);
#pragma unroll
      for (int s = 0; s < kSpans; ++s) {
        if constexpr (kVec)
          x[r][s].template load<kStream>(src + c + s * kApart);
        else
          x[r][s].load_each(src + c + s * kApart);
      }
      if constexpr (kMode != kAppendPairs) {
        if (w < 2 && !a.interleaved && c < a.rot) {  // the pairs' other channels
          if constexpr (kVec) {
            y[r].template load<false>(src + (c < half ? c + half : c - half));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int d = c + i;
              y[r].x[i] = d < a.rot ? src[d < half ? d + half : d - half] : (S)0.0f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      if (which[r] < 0) continue;
      const int64_t row = first_row[token[r]];
      if (which[r] > 0 && row < 0) continue;  // (for all lanes of a row alike)
      float v[kSpans][8];
#pragma unroll
      for (int s = 0; s < kSpans; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[s][i] = x[r][s].value(i);
      if (which[r] < 2) {
        const float2* f = factor + token[r] * half;
        if (a.interleaved) {
#pragma unroll
          for (int s = 0; s < kSpans; ++s)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const int d = c + s * kApart + i;
              if (d >= a.rot) break;
              const float2 cs = f[d >> 1];
              const float x1 = v[s][i], x2 = v[s][i + 1];
              v[s][i] = __builtin_fmaf(x1, cs.x, -(x2 * cs.y));
              v[s][i + 1] = __builtin_fmaf(x2, cs.x, x1 * cs.y);
            }
        } else if constexpr (kMode == kAppendPairs) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 cs = f[c + i];
            const float x1 = v[0][i], x2 = v[1][i];
            v[0][i] = __builtin_fmaf(x1, cs.x, -(x2 * cs.y));
            v[1][i] = __builtin_fmaf(x2, cs.x, x1 * cs.y);
          }
        } else if (c < a.rot) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = c + i;
            if (!kVec && d >= a.rot) break;
            const bool lower = d < half;
            const float2 cs = f[lower ? d : d - half];
            const float other = y[r].value(i) * cs.y;
            v[0][i] = __builtin_fmaf(v[0][i], cs.x, lower ? -other : other);
          }
        }
      }
      if (which[r] == 0) {
#pragma unroll
        for (int s = 0; s < kSpans; ++s) {
          S* dst = row_out[token[r]] + head[r] * a.out_h + c + s * kApart;
          Eight<S> out;
#pragma unroll
          for (int i = 0; i < 8; ++i) out.set(i, v[s][i]);
          if constexpr (kVec)
            out.store(dst);
          else
            out.store_each(dst);
        }
        continue;
      }
      const int64_t at = row + ((int64_t)head[r] << a.page_shift);
      const int w = which[r] - 1;
      void* cache = w ? a.cache[1] : a.cache[0];
      if constexpr (kCoded<C>) {
        put_codes<C, kDim, kSpans>(v, cache, w ? a.cache_scale[1] : a.cache_scale[0], at, c);
      } else {
#pragma unroll
        for (int s = 0; s < kSpans; ++s) {
          Eight<C> out;
#pragma unroll
          for (int i = 0; i < 8; ++i) out.set(i, v[s][i]);
          out.store(held_at<C, kDim>(cache, at, c + s * kApart));
        }
      }
    }
  }
}

template <typename S, typename C, int kDim>
hipError_t launch_append_dim(AppendArgs& a, hipStream_t stream) {
  // A unit for every thread, as long as the grid still covers the 256 CUs several
  // times over (as the rotation alone has it).
  const int half = a.rot / 2, rows = a.q_heads + 2 * a.heads;
  a.tt = 1;
  while (a.tt < kAppendTokens && a.total / (2 * a.tt) >= 2048 && 2 * a.tt * half <= kAppendAngles &&
         a.tt * rows * (kDim / 8) < kAppendThreads)
    a.tt *= 2;
  a.rows_magic = 0xffffffffu / (unsigned)rows + 1;
  uint64_t bytes = (uint64_t)(a.interleaved ? 0 : half) * sizeof(S);
  for (int w = 0; w < 3; ++w) {
    if (w == 0 && a.q_heads == 0) continue;
    bytes |= reinterpret_cast<uintptr_t>(a.in[w]) |
             (uint64_t)(a.in_b[w] | a.in_n[w] | a.in_h[w]) * sizeof(S);
  }
  if (a.q_heads > 0)
    bytes |= reinterpret_cast<uintptr_t>(a.q_out) |
             (uint64_t)(a.out_b | a.out_n | a.out_h) * sizeof(S);
  // (the vectors of 8 channels lie in one half of a turned part each, too)
  const bool vec = bytes % 16 == 0 && (a.interleaved || half % 8 == 0);
  const bool pairs = vec && (a.interleaved || a.rot == kDim);
  // rows that no cache holds anyway are streamed past them
  const bool once = a.total * rows * kDim * (int64_t)sizeof(S) >= kStreamBytes;
  hipError_t e = hipSuccess;
  for (int64_t first = 0; first < a.total && e == hipSuccess;
       first += (int64_t)kAppendMaxGroups * a.tt) {
    a.first = first;
    const int64_t left = (a.total - first + a.tt - 1) / a.tt;
    const unsigned blocks = (unsigned)(left < kAppendMaxGroups ? left : kAppendMaxGroups);
    if (pairs && once)
      cache_append_kernel<S, C, kDim, kAppendPairs, true><<<blocks, kAppendThreads, 0, stream>>>(a);
    else if (pairs)
      cache_append_kernel<S, C, kDim, kAppendPairs, false>
          <<<blocks, kAppendThreads, 0, stream>>>(a);
    else if (vec)
      cache_append_kernel<S, C, kDim, kAppendVector, false>
          <<<blocks, kAppendThreads, 0, stream>>>(a);
    else
      cache_append_kernel<S, C, kDim, kAppendEach, false><<<blocks, kAppendThreads, 0, stream>>>(a);
    e = hipGetLastError();
  }
  return e;
}

template <typename S, typename C>
hipError_t launch_append_type(AppendArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: return launch_append_dim<S, C, 32>(a, stream);
    case 64: return launch_append_dim<S, C, 64>(a, stream);
    case 128: return launch_append_dim<S, C, 128>(a, stream);
    default: return launch_append_dim<S, C, 256>(a, stream);
  }
}

template <typename S>
hipError_t launch_append_source(AppendArgs& a, hipStream_t stream) {
  switch (a.cache_dtype) {
    case 0: return launch_append_type<S, float>(a, stream);
    case 1: return launch_append_type<S, __bf16>(a, stream);
    case 2: return launch_append_type<S, _Float16>(a, stream);
    case 3: return launch_append_type<S, Fp8>(a, stream);
    case 4: return launch_append_type<S, Int8>(a, stream);
    default: return launch_append_type<S, Fp4>(a, stream);
  }
}

}  // namespace

hipError_t launch_cache_append(const AppendArgs& args, hipStream_t stream) {
  AppendArgs a = args;
  switch (a.row_dtype) {
    case 0: return launch_append_source<float>(a, stream);
    case 1: return launch_append_source<__bf16>(a, stream);
    default: return launch_append_source<_Float16>(a, stream);
  }
}

}  // namespace fpx
