// The paged key-value cache (fpx_cache_write, fpx_cache_read): rows of keys
// and values put at their slots, as they are or in 8 bits with a scale per
// row, and read back.
//
// 8-bit rows x of head_dim channels, top = max |x|:
//   FP8 (E4M3): scale = 2^e, the least e with top <= 448 * 2^e; codes
//     x / 2^e rounded to nearest even.  A power of two costs a floating format
//     no precision, makes the division exact, and is what the hardware's own
//     block scales are.
//   INT8: scale = top * (1/127), codes x * (1/scale) rounded to nearest even.
//   top < 2^-100: zeros with scale 0.  top infinite or NaN: zeros with scale
//     NaN, so the row reads back as NaN.
//
// Both kernels only move rows.  head_dim / 8 threads take a row, 8 channels
// each (16 bytes of BF16), so the row's maximum is a reduction of at most 32
// neighbouring lanes with no LDS; kRows rows of k and of v are in flight per
// thread.  Memory bounds the large ones: 64 098 tokens of 8 heads of 128 read
// back from FP8 as BF16, 403 MB, take 64 us, 6.3 TB/s, past the 5.3 of a plain
// copy, as most of it is writes.  7685 tokens of 16 heads of 64, FP16 and INT8,
// are written in 13 us and read back in 12, of which 3 to 4 are a launch.
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

#include <type_traits>

namespace fpx {
namespace {

constexpr int kCacheThreads = 256;
constexpr float kTinyRow = 0x1p-100f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Fp8 {};
struct Int8 {};

// ---- eight channels of a row: raw bits in registers, and their values
template <typename T>
struct Eight {
  typedef T Vec __attribute__((ext_vector_type(8)));
  Vec x;
  template <bool kStream>
  __device__ __forceinline__ void load(const T* p) {
    const Vec* v = reinterpret_cast<const Vec*>(p);
    x = kStream ? __builtin_nontemporal_load(v) : *v;
  }
  // rows of any alignment of T
  __device__ __forceinline__ void load_each(const T* p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Vec*>(p) = x; }
  __device__ __forceinline__ void store_each(T* p) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
  __device__ __forceinline__ float value(int i) const { return (float)x[i]; }
  __device__ __forceinline__ void set(int i, float v) { x[i] = (T)v; }
};

// Eight codes of a row.
struct Codes {
  u32x2 x;
  template <bool kStream>
  __device__ __forceinline__ void load(const uint8_t* p) {
    const u32x2* v = reinterpret_cast<const u32x2*>(p);
    x = kStream ? __builtin_nontemporal_load(v) : *v;
  }
  __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<u32x2*>(p) = x; }
};

template <typename C>
constexpr bool kCoded = __is_same(C, Fp8) || __is_same(C, Int8);
template <typename C>
using Held = std::conditional_t<kCoded<C>, Codes, Eight<C>>;  // eight channels in the cache
template <typename C>
using Elem = std::conditional_t<kCoded<C>, uint8_t, C>;       // one of them

template <int kGroup>
__device__ __forceinline__ float group_max(float v) {
  auto mx = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
  v = mx(v, dpp<0xB1>(v));                          // lane pairs
  v = mx(v, dpp<0x4E>(v));                          // quads
  if constexpr (kGroup >= 8) v = mx(v, dpp<0x141>(v));   // 8 lanes
  if constexpr (kGroup >= 16) v = mx(v, dpp<0x140>(v));  // 16 lanes
  if constexpr (kGroup >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v),
                                                    __builtin_bit_cast(unsigned, v), false, false);
    v = mx(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
  }
  return v;
}

// A row's scale and the factor of its codes, from its largest magnitude.
template <typename C>
__device__ __forceinline__ void row_scale(float top, float& scale, float& factor) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  if ((bits >> 23) == 255u) {
    scale = __builtin_nanf("");
    factor = 0.0f;
  } else if (top < kTinyRow) {
    scale = factor = 0.0f;
  } else if constexpr (__is_same(C, Fp8)) {
    // 448 = 1.75 * 2^8
    const uint32_t e = (bits >> 23) - 8u + ((bits & 0x7fffffu) > 0x600000u);
    scale = __builtin_bit_cast(float, e << 23);
    factor = __builtin_bit_cast(float, (254u - e) << 23);
  } else {
    scale = top * (1.0f / 127.0f);
    factor = 1.0f / scale;
  }
}

// Eight codes of values times the row's factor.  A row without a factor (all
// but zero, or not finite) holds zeros.
template <typename C>
__device__ __forceinline__ u32x2 encode(const float* x, float factor) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = factor == 0.0f ? 0.0f : x[i] * factor;
  u32x2 out;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (__is_same(C, Fp8)) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
      out[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], r, true);
    } else {
      uint32_t r = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r |= ((uint32_t)(int)__builtin_rintf(y[4 * w + i]) & 0xffu) << (8 * i);
      out[w] = r;
    }
  }
  return out;
}

template <typename C>
__device__ __forceinline__ void decode(u32x2 codes, float scale, float* x) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (__is_same(C, Fp8)) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], true);
      x[4 * w] = lo[0] * scale;
      x[4 * w + 1] = lo[1] * scale;
      x[4 * w + 2] = hi[0] * scale;
      x[4 * w + 3] = hi[1] * scale;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[4 * w + i] = (float)(int)(int8_t)(codes[w] >> (8 * i)) * scale;
    }
  }
}

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
        Held<C> y;
        if constexpr (kCoded<C>) {
          float v[8], top = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = x[r][w].value(i);
            top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[i]));
          }
          top = group_max<kGroup>(top);
          float scale, factor;
          row_scale<C>(top, scale, factor);
          y.x = encode<C>(v, factor);
          if (c == 0) a.scale[w][at[r]] = scale;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (__is_same(S, C))
              y.x[i] = x[r][w].x[i];
            else
              y.set(i, x[r][w].value(i));
          }
        }
        y.store(static_cast<Elem<C>*>(a.cache[w]) + at[r] * kDim + c);
      }
    }
  }
}

// The rows of `slots` back as S: zeros where there is no slot, NaN for a slot
// past the cache's end.
template <typename S, typename C, int kDim, bool kVec, bool kStream>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(CacheArgs a) {
  constexpr int kGroup = kDim / 8;
  constexpr int kPass = kCacheThreads / kGroup;
  constexpr int kRows = 4;
  const int c = (threadIdx.x & (kGroup - 1)) * 8;
  const int64_t rows = a.tokens * a.heads;
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
      t[r] = (uint32_t)row / (uint32_t)a.heads;
      h[r] = (int)((uint32_t)row - t[r] * (uint32_t)a.heads);
      at[r] = cache_row(a.slots[t[r]], h[r], a.pages, a.heads, a.page_shift);
    }
    Held<C> held[kRows][2];
    float scale[kRows][2];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (at[r] < 0) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        held[r][w].template load<kStream>(static_cast<const Elem<C>*>(a.cache[w]) + at[r] * kDim +
                                          c);
        if constexpr (kCoded<C>) scale[r][w] = a.scale[w][at[r]];
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (base + r * kPass >= rows) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        Eight<S> y;
        const float fill = at[r] == kSlotOutside ? __builtin_nanf("") : 0.0f;
        if constexpr (kCoded<C>) {
          float v[8];
          decode<C>(held[r][w].x, scale[r][w], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) y.set(i, at[r] < 0 ? fill : v[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (__is_same(S, C))
              y.x[i] = at[r] < 0 ? (S)fill : held[r][w].x[i];
            else
              y.set(i, at[r] < 0 ? fill : held[r][w].value(i));
          }
        }
        S* dst = const_cast<S*>(static_cast<const S*>(a.rows[w])) + t[r] * a.stride_t[w] +
                 h[r] * a.stride_h[w] + c;
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
  const int64_t per = kPass * (read ? 4 : 2);
  const int64_t blocks = (a.tokens * a.heads + per - 1) / per;
  // (the kernels walk on in strides of the grid)
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
  uint64_t bytes = 0;
  for (int w = 0; w < 2; ++w)
    bytes |= reinterpret_cast<uintptr_t>(a.rows[w]) |
             (uint64_t)(a.stride_t[w] | a.stride_h[w]) * sizeof(S);
  const bool vec = bytes % 16 == 0;
  // what is read and no cache holds anyway is streamed past them
  const int64_t row = kDim * (read ? (int64_t)sizeof(Elem<C>) : (int64_t)sizeof(S));
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
    default: return launch_cache_type<S, Int8>(a, read, stream);
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
