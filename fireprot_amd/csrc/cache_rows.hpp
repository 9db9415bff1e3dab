// Rows of the paged key-value cache as its kernels hold them: eight channels to a
// thread, converted to a plain type or to codes with scales as they are written, and
// back.
//
// 8-bit rows x of head_dim channels, top = max |x|:
//   FP8 (E4M3): scale = 2^e, the least e with top <= 448 * 2^e; codes
//     x / 2^e rounded to nearest even.  A power of two costs a floating format
//     no precision, makes the division exact, and is what the hardware's own
//     block scales are.
//   INT8: scale = top * (1/127), codes x * (1/scale) rounded to nearest even.
//   top < 2^-100: zeros with scale 0.  top infinite or NaN: zeros with scale
//     NaN, so the row reads back as NaN.
// 4-bit rows (FP4) go by blocks of 32 channels, with a top and a scale each:
//   codes E2M1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), two to a byte, the first in
//     its low half: x / 2^e rounded to nearest even, at most 6; scale 2^e in one byte
//     (e + 127), the least e with top <= 7 * 2^e, and 125 at most, so that no code
//     stands for an infinite value.  Up to 7 the largest code is off by no more than
//     half of its step, as any other; a block scaled for 6 would lose a bit of all its
//     values where top lies between.
//   top < 2^-100: zeros with scale 2^-127.  top infinite or NaN: scale 255, which is
//     NaN, so the block reads back as NaN.
#pragma once

#include "common.hpp"

#include <type_traits>

namespace fpx {

constexpr float kTinyRow = 0x1p-100f;
constexpr int kBlock4 = 32;  // channels that share a scale in 4 bits

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Fp8 {};
struct Int8 {};
struct Fp4 {};

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

// Eight codes of a row, of 8 or 4 bits.
template <typename Word>
struct Codes {
  Word x;
  template <bool kStream>
  __device__ __forceinline__ void load(const uint8_t* p) {
    const Word* v = reinterpret_cast<const Word*>(p);
    x = kStream ? __builtin_nontemporal_load(v) : *v;
  }
  __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<Word*>(p) = x; }
};

template <typename C>
constexpr bool kByteCoded = __is_same(C, Fp8) || __is_same(C, Int8);
template <typename C>
constexpr bool kCoded = kByteCoded<C> || __is_same(C, Fp4);
// eight channels in the cache, and one of its elements (FP4: two channels)
template <typename C>
using Held = std::conditional_t<__is_same(C, Fp4), Codes<uint32_t>,
                                std::conditional_t<kByteCoded<C>, Codes<u32x2>, Eight<C>>>;
template <typename C>
using Elem = std::conditional_t<kCoded<C>, uint8_t, C>;

// Bytes of a row's `channels`.
template <typename C>
constexpr int64_t held_bytes(int64_t channels) {
  return __is_same(C, Fp4) ? channels / 2 : channels * (int64_t)sizeof(Elem<C>);
}

// Channel c (a multiple of 8) of a row of kDim, and its scale.
template <typename C, int kDim, typename P>
__device__ __forceinline__ auto held_at(P* cache, int64_t row, int c) {
  using E = std::conditional_t<std::is_const_v<P>, const Elem<C>, Elem<C>>;
  E* rows = static_cast<E*>(cache);
  if constexpr (__is_same(C, Fp4))
    return rows + (row * kDim + c) / 2;
  else
    return rows + row * kDim + c;
}

template <typename C, int kDim>
__device__ __forceinline__ float scale_at(const void* scale, int64_t row, int c) {
  if constexpr (__is_same(C, Fp4)) {
    const uint32_t e = static_cast<const uint8_t*>(scale)[(row * kDim + c) / kBlock4];
    return __builtin_bit_cast(float, e << 23);  // as the conversions take it
  } else {
    return static_cast<const float*>(scale)[row];
  }
}

// The maximum over kGroup neighbouring lanes (2 to 32, aligned), in each.
template <int kGroup>
__device__ __forceinline__ float group_max(float v) {
  auto mx = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
  v = mx(v, dpp<0xB1>(v));                          // lane pairs
  if constexpr (kGroup >= 4) v = mx(v, dpp<0x4E>(v));    // quads
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

// A 4-bit block's scale byte.
__device__ __forceinline__ uint32_t block_scale(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  if ((bits >> 23) == 255u) return 255u;
  if (top < kTinyRow) return 0u;
  // 7 = 1.75 * 2^2
  return min((bits >> 23) - 2u + ((bits & 0x7fffffu) > 0x600000u), 252u);
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

// Eight 4-bit codes by their block's scale byte; zeros where that is 0 or 255.
__device__ __forceinline__ uint32_t encode4(const float* x, uint32_t e) {
  const float scale = __builtin_bit_cast(float, e << 23);
  uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
  return e == 0u || e == 255u ? 0u : r;
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

template <typename C>
__device__ __forceinline__ void decode(uint32_t codes, float scale, float* x) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  x[0] = a[0];
  x[1] = a[1];
  x[2] = b[0];
  x[3] = b[1];
  x[4] = c[0];
  x[5] = c[1];
  x[6] = d[0];
  x[7] = d[1];
}

// Channels c + s * kDim / kSpans to c + 7 + s * kDim / kSpans of a row into a coded
// cache, v[s] their values; the row's kDim / 8 / kSpans threads are neighbouring lanes that
// all call this, with c from 0 in steps of 8.
template <typename C, int kDim, int kSpans>
__device__ __forceinline__ void put_codes(const float (*v)[8], void* cache, void* scales,
                                          int64_t row, int c) {
  constexpr int kLanes = kDim / 8 / kSpans;
  float top[kSpans];
#pragma unroll
  for (int s = 0; s < kSpans; ++s) {
    top[s] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      top[s] = __builtin_elementwise_maximum(top[s], __builtin_fabsf(v[s][i]));
  }
  // (a 4-bit block of 32 channels is that of four lanes, or of all spans of fewer)
  constexpr bool kTogether = !__is_same(C, Fp4) || kLanes < kBlock4 / 8;
  if constexpr (kTogether) {
#pragma unroll
    for (int s = 1; s < kSpans; ++s) top[0] = __builtin_elementwise_maximum(top[0], top[s]);
    top[0] = group_max<kLanes>(top[0]);
  }
  float scale = 0.0f, factor = 0.0f;
  if constexpr (!__is_same(C, Fp4)) {
    row_scale<C>(top[0], scale, factor);
    if (c == 0) static_cast<float*>(scales)[row] = scale;
  }
#pragma unroll
  for (int s = 0; s < kSpans; ++s) {
    const int at = c + s * (kDim / kSpans);
    Held<C> y;
    if constexpr (__is_same(C, Fp4)) {
      const uint32_t e = block_scale(kTogether ? top[0] : group_max<kBlock4 / 8>(top[s]));
      y.x = encode4(v[s], e);
      if (at % kBlock4 == 0)
        static_cast<uint8_t*>(scales)[(row * kDim + at) / kBlock4] = (uint8_t)e;
    } else {
      y.x = encode<C>(v[s], factor);
    }
    y.store(held_at<C, kDim>(cache, row, at));
  }
}

}  // namespace fpx
