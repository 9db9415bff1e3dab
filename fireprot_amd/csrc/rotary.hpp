// The rotation of a position, shared by the kernels that turn rows by it.
#pragma once

#include "common.hpp"

namespace fpx {

// cos and sin of pos * freq, in FP32 to a few units of 2^-24.  The product is
// taken in FP64 and reduced to turns with a two-term 1 / (2 pi), since an
// FP32 angle of position 2^20 has already lost its last four decimal digits;
// the quarter turn's rest, within pi/4, goes through the Taylor series (the
// first terms left out are below 3e-9).
__device__ __forceinline__ float2 turn(double pos, double freq) {
  constexpr double kInv2Pi = 0.15915494309189535;
  constexpr double kInv2PiLow = -9.839338337591243e-18;  // 1/(2 pi) - kInv2Pi
  const double a = pos * freq;
  const double hi = a * kInv2Pi;
  const double lo = __builtin_fma(a, kInv2Pi, -hi) + a * kInv2PiLow;
  const double t = ((hi - __builtin_rint(hi)) + lo) * 4.0;  // quarter turns
  const double quarter = __builtin_rint(t);
  const float x = (float)((t - quarter) * 1.57079632679489661923);
  const float z = x * x;
  float s = 1.0f / 362880.0f;
  s = __builtin_fmaf(s, z, -1.0f / 5040.0f);
  s = __builtin_fmaf(s, z, 1.0f / 120.0f);
  s = __builtin_fmaf(s, z, -1.0f / 6.0f);
  s = __builtin_fmaf(x * z, s, x);
  float c = -1.0f / 3628800.0f;
  c = __builtin_fmaf(c, z, 1.0f / 40320.0f);
  c = __builtin_fmaf(c, z, -1.0f / 720.0f);
  c = __builtin_fmaf(c, z, 1.0f / 24.0f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  const int q = (int)quarter & 3;
  const float cs = (q & 1) ? s : c;
  const float sn = (q & 1) ? c : s;
  return {(q == 1 || q == 2) ? -cs : cs, (q >= 2) ? -sn : sn};
}

// x / n by n's magic number 2^32 / n + 1, for x * n < 2^32.
__device__ __forceinline__ int divide(int x, int n, unsigned magic) {
  return n == 1 ? x : (int)__umulhi((unsigned)x, magic);
}

}  // namespace fpx
