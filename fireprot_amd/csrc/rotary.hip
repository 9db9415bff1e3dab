// Rotary positions (fpx_rotary): rows x[b][n][h] of head_dim channels, the
// first `rot` of them turned in pairs by the angle position(b, n) * freq[i]:
//
//   y1 = s (x1 cos a - x2 sin a),   y2 = s (x2 cos a + x1 sin a)
//
// with pairs (i, i + rot/2) (half layout) or (2i, 2i + 1) (interleaved); the
// remaining channels are copied.  The rotation is orthogonal, so the gradient
// is the same map with the angle negated (`inverse`).
#include "common.hpp"
#include "kernels.hpp"
#include "rotary.hpp"

#include <type_traits>

namespace fpx {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBatch = 4;       // rows in flight per thread
constexpr int kRotaryTokens = 16;      // at most, per work-group
constexpr int kRotaryMaxGroups = 1 << 22;  // work-groups of a launch
constexpr int kRotaryAngles = 2048;   // (token, pair) factors held in LDS: 16 KB

// Work-group: `tt` tokens of all heads of both tensors.  The factors of each
// (token, pair) are computed once, into LDS, and serve every head.  Then the
// threads take the units of all rows (token, head) in turn, one W-byte vector of
// each half (or one vector of pairs) to a unit, kRotaryBatch at a time with their
// loads issued before the first use.  In place is safe: a thread's stores go to
// exactly the channels it has read.  Bound by memory: 16384 tokens of 40 BF16
// heads of 128, 336 MB read and written, take 56 us, 6.0 TB/s (a plain copy
// reaches 5.3); the FP64 angles are a fortieth of what they would be row by row.
template <typename T, int W, bool kInterleaved, bool kStream>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int kElems = W / (int)sizeof(T);                // of one vector
  constexpr bool kPairVector = kInterleaved && kElems >= 2; // a vector holds whole pairs
  constexpr int kPairs = kPairVector ? kElems / 2 : kElems; // of one unit
  typedef T Vec __attribute__((ext_vector_type(kElems)));
  __shared__ float2 factor[kRotaryAngles];
  __shared__ const T* row_in[kRotaryTokens][2];
  __shared__ T* row_out[kRotaryTokens][2];

  const int half = a.rot >> 1;
  const int first = a.first + blockIdx.x * a.tt;
  const int tokens = min(a.total - first, a.tt);
  for (int i = threadIdx.x; i < tokens * half; i += kRotaryThreads) {
    const int tl = i / half, p = i - tl * half;
    const int t = first + tl, b = t / a.tokens, n = t - b * a.tokens;
    const int64_t at = b * a.pos_b + n * a.pos_n;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at]
                               : (double)static_cast<const int32_t*>(a.pos)[at];
    const float2 cs = turn(pos, a.freq[p]);
    factor[i] = {cs.x * a.scale, (a.inverse ? -cs.y : cs.y) * a.scale};
  }
  if ((int)threadIdx.x < 2 * tokens) {
    const int tl = threadIdx.x >> 1, w = threadIdx.x & 1;
    const int64_t t = first + tl, b = t / a.tokens, n = t - b * a.tokens;
    const RotaryTensor x = w ? a.x[1] : a.x[0];
    row_in[tl][w] = static_cast<const T*>(x.in) + b * x.in_b + n * x.in_n;
    row_out[tl][w] = static_cast<T*>(x.out) + b * x.out_b + n * x.out_n;
  }
  __syncthreads();

  const int q_heads = a.x[0].heads, heads = q_heads + a.x[1].heads;
  const int items = tokens * heads * a.units;
  const int rot_units = half / kPairs;
  for (int base = threadIdx.x; base < items; base += kRotaryThreads * kRotaryBatch) {
    Vec u[kRotaryBatch], v[kRotaryBatch];
    T* dst[kRotaryBatch];   // the unit's first channel
    int local[kRotaryBatch];  // its first factor; negative: a copy
#pragma unroll
    for (int r = 0; r < kRotaryBatch; ++r) {
      const int item = base + r * kRotaryThreads;
      if (item >= items) continue;
      const int row = divide(item, a.units, a.units_magic);
      const int unit = item - row * a.units;
      const int tl = divide(row, heads, a.heads_magic);
      int h = row - tl * heads;
      const int w = h >= q_heads;
      h -= w ? q_heads : 0;
      // a unit past the rotated part copies one vector
      const bool turned = unit < rot_units;
      const int c0 = !turned        ? a.rot + (unit - rot_units) * kElems
                     : kInterleaved ? 2 * unit * kPairs
                                    : unit * kPairs;
      const T* src = row_in[tl][w] + h * (w ? a.x[1].in_h : a.x[0].in_h) + c0;
      dst[r] = row_out[tl][w] + h * (w ? a.x[1].out_h : a.x[0].out_h) + c0;
      local[r] = turned ? tl * half + unit * kPairs : -1;
      const Vec* p0 = reinterpret_cast<const Vec*>(src);
      u[r] = kStream ? __builtin_nontemporal_load(p0) : *p0;
      if (turned && !kPairVector) {
        const Vec* p1 = reinterpret_cast<const Vec*>(src + (kInterleaved ? 1 : half));
        v[r] = kStream ? __builtin_nontemporal_load(p1) : *p1;
      }
    }
#pragma unroll
    for (int r = 0; r < kRotaryBatch; ++r) {
      if (base + r * kRotaryThreads >= items) continue;
      if (local[r] >= 0) {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
          const float2 f = factor[local[r] + p];
          if constexpr (kPairVector) {
            const float x1 = (float)u[r][2 * p], x2 = (float)u[r][2 * p + 1];
            u[r][2 * p] = (T)__builtin_fmaf(x1, f.x, -(x2 * f.y));
            u[r][2 * p + 1] = (T)__builtin_fmaf(x2, f.x, x1 * f.y);
          } else {
            const float x1 = (float)u[r][p], x2 = (float)v[r][p];
            u[r][p] = (T)__builtin_fmaf(x1, f.x, -(x2 * f.y));
            v[r][p] = (T)__builtin_fmaf(x2, f.x, x1 * f.y);
          }
        }
        if constexpr (!kPairVector)
          *reinterpret_cast<Vec*>(dst[r] + (kInterleaved ? 1 : half)) = v[r];
      }
      *reinterpret_cast<Vec*>(dst[r]) = u[r];
    }
  }
}

template <typename T, int W, bool kStream>
hipError_t launch_width(const RotaryArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.interleaved)
    rotary_kernel<T, W, true, kStream><<<blocks, kRotaryThreads, 0, stream>>>(a);
  else
    rotary_kernel<T, W, false, kStream><<<blocks, kRotaryThreads, 0, stream>>>(a);
  return hipGetLastError();
}

// Largest vector, in bytes, that divides every row's base, the rotated halves
// (or pairs) and the copied rest.
int vector_bytes(const RotaryArgs& a, int elem) {
  uint64_t bits = (uint64_t)(a.interleaved ? a.rot : a.rot / 2) | (uint64_t)(a.head_dim - a.rot);
  uint64_t bytes = 0;
  for (const RotaryTensor& x : a.x) {
    if (x.heads == 0) continue;
    bits |= (uint64_t)(x.in_b | x.in_n | x.in_h | x.out_b | x.out_n | x.out_h);
    bytes |= reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out);
  }
  bytes |= bits * elem;
  int w = 16;
  while (w > elem && bytes % w) w >>= 1;
  return w;
}

template <typename T>
hipError_t launch_type(RotaryArgs& a, hipStream_t stream) {
  int w = vector_bytes(a, sizeof(T));
  const int elems = w / (int)sizeof(T);
  const int half = a.rot / 2;
  const int pairs = a.interleaved && elems >= 2 ? elems / 2 : elems;
  // rows in place keep the channels past the rotated ones as they are
  bool copies = a.head_dim > a.rot;
  if (copies && a.x[0].in == a.x[0].out && (a.x[1].heads == 0 || a.x[1].in == a.x[1].out))
    copies = false;
  a.units = half / pairs + (copies ? (a.head_dim - a.rot) / elems : 0);
  // Tokens of a work-group: a unit for every thread, as long as the grid still
  // covers the 256 CUs several times over (16384 tokens of 40 heads of 128 take
  // 56 us with one token, 62 with four; 32768 tokens of 4 heads of 64 take 11 us
  // with sixteen, 40 with one).
  a.tt = 1;
  const int heads = a.x[0].heads + a.x[1].heads;
  a.units_magic = 0xffffffffu / (unsigned)a.units + 1;
  a.heads_magic = 0xffffffffu / (unsigned)heads + 1;
  while (a.tt < kRotaryTokens && a.total / (2 * a.tt) >= 2048 && 2 * a.tt * half <= kRotaryAngles &&
         a.tt * heads * a.units < kRotaryThreads)
    a.tt *= 2;
  // Rows of whole 16-byte vectors that no cache holds anyway are streamed past
  // them (see kStreamBytes); narrower vectors read a line several times over.
  const bool stream_rows =
      (int64_t)a.total * heads * a.head_dim * (int64_t)sizeof(T) >= kStreamBytes;
  hipError_t e = hipSuccess;
  for (int64_t first = 0; first < a.total && e == hipSuccess;
       first += (int64_t)kRotaryMaxGroups * a.tt) {
    a.first = (int)first;
    const int64_t left = (a.total - first + a.tt - 1) / a.tt;
    const unsigned blocks = (unsigned)(left < kRotaryMaxGroups ? left : kRotaryMaxGroups);
    switch (w) {
      case 16:
        e = stream_rows ? launch_width<T, 16, true>(a, blocks, stream)
                        : launch_width<T, 16, false>(a, blocks, stream);
        break;
      case 8: e = launch_width<T, 8, false>(a, blocks, stream); break;
      case 4: e = launch_width<T, 4, false>(a, blocks, stream); break;
      default:
        e = hipErrorInvalidValue;
        if constexpr (sizeof(T) == 2) e = launch_width<T, 2, false>(a, blocks, stream);
    }
  }
  return e;
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& args, hipStream_t stream) {
  RotaryArgs a = args;
  switch (a.dtype) {
    case 0: return launch_type<float>(a, stream);
    case 1: return launch_type<__bf16>(a, stream);
    default: return launch_type<_Float16>(a, stream);
  }
}

}  // namespace fpx
