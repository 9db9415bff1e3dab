// Which pages of the paged cache a new token's queries can hardly do without
// (fpx_page_bounds, fpx_select_pages).
//
//   bounds[page][head] = (lo, hi), channel by channel over the page's keys
//   score(b, h, page)  = max over head h's queries of sum_c max(q_c lo_c, q_c hi_c),
//
// no less than any q . k of the page.  With q+ = max(q, 0) and q- = min(q, 0) it is a
// product, q+ . hi + q- . lo, which runs on the FP64 matrix cores: two pages next to
// each other in rank must come out in the same order whatever order the sum is taken
// in, and an FP32 sum of 128 terms is off by more than the step between scores where
// thousands of pages compete for the last place.  FP64 costs nothing here: a page of 64
// keys, BF16, 128 channels, is 512 bytes of bounds and 32 of the matrix cores' FP64
// instructions for each 16 pages and queries, 1.7 us of one SIMD.  The sum is rounded
// to FP32 once; of pages alike the lower is preferred.
#include "cache_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kBoundsThreads = 256;
constexpr int kScoreThreads = 256;
constexpr int kScorePages = 64;  // of a work-group

__device__ __forceinline__ float lesser(float x, float y) {
  return __builtin_elementwise_minimum(x, y);
}
__device__ __forceinline__ float greater(float x, float y) {
  return __builtin_elementwise_maximum(x, y);
}

// A bound in its type: exact for a plain cache's values, in BF16 the next number not
// above (below) the value of a code.
template <typename T>
__device__ __forceinline__ T bound(float x, bool upper) {
  if constexpr (__is_same(T, __bf16)) {
    uint32_t bits = __builtin_bit_cast(uint32_t, x);
    if (!(x == x)) return (__bf16)x;
    // cut towards zero, and away from it where that would cut the bound
    if ((bits & 0xffffu) && (x > 0.0f) == upper) bits += 0x10000u;
    return __builtin_bit_cast(__bf16, (uint16_t)(bits >> 16));
  } else {
    return (T)x;
  }
}

// The bounds of the pages that hold the last `fresh` tokens of each sequence: one
// work-group to a (sequence, cache head, page).
template <typename C, typename T, int kDim>
__global__ __launch_bounds__(kBoundsThreads) void page_bounds_kernel(BoundsArgs a) {
  constexpr int kGroup = kDim / 8;                     // threads of a row
  constexpr int kPass = kBoundsThreads / kGroup;       // rows of a pass
  constexpr int kRows = 4;                             // passes in flight
  constexpr int kWaves = kBoundsThreads / kWave;
  __shared__ float part[2][kWaves][kDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (threadIdx.x & (kGroup - 1)) * 8;
  const int64_t item = blockIdx.x;
  const int64_t seq_head = item / a.each;
  const int i = (int)(item - seq_head * a.each);
  const int64_t b = seq_head / a.heads;
  const int h = (int)(seq_head - b * a.heads);
  const KeyRange range = key_range(a.lengths[b], a.max_length, 0);
  if (!range.valid) return;
  const int from = range.end > a.fresh ? range.end - a.fresh : 0;
  const int64_t at = (int64_t)(from >> a.page_shift) + i;
  const int64_t left = range.end - (at << a.page_shift);  // keys from the page on
  if (left <= 0) return;
  const int page = a.table[b * a.table_b + at];
  if (!page_valid(page, a.pages)) return;
  const int size = 1 << a.page_shift;
  const int rows = left < size ? (int)left : size;
  const int64_t first = ((int64_t)page * a.heads + h) << a.page_shift;

  float lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo[j] = __builtin_inff();
    hi[j] = -__builtin_inff();
  }
  for (int base = threadIdx.x / kGroup; base < rows; base += kPass * kRows) {
    Held<C> x[kRows];
    float scale[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      // (past the last row the last again)
      const int64_t row = first + min(base + r * kPass, rows - 1);
      x[r].template load<false>(held_at<C, kDim>(a.k, row, c));
      if constexpr (kCoded<C>) scale[r] = scale_at<C, kDim>(a.k_scale, row, c);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float v[8];
      if constexpr (kCoded<C>) {
        decode<C>(x[r].x, scale[r], v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[r].value(j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = lesser(lo[j], v[j]);
        hi[j] = greater(hi[j], v[j]);
      }
    }
  }
  // lanes that hold the same channels, then the waves
#pragma unroll
  for (int d = kGroup; d < kWave; d *= 2)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = lesser(lo[j], __shfl_xor(lo[j], d));
      hi[j] = greater(hi[j], __shfl_xor(hi[j], d));
    }
  if (lane < kGroup) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      part[0][wave][c + j] = lo[j];
      part[1][wave][c + j] = hi[j];
    }
  }
  __syncthreads();
  T* out = static_cast<T*>(a.bounds) + ((int64_t)page * a.heads + h) * 2 * kDim;
  for (int t = threadIdx.x; t < 2 * kDim; t += kBoundsThreads) {
    const int upper = t / kDim, ch = t - upper * kDim;
    float x = part[upper][0][ch];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const float y = part[upper][w][ch];
      x = upper ? greater(x, y) : lesser(x, y);
    }
    out[t] = bound<T>(x, upper);
  }
}

// A score as a number that grows with it: NaN above all others, and above NaN the pages
// that are taken whatever their score.
constexpr uint32_t kForced = 0xffffffffu, kNanRank = 0xfffffffeu;

__device__ __forceinline__ uint32_t rank_of(float score) {
  if (!(score == score)) return kNanRank;
  const uint32_t bits = __builtin_bit_cast(uint32_t, score + 0.0f);  // (no -0)
  return bits >> 31 ? ~bits : bits | 0x80000000u;
}

// The ranks of 64 pages of one sequence for one cache head, 16 to a wave: queries are
// the rows of the products, pages the columns.  A lane holds a quarter of its page's
// (and of its query's) channels, as they lie in memory: in which order the channels are
// contracted is no matter as long as both sides have the same.
template <typename Q, typename T, int kDim>
__global__ __launch_bounds__(kScoreThreads) void page_rank_kernel(SelectArgs a) {
  constexpr int kQuarter = kDim / 4;
  typedef Q QVec __attribute__((ext_vector_type(8)));
  typedef T TVec __attribute__((ext_vector_type(8)));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int64_t seq_head = blockIdx.x / (unsigned)a.tiles;
  const int tile = (int)(blockIdx.x - seq_head * a.tiles);
  const int64_t b = seq_head / a.heads;
  const int h = (int)(seq_head - b * a.heads);
  const KeyRange range = key_range(__builtin_amdgcn_readfirstlane(a.lengths[b]), a.max_length, 0);
  const int total = (range.end + (1 << a.page_shift) - 1) >> a.page_shift;  // pages
  const int page0 = tile * kScorePages + wave * 16;
  if (total <= a.count || page0 >= total) return;  // (all pages are taken: no ranks)
  const int at = min(page0 + col, total - 1);
  const int page = a.table[b * a.table_b + at];
  const bool ok = page_valid(page, a.pages);
  const T* lo = static_cast<const T*>(a.bounds) +
                ((int64_t)(ok ? page : 0) * a.heads + h) * 2 * kDim + g * kQuarter;
  float best = -__builtin_inff();
  for (int q0 = 0; q0 < a.group; q0 += 16) {
    // (rows past the head's last query have its first one again)
    const int qi = q0 + col < a.group ? q0 + col : 0;
    const Q* q = static_cast<const Q*>(a.q) + b * a.q_b + ((int64_t)h * a.group + qi) * a.q_h +
                 g * kQuarter;
    f64x4 above = {0.0, 0.0, 0.0, 0.0}, below = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int s = 0; s < kQuarter; s += 8) {
      const QVec x = *reinterpret_cast<const QVec*>(q + s);
      const TVec l = *reinterpret_cast<const TVec*>(lo + s);
      const TVec u = *reinterpret_cast<const TVec*>(lo + kDim + s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = (float)x[j];
        above = __builtin_amdgcn_mfma_f64_16x16x4f64((double)greater(y, 0.0f), (double)(float)u[j],
                                                     above, 0, 0, 0);
        below = __builtin_amdgcn_mfma_f64_16x16x4f64((double)lesser(y, 0.0f), (double)(float)l[j],
                                                     below, 0, 0, 0);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) best = greater(best, (float)(above[r] + below[r]));
  }
  // the queries of the other lane groups
  best = greater(best, __shfl_xor(best, 16));
  best = greater(best, __shfl_xor(best, 32));
  if (g == 0 && page0 + col < total) {
    const bool forced = at < a.sinks || at >= total - a.recent;
    a.ranks[seq_head * a.max_pages + at] = forced ? kForced : ok ? rank_of(best) : kNanRank;
  }
}

// The `count` pages of highest rank of one (sequence, cache head), in the order of the
// sequence: the rank of the last of them is found byte by byte from the counts of each
// byte's values, then every thread lists its run of pages.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void page_select_kernel(SelectArgs a) {
  constexpr int kWaves = kThreads / kWave;
  constexpr int kCopies = 8;  // of the counts: neighbouring lanes' ranks begin alike
  __shared__ uint32_t counts[256][kCopies];
  __shared__ uint32_t found[2];
  __shared__ int wave_sum[2][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t seq_head = blockIdx.x;
  const int64_t b = seq_head / a.heads;
  const KeyRange range = key_range(__builtin_amdgcn_readfirstlane(a.lengths[b]), a.max_length, 0);
  const int size = 1 << a.page_shift;
  const int total = range.valid ? (range.end + size - 1) >> a.page_shift : 0;
  const int kept = total < a.count ? total : a.count;
  const int32_t* table = a.table + b * a.table_b;
  int32_t* index = a.index + seq_head * a.count;
  int32_t* out = a.table_out + seq_head * a.count;
  if (threadIdx.x == 0 && seq_head == b * a.heads)
    a.lengths_out[b] = range.valid ? range.end - ((total - kept) << a.page_shift) : -1;
  for (int i = kept + threadIdx.x; i < a.count; i += kThreads) index[i] = out[i] = -1;
  if (total <= a.count) {
    for (int i = threadIdx.x; i < total; i += kThreads) {
      index[i] = i;
      out[i] = table[i];
    }
    return;
  }
  const uint32_t* ranks = a.ranks + seq_head * a.max_pages;
  uint32_t least = 0, mask = 0;  // the bytes found so far
  uint32_t wanted = (uint32_t)a.count;  // pages among those that begin with them
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256 * kCopies; i += kThreads)
      counts[i / kCopies][i % kCopies] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const uint32_t r = ranks[i];
      if (((r ^ least) & mask) == 0) atomicAdd(&counts[(r >> shift) & 255][lane % kCopies], 1u);
    }
    __syncthreads();
    if (wave == 0) {
      // lane l has the values 4l to 4l + 3; `upto`: pages of its and all higher ones
      uint32_t own[4], sum = 0;
#pragma unroll
      for (int v = 3; v >= 0; --v) {
        own[v] = 0;
#pragma unroll
        for (int k = 0; k < kCopies; ++k) own[v] += counts[4 * lane + v][k];
        sum += own[v];
      }
      uint32_t upto = sum;
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) {
        const uint32_t above = __shfl_down(upto, d);
        upto += lane + d < kWave ? above : 0;
      }
      uint32_t above = upto - sum;
      if (above < wanted && wanted <= upto) {
        int v = 3;
        while (v > 0 && above + own[v] < wanted) above += own[v--];
        found[0] = (uint32_t)(4 * lane + v);
        found[1] = wanted - above;
      }
    }
    __syncthreads();
    least |= found[0] << shift;
    wanted = found[1];
    mask |= 255u << shift;
  }
  // ---- pages of a higher rank, and the first `wanted` of that rank itself
  const int per = (total + kThreads - 1) / kThreads;
  const int begin = min(total, (int)threadIdx.x * per), end = min(total, begin + per);
  int higher = 0, equal = 0;
  for (int i = begin; i < end; ++i) {
    higher += ranks[i] > least;
    equal += ranks[i] == least;
  }
  int before[2] = {higher, equal};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int x = __shfl_up(before[w], d);
      before[w] += lane >= d ? x : 0;
    }
    if (lane == kWave - 1) wave_sum[w][wave] = before[w];
  }
  __syncthreads();
  before[0] -= higher;
  before[1] -= equal;
  for (int w = 0; w < wave; ++w) {
    before[0] += wave_sum[0][w];
    before[1] += wave_sum[1][w];
  }
  for (int i = begin; i < end; ++i) {
    const uint32_t r = ranks[i];
    const bool taken = r > least || (r == least && before[1] < (int)wanted);
    if (taken) {
      const int to = before[0] + min(before[1], (int)wanted);
      index[to] = i;
      out[to] = table[i];
    }
    before[0] += r > least;
    before[1] += r == least;
  }
}

template <typename C, typename T>
hipError_t launch_bounds_type(const BoundsArgs& a, unsigned groups, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: page_bounds_kernel<C, T, 32><<<groups, kBoundsThreads, 0, stream>>>(a); break;
    case 64: page_bounds_kernel<C, T, 64><<<groups, kBoundsThreads, 0, stream>>>(a); break;
    case 128: page_bounds_kernel<C, T, 128><<<groups, kBoundsThreads, 0, stream>>>(a); break;
    default: page_bounds_kernel<C, T, 256><<<groups, kBoundsThreads, 0, stream>>>(a); break;
  }
  return hipGetLastError();
}

template <typename Q, typename T>
void launch_rank_type(const SelectArgs& a, unsigned groups, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: page_rank_kernel<Q, T, 32><<<groups, kScoreThreads, 0, stream>>>(a); break;
    case 64: page_rank_kernel<Q, T, 64><<<groups, kScoreThreads, 0, stream>>>(a); break;
    case 128: page_rank_kernel<Q, T, 128><<<groups, kScoreThreads, 0, stream>>>(a); break;
    default: page_rank_kernel<Q, T, 256><<<groups, kScoreThreads, 0, stream>>>(a); break;
  }
}

template <typename Q>
void launch_rank(const SelectArgs& a, unsigned groups, hipStream_t stream) {
  switch (a.bounds_dtype) {
    case 0: launch_rank_type<Q, float>(a, groups, stream); break;
    case 1: launch_rank_type<Q, __bf16>(a, groups, stream); break;
    default: launch_rank_type<Q, _Float16>(a, groups, stream); break;
  }
}

}  // namespace

hipError_t launch_page_bounds(const BoundsArgs& a, hipStream_t stream) {
  const unsigned groups = (unsigned)((int64_t)a.batch * a.heads * a.each);
  switch (a.cache_dtype) {
    case 0: return launch_bounds_type<float, float>(a, groups, stream);
    case 1: return launch_bounds_type<__bf16, __bf16>(a, groups, stream);
    case 2: return launch_bounds_type<_Float16, _Float16>(a, groups, stream);
    case 3: return launch_bounds_type<Fp8, __bf16>(a, groups, stream);
    case 4: return launch_bounds_type<Int8, __bf16>(a, groups, stream);
    default: return launch_bounds_type<Fp4, __bf16>(a, groups, stream);
  }
}

hipError_t launch_select_pages(const SelectArgs& args, hipStream_t stream) {
  SelectArgs a = args;
  const int64_t rows = (int64_t)a.batch * a.heads;
  if (a.max_pages > a.count) {
    a.tiles = (int)((a.max_pages + kScorePages - 1) / kScorePages);
    const unsigned groups = (unsigned)(rows * a.tiles);
    switch (a.dtype) {
      case 0: launch_rank<float>(a, groups, stream); break;
      case 1: launch_rank<__bf16>(a, groups, stream); break;
      default: launch_rank<_Float16>(a, groups, stream); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.max_pages > 1024)
    page_select_kernel<1024><<<(unsigned)rows, 1024, 0, stream>>>(a);
  else
    page_select_kernel<256><<<(unsigned)rows, 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace fpx
