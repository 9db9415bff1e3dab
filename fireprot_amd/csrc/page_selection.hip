// Which pages of the paged cache a new token's queries can hardly do without
// (fpx_page_bounds, fpx_select_pages).
//
//   bounds[page][head] = (lo, hi), channel by channel over the page's keys
//   score(b, h, page)  = max over head h's queries of sum_c max(q_c lo_c, q_c hi_c),
//
// no less than any q . k of the page.  With q+ = max(q, 0) and q- = min(q, 0) it is, for
// finite bounds, a product, q+ . hi + q- . lo, which runs on the FP64 matrix cores: two
// pages next to each other in rank must come out in the same order whatever order the sum
// is taken in, and an FP32 sum of 128 terms is off by more than the step between scores
// where thousands of pages compete for the last place.  The sum is rounded to FP32 once;
// of pages alike the lower is preferred.
//
// What bounds the ranks is the bounds' way from memory.  16 sequences of equal length, 8
// cache heads of 128 BF16 channels with 8 queries each: 11.4 us with 384 pages a sequence,
// and 5.4 for each further 384 (25 MB, 4.7 TB/s).  The FP64 products are 3.0 of those 5.4
// (16 to 17 clocks each for 16 pages, 4 queries and 4 channels; the form with 16 queries
// takes 78: ranks in 49 us), the waves' exchange 0.4, and the conversions to FP64 go on
// beside them.  6 us are fixed: a launch, and three looks at memory of which each needs the
// one before (length, page, bounds).  626 to 2048 pages, 88 MB: 26.7 us by itself, of which
// uneven rows are 2, and 29 to 31 between the other kernels of a step.  4 queries to a head,
// 8 heads of one sequence of 2048 pages, 8.5 MB: 5.7 us, a launch being 3 to 4.
#include "cache_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

constexpr int kBoundsThreads = 256;
constexpr int64_t kBoundsMaxGroups = 1 << 22;  // work-groups of a launch
constexpr int kScoreThreads = 256;
constexpr int kScorePages = 64;    // of a work-group at a time
constexpr int kScoreGroups = 768;  // work-groups, about

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
  const uint32_t item = a.first + blockIdx.x;
  const uint32_t seq_head = item / (uint32_t)a.each;
  const int i = (int)(item - seq_head * (uint32_t)a.each);
  const int64_t b = seq_head / (uint32_t)a.heads;
  const int h = (int)(seq_head - (uint32_t)b * (uint32_t)a.heads);
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

// Pages of sequence b: 0 where its length does not fit the call.
__device__ __forceinline__ int pages_of(const SelectArgs& a, int b) {
  const KeyRange range = key_range(__builtin_amdgcn_readfirstlane(a.lengths[b]), a.max_length, 0);
  return (int)(((int64_t)range.end + (1 << a.page_shift) - 1) >> a.page_shift);
}

__device__ __forceinline__ int lane_of() {
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
}

// A query's sum_c max(q_c lo_c, q_c hi_c) term by term: each is the product with the bound
// that its sign asks for.  In the product form the other bound meets a zero, which makes NaN
// of an infinite one; here only a zero of the query's own does, a bound that is NaN itself,
// and a sum of both infinities.  (16 bytes of each bound at a time: 16 sequences of 1337
// pages that all have an infinite channel, 8 heads of 128, 8 queries each, are ranked and
// chosen from in 116 us, with 8 bytes in 195, without such a channel in 29.)
template <typename Q, typename T, int kDim>
__device__ __forceinline__ double score_by_terms(const Q* q, const T* edge) {
  constexpr int kStep = 16 / (int)sizeof(T);
  typedef Q QVec __attribute__((ext_vector_type(kStep)));
  typedef T TVec __attribute__((ext_vector_type(kStep)));
  double sum = 0.0;
  bool bad = false;
#pragma unroll 1
  for (int c = 0; c < kDim; c += kStep) {
    const QVec x = *reinterpret_cast<const QVec*>(q + c);
    const TVec lo = *reinterpret_cast<const TVec*>(edge + c);
    const TVec hi = *reinterpret_cast<const TVec*>(edge + kDim + c);
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const float xi = (float)x[i], l = (float)lo[i], u = (float)hi[i];
      sum = __builtin_fma((double)xi, (double)(xi > 0.0f ? u : l), sum);  // (exact products)
      const float other = (xi > 0.0f ? l : u) * (xi == 0.0f ? 0.0f : 1.0f);
      bad |= !(other == other);
    }
  }
  return bad ? __builtin_nan("") : sum;
}

// The ranks of a sequence's pages for one cache head, 64 at a time.  In a product the
// pages are the columns (one to a lane % 16), four queries the rows, and the lane groups
// (lane / 16) the four channels that are contracted.  Each of the four waves contracts a
// quarter of the channels for all 64 pages, so that it converts its part of the queries
// to FP64 once for them (8 VGPRs a channel of eight queries), and the waves' sums meet in
// LDS.  kTiles: fours of queries at a time; kMany: there are more than those.
template <int kTiles>
using Sums = double[2][4][kScorePages / 16][kTiles][kWave];

// rank(place), a reference, for the pages of tiles `tile`, `tile` + step and so on of the
// `total` pages of sequence b, cache head h.
template <typename Q, typename T, int kDim, int kTiles, bool kMany, typename Rank>
__device__ __forceinline__ void rank_tiles(const SelectArgs& a, Sums<kTiles>& sums, int b, int h,
                                           int total, int tile, int step, Rank rank) {
  constexpr int kEach = kDim / 16;  // channels of a lane
  constexpr int kParts = kScorePages / 16;
  typedef Q QVec __attribute__((ext_vector_type(kEach)));
  typedef T TVec __attribute__((ext_vector_type(kEach)));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int channel = (4 * wave + g) * kEach;
  const int32_t* table = a.table + b * a.table_b;
  int page[kParts], later[kParts];  // of the tile after this one, and of that after it
  TVec lo[kParts], hi[kParts];
  uint32_t inside = 0;  // bit p: the lane's page of part p is one of the cache
  auto look_up = [&](int at_tile, int* to) {  // (past the last page the last again)
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      to[p] = table[min(at_tile * kScorePages + 16 * p + col, total - 1)];
  };
  auto edge_of = [&](int number) {  // (of a page outside the cache the first's)
    return static_cast<const T*>(a.bounds) +
           ((int64_t)(page_valid(number, a.pages) ? number : 0) * a.heads + h) * 2 * kDim;
  };
  auto query_of = [&](int qi) {  // (rows past the head's last query have its first one again)
    return static_cast<const Q*>(a.q) + b * a.q_b +
           ((int64_t)h * a.group + (qi < a.group ? qi : 0)) * a.q_h;
  };
  auto load = [&](int p) {
    inside = (inside & ~(1u << p)) | (uint32_t)page_valid(page[p], a.pages) << p;
    const T* edge = edge_of(page[p]) + channel;
    lo[p] = *reinterpret_cast<const TVec*>(edge);
    hi[p] = *reinterpret_cast<const TVec*>(edge + kDim);
  };
  double above[kTiles][kEach], below[kTiles][kEach];  // max(q, 0) and min(q, 0)
  auto load_queries = [&](int q0) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const QVec x =
          *reinterpret_cast<const QVec*>(query_of(q0 + 4 * t + (lane & 3)) + channel);
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        above[t][j] = (double)greater((float)x[j], 0.0f);
        below[t][j] = (double)lesser((float)x[j], 0.0f);
      }
    }
  };
  // ---- tile by tile.  A part's bounds for the next tile are asked for as soon as this
  // tile's are used, and its page numbers a tile before that.  (Past the last tile the
  // last page is read again: the loads are not branched around, which would make every
  // wait one for all of them.)
  const int first_tile = tile;
  uint64_t unsure = 0;  // lanes with a score that is NaN
  look_up(tile, page);
  look_up(tile + step, later);
  if (!kMany) load_queries(0);
#pragma unroll
  for (int p = 0; p < kParts; ++p) load(p);
  for (int buffer = 0;; buffer ^= 1) {
    const uint32_t now_inside = inside;
#pragma unroll
    for (int p = 0; p < kParts; ++p) page[p] = later[p];
    look_up(tile + 2 * step, later);
    float best = -__builtin_inff();  // of the page part `wave`
    for (int q0 = 0;; q0 += 4 * kTiles) {
      const bool last = !kMany || q0 + 4 * kTiles >= a.group;
      if (kMany) load_queries(q0);
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        // (several sums, so that an instruction need not wait for the one before)
        double up[kTiles] = {}, down[kTiles] = {};
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const double u = (double)(float)hi[p][j], l = (double)(float)lo[p][j];
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            up[t] = __builtin_amdgcn_mfma_f64_4x4x4f64(above[t][j], u, up[t], 0, 0, 0);
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            down[t] = __builtin_amdgcn_mfma_f64_4x4x4f64(below[t][j], l, down[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) sums[buffer][wave][p][t][lane] = up[t] + down[t];
        if (last) load(p);
      }
      // (one barrier a turn: what the next one writes is the other buffer)
      __syncthreads();
      // (lane group g has query 4t + g)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        double x = sums[buffer][0][wave][t][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) x += sums[buffer][w][wave][t][lane];
        best = greater(best, (float)x);
      }
      if (last) break;
      buffer ^= 1;
    }
    best = greater(best, __shfl_xor(best, 16));
    best = greater(best, __shfl_xor(best, 32));
    const int at = tile * kScorePages + 16 * wave + col;
    if (g == 0 && at < total) {
      const bool forced = at < a.sinks || at >= total - a.recent;
      const bool ok = (now_inside >> wave) & 1;
      rank(at) = forced ? kForced : ok ? rank_of(best) : kNanRank;
    }
    unsure |= __ballot(!(best == best));
    tile += step;
    if (tile * kScorePages >= total) break;
  }
  // ---- pages that a NaN has ranked, by the terms of their scores: after all tiles, and
  // with the lane's number formed anew, so that it takes no registers in their loop (30
  // more there, and at 128 FP32 channels a work-group less to a CU)
  if (unsure == 0) return;
  const int me = lane_of(), my_group = me >> 4;
  for (tile = first_tile; tile * kScorePages < total; tile += step) {
    const int at = tile * kScorePages + 16 * wave + (me & 15);
    // (each lane reads what it has put itself)
    const uint32_t put = my_group == 0 && at < total ? rank(at) : 0u;
    const int number = table[min(at, total - 1)];
    const bool again =
        (uint32_t)__shfl((int)put, me & 15) == kNanRank && page_valid(number, a.pages);
    float best = -__builtin_inff();
    if (again)
      for (int qi = my_group; qi < a.group; qi += 4)
        best = greater(best,
                       (float)score_by_terms<Q, T, kDim>(query_of(qi), edge_of(number)));
    best = greater(best, __shfl_xor(best, 16));
    best = greater(best, __shfl_xor(best, 32));
    if (my_group == 0 && again) rank(at) = rank_of(best);
  }
}

template <typename Q, typename T, int kDim, int kTiles, bool kMany>
__global__ __launch_bounds__(kScoreThreads) void page_rank_kernel(SelectArgs a) {
  __shared__ Sums<kTiles> sums;
  // heads fastest: their bounds of a page lie next to each other
  const int h = (int)(blockIdx.x % (unsigned)a.heads);
  const int seq_chunk = (int)(blockIdx.x / (unsigned)a.heads);
  const int b = seq_chunk / a.chunks;
  const int tile = seq_chunk - b * a.chunks;
  const int total = pages_of(a, b);
  if (total <= a.count || tile * kScorePages >= total) return;  // (all taken: no ranks)
  uint32_t* ranks = a.ranks + ((int64_t)b * a.heads + h) * a.max_pages;
  rank_tiles<Q, T, kDim, kTiles, kMany>(a, sums, b, h, total, tile, a.chunks,
                                        [&](int at) -> uint32_t& { return ranks[at]; });
}

// Sum over the lanes up to and with this one: rows of 16 lanes by shifts, then the rows
// before by broadcasts of their last lanes.
__device__ __forceinline__ int wave_prefix(int x) {
  auto add = [](int v, int shifted) { return v + shifted; };
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));  // row_shr:1
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15
  x = add(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return x;
}

// The outputs of one (sequence, cache head) that need no ranks: the keys of the chosen
// pages, entries that name none, and the pages of a sequence that keeps them all.
__device__ __forceinline__ void select_plain(const SelectArgs& a, int row, int total,
                                             int threads) {
  const int b = row / a.heads;
  const int kept = total < a.count ? total : a.count;
  int32_t* index = a.index + (int64_t)row * a.count;
  int32_t* out = a.table_out + (int64_t)row * a.count;
  if (threadIdx.x == 0 && row == b * a.heads) {
    const KeyRange range = key_range(a.lengths[b], a.max_length, 0);
    a.lengths_out[b] = range.valid ? range.end - ((total - kept) << a.page_shift) : -1;
  }
  for (int i = threadIdx.x; i < a.count; i += threads) {
    if (i < kept && total > a.count) break;
    index[i] = i < kept ? i : -1;
    out[i] = i < kept ? a.table[b * a.table_b + i] : -1;
  }
}

// The `count` pages of highest rank of one (sequence, cache head), in the order of the
// sequence: the rank of the last of them is found byte by byte from the counts of each
// byte's values, then every thread lists its run of pages.  kKeys: pages of a thread,
// whose ranks (and numbers) it keeps in registers; 0: any number, read again every time.
// 128 rows of 626 to 2048 pages, 128 of them chosen, take 4.9 us, 8 rows of 2048 5.2: a
// launch, and eight barriers with a look into LDS between them (with one copy of the
// counts, and ranks read again in each turn, 9.1 and 8.9).  Rows too long for registers
// read them again: ranks and choice of 8 rows of 8192 pages are 22 us, of 8193 27, of
// 16384 65.
constexpr int kCopies = 8;  // of the counts: neighbouring pages' ranks begin alike
constexpr int kBins = 256 + 4;  // of a copy, which begins four banks after the one before

template <int kThreads>
struct SelectShared {
  __attribute__((aligned(16))) int counts[2][kCopies][kBins];
  uint32_t found[2];
  int wave_sum[2][kThreads / kWave];
};

template <int kThreads, int kKeys>
__device__ __forceinline__ void select_row(const SelectArgs& a, SelectShared<kThreads>& shared,
                                           int row, int total, const uint32_t* ranks) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* table = a.table + row / a.heads * a.table_b;
  int32_t* index = a.index + (int64_t)row * a.count;
  int32_t* out = a.table_out + (int64_t)row * a.count;
  const int per = kKeys > 0 ? kKeys : (total + kThreads - 1) / kThreads;
  const int begin = min(total, tid * per), end = min(total, begin + per);
  uint32_t held[kKeys > 0 ? kKeys : 1];
  int page[kKeys > 0 ? kKeys : 1];
#pragma unroll
  for (int k = 0; k < kKeys; ++k) {
    held[k] = begin + k < end ? ranks[begin + k] : 0;
    page[k] = begin + k < end ? table[begin + k] : 0;
  }
  // f(place, rank, number of the place among the thread's) for the thread's pages
  auto each = [&](auto f) {
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int k = 0; k < kKeys; ++k)
        if (begin + k < end) f(begin + k, held[k], k);
    } else {
      for (int i = begin; i < end; ++i) f(i, ranks[i], 0);
    }
  };
  auto clear = [&](int(*counts)[kBins]) {
    for (int i = tid; i < kCopies * kBins; i += kThreads) counts[0][i] = 0;
  };
  clear(shared.counts[0]);
  __syncthreads();
  uint32_t least = 0, mask = 0;  // the bytes found so far
  int wanted = a.count;          // pages among those that begin with them
  for (int turn = 0; turn < 4; ++turn) {
    const int shift = 24 - 8 * turn;
    int(*now)[kBins] = shared.counts[turn & 1];
    each([&](int, uint32_t r, int) {
      if (((r ^ least) & mask) == 0) atomicAdd(&now[lane % kCopies][(r >> shift) & 255], 1);
    });
    if (turn < 3) clear(shared.counts[(turn + 1) & 1]);
    __syncthreads();
    if (wave == 0) {
      // lane l has the values 255 - 4l to 252 - 4l
      typedef int Four __attribute__((ext_vector_type(4)));
      Four bins = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < kCopies; ++k)
        bins += *reinterpret_cast<const Four*>(&now[k][252 - 4 * lane]);
      const int own[4] = {bins[3], bins[2], bins[1], bins[0]};
      const int sum = bins[0] + bins[1] + bins[2] + bins[3];
      const int upto = wave_prefix(sum);
      int above = upto - sum;
      if (above < wanted && wanted <= upto) {
        int v = 0;
#pragma unroll
        for (int u = 0; u < 3; ++u)
          if (v == u && above + own[u] < wanted) {
            above += own[u];
            v = u + 1;
          }
        shared.found[0] = (uint32_t)(255 - 4 * lane - v);
        shared.found[1] = (uint32_t)(wanted - above);
      }
    }
    __syncthreads();
    least |= shared.found[0] << shift;
    wanted = (int)shared.found[1];
    mask |= 255u << shift;
  }
  // ---- pages of a higher rank, and the first `wanted` of that rank itself
  int own[2] = {0, 0}, before[2];
  each([&](int, uint32_t r, int) {
    own[0] += r > least;
    own[1] += r == least;
  });
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    before[w] = wave_prefix(own[w]);
    if (lane == kWave - 1) shared.wave_sum[w][wave] = before[w];
    before[w] -= own[w];
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    before[0] += shared.wave_sum[0][w];
    before[1] += shared.wave_sum[1][w];
  }
  each([&](int i, uint32_t r, int k) {
    if (r > least || (r == least && before[1] < wanted)) {
      const int to = before[0] + min(before[1], wanted);
      index[to] = i;
      out[to] = kKeys > 0 ? page[k] : table[i];
    }
    before[0] += r > least;
    before[1] += r == least;
  });
}

template <int kThreads, int kKeys>
__global__ __launch_bounds__(kThreads) void page_select_kernel(SelectArgs a) {
  __shared__ SelectShared<kThreads> shared;
  const int row = blockIdx.x;
  const int total = pages_of(a, row / a.heads);
  select_plain(a, row, total, kThreads);
  if (total > a.count)
    select_row<kThreads, kKeys>(a, shared, row, total, a.ranks + row * a.max_pages);
}

// Both in one launch, for rows of few pages: a work-group ranks them all, in LDS.
template <typename Q, typename T, int kDim, int kTiles, bool kMany>
__global__ __launch_bounds__(kScoreThreads) void page_rank_select_kernel(SelectArgs a) {
  __shared__ union {
    Sums<kTiles> sums;
    SelectShared<kScoreThreads> select;
  } shared;
  static_assert(kFewPages <= kScoreThreads, "a page to a thread");
  __shared__ uint32_t ranks[kFewPages];
  const int row = blockIdx.x;
  const int b = row / a.heads, h = row - b * a.heads;
  const int total = pages_of(a, b);
  select_plain(a, row, total, kScoreThreads);
  if (total <= a.count) return;
  rank_tiles<Q, T, kDim, kTiles, kMany>(a, shared.sums, b, h, total, 0, 1,
                                        [&](int at) -> uint32_t& { return ranks[at]; });
  __syncthreads();
  select_row<kScoreThreads, 1>(a, shared.select, row, total, ranks);
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

template <typename Q, typename T, int kDim>
void launch_rank_dim(const SelectArgs& a, unsigned groups, hipStream_t stream) {
  auto run = [&](auto tiles, auto many) {
    constexpr int kTiles = decltype(tiles)::value;
    constexpr bool kMany = decltype(many)::value;
    if (a.max_pages <= kFewPages)
      page_rank_select_kernel<Q, T, kDim, kTiles, kMany>
          <<<groups, kScoreThreads, 0, stream>>>(a);
    else
      page_rank_kernel<Q, T, kDim, kTiles, kMany><<<groups, kScoreThreads, 0, stream>>>(a);
  };
  using std::integral_constant;
  if (a.group <= 4)
    run(integral_constant<int, 1>(), std::false_type());
  else if (a.group <= 8)
    run(integral_constant<int, 2>(), std::false_type());
  else
    run(integral_constant<int, 2>(), std::true_type());
}

template <typename Q, typename T>
void launch_rank_type(const SelectArgs& a, unsigned groups, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: launch_rank_dim<Q, T, 32>(a, groups, stream); break;
    case 64: launch_rank_dim<Q, T, 64>(a, groups, stream); break;
    case 128: launch_rank_dim<Q, T, 128>(a, groups, stream); break;
    default: launch_rank_dim<Q, T, 256>(a, groups, stream); break;
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

hipError_t launch_page_bounds(const BoundsArgs& args, hipStream_t stream) {
  BoundsArgs a = args;
  const int64_t items = (int64_t)a.batch * a.heads * a.each;
  hipError_t e = hipSuccess;
  for (int64_t first = 0; first < items && e == hipSuccess; first += kBoundsMaxGroups) {
    a.first = (uint32_t)first;
    const int64_t left = items - first;
    const unsigned groups = (unsigned)(left < kBoundsMaxGroups ? left : kBoundsMaxGroups);
    switch (a.cache_dtype) {
      case 0: e = launch_bounds_type<float, float>(a, groups, stream); break;
      case 1: e = launch_bounds_type<__bf16, __bf16>(a, groups, stream); break;
      case 2: e = launch_bounds_type<_Float16, _Float16>(a, groups, stream); break;
      case 3: e = launch_bounds_type<Fp8, __bf16>(a, groups, stream); break;
      case 4: e = launch_bounds_type<Int8, __bf16>(a, groups, stream); break;
      default: e = launch_bounds_type<Fp4, __bf16>(a, groups, stream);
    }
  }
  return e;
}

hipError_t launch_select_pages(const SelectArgs& args, hipStream_t stream) {
  SelectArgs a = args;
  const int64_t rows = (int64_t)a.batch * a.heads;
  if (a.max_pages > a.count) {
    // work-groups of a row: one where it has few pages, otherwise as many as there are
    // tiles, but not many more in all than the card holds at once
    const int64_t tiles = (a.max_pages + kScorePages - 1) / kScorePages;
    const int64_t most = a.max_pages <= kFewPages ? 1 : (kScoreGroups + rows - 1) / rows;
    a.chunks = (int)(tiles < most ? tiles : most);
    const unsigned groups = (unsigned)(rows * a.chunks);
    switch (a.dtype) {
      case 0: launch_rank<float>(a, groups, stream); break;
      case 1: launch_rank<__bf16>(a, groups, stream); break;
      default: launch_rank<_Float16>(a, groups, stream); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.max_pages <= kFewPages) return e;
  }
  const unsigned groups = (unsigned)rows;
  if (a.max_pages <= 256)
    page_select_kernel<256, 1><<<groups, 256, 0, stream>>>(a);
  else if (a.max_pages <= 1024)
    page_select_kernel<256, 4><<<groups, 256, 0, stream>>>(a);
  else if (a.max_pages <= 2048)
    page_select_kernel<1024, 2><<<groups, 1024, 0, stream>>>(a);
  else if (a.max_pages <= 8192)
    page_select_kernel<1024, 8><<<groups, 1024, 0, stream>>>(a);
  else
    page_select_kernel<1024, 0><<<groups, 1024, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace fpx
