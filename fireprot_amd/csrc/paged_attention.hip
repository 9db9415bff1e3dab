// Attention over the paged cache: how its work is cut, the join of rows that
// work-groups shared, and the choice of kernel (paged_attention.hpp).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

constexpr int kJoinThreads = 256;
constexpr int kJoinFewRows = 256;   // rows that take several work-groups each

// One work-group per kChannels channels of a (sequence, query head) whose keys
// several shares covered: their (max, sum) become weights in LDS, 4-channel
// vectors of their outputs are summed kLanes shares at a time, and those sums in
// a fixed order.
template <typename Q, int D, int kChannels>
__global__ __launch_bounds__(kJoinThreads) void join_shares_kernel(PagedArgs a) {
  constexpr int kVecs = kChannels / 4;
  constexpr int kLanes = kJoinThreads / kVecs;
  constexpr int kEach = kPagedMaxGroups / kJoinThreads;
  __shared__ float weight[kPagedMaxGroups];
  __shared__ float red[2][kJoinThreads / kWave];
  __shared__ f32x4 sums[kLanes][kVecs];
  const int tid = threadIdx.x;
  const int q_heads = a.heads * a.group;
  const int b = blockIdx.x / (unsigned)q_heads, hq = blockIdx.x - b * q_heads;
  const int head = hq / a.group, qi = hq - head * a.group;
  const int tile = 16 * a.query_tiles;
  const int qtile = qi / tile;
  const int* info = a.row_info + ((int64_t)(b * a.heads + head) * a.qtiles + qtile) * 2;
  const int place = info[0], count = info[1];
  if (count <= 1) return;  // written by its only work-group
  // (lengths that another stream changes during the call could leave anything
  // here: nothing outside the places is read for it)
  if (place < 0 || place >= 2 * a.groups || count > a.groups - place / 2) return;
  // the row's part from work-group place / 2 + i
  auto part_row = [&](int i) -> int64_t {
    const int p = i == 0 ? place : (place / 2 + i) * 2;
    return (int64_t)p * a.tile_queries + (qi - qtile * tile);
  };
  const int vec = tid % kVecs, first = tid / kVecs;
  const float* column = a.part + blockIdx.y * kChannels + 4 * vec;
  f32x4 ahead = {0.0f, 0.0f, 0.0f, 0.0f};
  if (first < count) ahead = *reinterpret_cast<const f32x4*>(column + part_row(first) * D);

  float m[kEach], l[kEach];
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int c = tid + i * kJoinThreads;
    m[i] = -__builtin_inff();
    l[i] = 0.0f;
    if (c < count) {
      m[i] = a.part_ml[part_row(c) * 2];
      l[i] = a.part_ml[part_row(c) * 2 + 1];
    }
    // (a maximum is never NaN: a NaN score leaves it alone and makes the sum NaN)
    top = fmaxf(top, m[i]);
  }
  top = wave_max(top);
  if ((tid & 63) == 0) red[0][tid >> 6] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (int w = 1; w < kJoinThreads / kWave; ++w) top = fmaxf(top, red[0][w]);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float part = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float w = exp2_fast(m[i] - ref);
    weight[tid + i * kJoinThreads] = w;
    part += w * l[i];
  }
  part = wave_sum(part);
  if ((tid & 63) == 0) red[1][tid >> 6] = part;
  __syncthreads();
  float total = red[1][0];
#pragma unroll
  for (int i = 1; i < kJoinThreads / kWave; ++i) total += red[1][i];

  f32x4 acc = first < count ? ahead * weight[first] : ahead;
  for (int c = first + kLanes; c < count; c += kLanes)
    acc += *reinterpret_cast<const f32x4*>(column + part_row(c) * D) * weight[c];
  sums[first][vec] = acc;
  __syncthreads();
  if (tid < kChannels) {
    const float* sum = reinterpret_cast<const float*>(sums) + tid;
    const int used = count < kLanes ? count : kLanes;
    float x = 0.0f;
    for (int i = 0; i < used; ++i) x += sum[i * kChannels];
    static_cast<Q*>(a.out)[b * a.o_b + hq * a.o_h + blockIdx.y * kChannels + tid] =
        (Q)(x / total);
  }
  if (tid == 0 && blockIdx.y == 0 && a.lse)
    a.lse[blockIdx.x] =
        (top + __builtin_amdgcn_logf(total) - a.weight_shift) * 0.69314718055994531f;
}

// 32 channels to a work-group while there are few rows (32 rows of 256 shares:
// 5.5 us, 15 us with whole rows), whole rows otherwise (1024 rows of 7 shares:
// 4.9 us, 7.0 us in 32s).
template <typename Q, int D>
void launch_join_dim(const PagedArgs& a, unsigned rows, hipStream_t stream) {
  if (D > 32 && rows <= kJoinFewRows)
    join_shares_kernel<Q, D, 32><<<dim3(rows, D / 32), kJoinThreads, 0, stream>>>(a);
  else
    join_shares_kernel<Q, D, D><<<rows, kJoinThreads, 0, stream>>>(a);
}

template <typename Q>
void launch_join(const PagedArgs& a, unsigned rows, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: launch_join_dim<Q, 32>(a, rows, stream); break;
    case 64: launch_join_dim<Q, 64>(a, rows, stream); break;
    case 128: launch_join_dim<Q, 128>(a, rows, stream); break;
    default: launch_join_dim<Q, 256>(a, rows, stream); break;
  }
}

}  // namespace

PagedPlan plan_paged(int dtype, int cache_dtype, int64_t batch, int heads, int group, int head_dim,
                     int64_t max_length, int64_t window) {
  PagedPlan p{};
  p.query_tiles = group > 16 && head_dim <= 128 ? 2 : 1;
  p.qtiles = (group + 16 * p.query_tiles - 1) / (16 * p.query_tiles);
  p.tile_queries = group < 16 * p.query_tiles ? group : 16 * p.query_tiles;
  const int row_bytes = head_dim * (cache_dtype == 0 ? 4 : cache_dtype <= 2 ? 2 : 1);
  const int tile = cache_dtype == 0 ? 64 : 128;  // keys: one of PagedTraits::kTile a wave
  const int64_t rows = batch * heads * p.qtiles;
  const int64_t span = unit_limit(max_length, window, 1);
  if (rows < 1 || rows >= (1ll << 31) || (span + tile - 1) / tile >= (1ll << 31) / rows) return p;
  // Small calls: a unit of a row to a work-group, of kPagedUnit keys, or fewer
  // where that leaves CUs without work and the row is long enough to pay for the
  // join: longer than a unit, or of more than kPagedUnitBytes.  (8 sequences of
  // 500 keys, 4 heads: FP32 rows of 256 channels 33.8 us in one part, 15.8 in more;
  // BF16 rows of 128, 8 heads, 11.2 in one, 12.2 in two.  FP32 rows of 64, 2000
  // keys: 18.4 us in 128 work-groups, 14.0 in 256; BF16 rows of 128, 8 heads of
  // 1500 keys: 16.0 in 192, 17.0 in 384.)
  const bool splits = span > kPagedUnit || 2 * span * row_bytes > kPagedUnitBytes;
  int64_t unit = kPagedUnit;
  while (splits && unit > tile && rows * ((span + unit - 1) / unit) < kPagedEnough) unit /= 2;
  const int64_t each = (span + unit - 1) / unit;
  // This starts sooner than a share, but sequences shorter than the longest leave
  // work-groups idle: not beyond kPagedFixedBytes that the call may read.  How many
  // work-groups that makes is no matter.  Both cuts were timed on calls of 13 kinds (8
  // and 16 bits and FP32, heads of 32 to 256, lengths alike or from 1 on, 1 to 16
  // queries to a cache head) that read up to 134 MB: of 73 with 512 to 1151 work-groups
  // this took 0.957 of the shares' time in the mean (0.84 to 1.09), of 72 with 1152 and
  // more 0.916 (0.67 to 1.19, five above 1): INT8, 16 heads of 64, window 1000, 62
  // sequences, 2976 work-groups, 36.1 us and 38.8; FP8, 8 heads of 64, 16 queries each,
  // 98 sequences of 1000, 1568: 40.5 and 34.1.  32 queries to a cache head: 0.939 (0.77
  // to 1.17).  Below 512 it is 1.03 (0.86 to 1.27).  Past the limit a batch of few long
  // sequences gains most from shares: 8 of 1 to 8000 BF16 keys, 8 heads of 128, 262 MB:
  // 35.9 us, in shares 30.0.
  const bool small =
      each <= kPagedMaxGroups && rows * span * 2 * row_bytes <= kPagedFixedBytes;
  if ((each == 1 || small) && batch <= 65535) {
    p.unit = (int)unit;
    p.each = (int)each;
    p.split = each > 1;
    p.groups = (int)(rows * each);
    return p;
  }
  // Others: equal shares for as many work-groups to a CU as bring their waves'
  // tiles in flight to kPagedFlight bytes and its registers hold at once.  (One more
  // to a CU than they hold runs by itself when the others are done: 16 sequences of
  // 2001 to 16384 keys, 8 heads of 128, 32 queries, INT8: FP16 queries 80.1 us in 768
  // work-groups, 66.0 in 512; FP32 83.5 and 69.6; BF16, of which three fit, 65.0 and
  // 67.0.)
  p.unit = tile;
  p.split = 1;
  const int64_t each_cu = kPagedFlight / (2 * tile * row_bytes);
  const int64_t most = resident_groups(cache_dtype > 2 && dtype != 1, head_dim, p.query_tiles);
  const int64_t wanted = 256 * (each_cu < 1 ? 1 : each_cu > most ? most : each_cu);
  const int64_t units = rows * ((span + tile - 1) / tile);
  p.groups = (int)(units < wanted ? units : wanted);
  return p;
}

hipError_t launch_paged_attention(const PagedArgs& a, hipStream_t stream) {
  hipError_t e;
  switch (a.cache_dtype) {
    case 0: e = launch_paged_f32(a, stream); break;
    case 1: e = launch_paged_bf16(a, stream); break;
    case 2: e = launch_paged_f16(a, stream); break;
    case 3: e = launch_paged_fp8(a, stream); break;
    default: e = launch_paged_int8(a, stream); break;
  }
  if (e != hipSuccess || !a.split) return e;
  const unsigned rows = (unsigned)((int64_t)a.batch * a.heads * a.group);
  switch (a.dtype) {
    case 0: launch_join<float>(a, rows, stream); break;
    case 1: launch_join<__bf16>(a, rows, stream); break;
    default: launch_join<_Float16>(a, rows, stream); break;
  }
  return hipGetLastError();
}

}  // namespace fpx
