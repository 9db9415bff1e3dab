// Attention over the paged cache: how its work is cut, the join of a row's
// chunks, and the choice of kernel (paged_attention.hpp).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

constexpr int kCombineThreads = 256;
constexpr int kCombineAhead = 4;       // chunks of a thread
constexpr int kCombineFewRows = 256;   // rows that take several work-groups each

// One work-group per kChannels channels of a (sequence, query head): the
// chunks' (max, sum) become weights in LDS, 4-channel vectors of the chunks'
// outputs are summed kLanes chunks at a time, and those sums in a fixed order.
// The launch is a chain of waits and little else, so the first outputs are
// asked for before anything is known of the chunks' number (their places exist
// in every row; those past the row's chunks are never used).
template <typename Q, int D, int kChannels>
__global__ __launch_bounds__(kCombineThreads) void combine_chunks_kernel(PagedArgs a) {
  constexpr int kVecs = kChannels / 4;
  constexpr int kLanes = kCombineThreads / kVecs;
  __shared__ float weight[kMaxChunks];
  __shared__ float red[2][kCombineThreads / kWave];
  __shared__ f32x4 sums[kLanes][kVecs];
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int vec = tid % kVecs, first = tid / kVecs;
  const f32x4* parts = reinterpret_cast<const f32x4*>(a.part + (int64_t)row * a.splits * D +
                                                      blockIdx.y * kChannels) + vec;
  const float* ml = a.part_ml + (int64_t)row * a.splits * 2;
  f32x4 ahead[kCombineAhead];
#pragma unroll
  for (int i = 0; i < kCombineAhead; ++i) {
    const int c = first + i * kLanes;
    if (c < a.splits) ahead[i] = parts[(int64_t)c * (D / 4)];
  }
  float m = -__builtin_inff(), l = 0.0f;
  if (tid < a.splits) {
    m = ml[2 * tid];
    l = ml[2 * tid + 1];
  }
  const int q_heads = a.heads * a.group;
  const int b = row / q_heads, hq = row - b * q_heads;
  const int chunks = chunk_count(key_range(a.lengths[b], a.max_length, a.window), a.chunk);
  if (chunks <= 1) return;  // written by its only work-group
  if (tid >= chunks) {
    m = -__builtin_inff();
    l = 0.0f;
  }
  // (a maximum is never NaN: a NaN score leaves it alone and makes the sum NaN)
  float top = wave_max(m);
  if ((tid & 63) == 0) red[0][tid >> 6] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (int w = 1; w < kCombineThreads / kWave; ++w) top = fmaxf(top, red[0][w]);
  const float w = exp2_fast(m - (top == -__builtin_inff() ? 0.0f : top));
  weight[tid] = w;
  const float part = wave_sum(w * l);
  if ((tid & 63) == 0) red[1][tid >> 6] = part;
  __syncthreads();
  float total = red[1][0];
#pragma unroll
  for (int i = 1; i < kCombineThreads / kWave; ++i) total += red[1][i];

  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kCombineAhead; ++i) {
    const int c = first + i * kLanes;
    if (c < chunks) acc += ahead[i] * weight[c];
  }
  for (int c = first + kCombineAhead * kLanes; c < chunks; c += kLanes)
    acc += parts[(int64_t)c * (D / 4)] * weight[c];
  sums[first][vec] = acc;
  __syncthreads();
  if (tid < kChannels) {
    const float* column = reinterpret_cast<const float*>(sums) + tid;
    const int used = chunks < kLanes ? chunks : kLanes;
    float x = 0.0f;
    for (int i = 0; i < used; ++i) x += column[i * kChannels];
    static_cast<Q*>(a.out)[b * a.o_b + hq * a.o_h + blockIdx.y * kChannels + tid] =
        (Q)(x / total);
  }
  if (tid == 0 && blockIdx.y == 0 && a.lse)
    a.lse[row] = (top + __builtin_amdgcn_logf(total) - a.weight_shift) * 0.69314718055994531f;
}

// 32 channels to a work-group while there are few rows (32 rows of 256 chunks:
// 5.5 us, 15 us with whole rows), whole rows otherwise (1024 rows of 7 chunks:
// 4.9 us, 7.0 us in 32s).
template <typename Q, int D>
void launch_combine_dim(const PagedArgs& a, unsigned rows, hipStream_t stream) {
  if (D > 32 && rows <= kCombineFewRows)
    combine_chunks_kernel<Q, D, 32><<<dim3(rows, D / 32), kCombineThreads, 0, stream>>>(a);
  else
    combine_chunks_kernel<Q, D, D><<<rows, kCombineThreads, 0, stream>>>(a);
}

template <typename Q>
void launch_combine(const PagedArgs& a, unsigned rows, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: launch_combine_dim<Q, 32>(a, rows, stream); break;
    case 64: launch_combine_dim<Q, 64>(a, rows, stream); break;
    case 128: launch_combine_dim<Q, 128>(a, rows, stream); break;
    default: launch_combine_dim<Q, 256>(a, rows, stream); break;
  }
}

}  // namespace

PagedPlan plan_paged(int64_t batch, int heads, int group, int head_dim, int max_length,
                     int window) {
  PagedPlan p{};
  p.query_tiles = group > 16 && head_dim <= 128 ? 2 : 1;
  p.qtiles = (group + 16 * p.query_tiles - 1) / (16 * p.query_tiles);
  const int64_t rows = batch * heads * p.qtiles;
  const int64_t span = window > 0 && (int64_t)window + kKeyTile - 1 < max_length
                           ? (int64_t)window + kKeyTile - 1
                           : max_length;
  const int64_t unit = kKeyTile * 4;  // every wave a tile
  const int64_t wanted = (span * rows + kPagedGroups - 1) / kPagedGroups;
  int64_t chunk = (wanted + unit - 1) / unit * unit;
  const int64_t least = (span + kMaxChunks - 1) / kMaxChunks;
  if (chunk < least) chunk = (least + unit - 1) / unit * unit;
  if (chunk < 2 * unit) chunk = 2 * unit;
  if (chunk > (1 << 30)) chunk = 1 << 30;
  p.chunk = (int)chunk;
  p.splits = chunk_limit(max_length, window, p.chunk);
  if (p.splits < 1) p.splits = 1;
  p.blocks = rows * p.splits;
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
  if (e != hipSuccess || a.splits == 1) return e;
  const unsigned rows = (unsigned)((int64_t)a.batch * a.heads * a.group);
  switch (a.dtype) {
    case 0: launch_combine<float>(a, rows, stream); break;
    case 1: launch_combine<__bf16>(a, rows, stream); break;
    default: launch_combine<_Float16>(a, rows, stream); break;
  }
  return hipGetLastError();
}

}  // namespace fpx
