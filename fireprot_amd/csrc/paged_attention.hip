// Attention over the paged cache: how its work is cut, the join of a row's
// chunks, and the choice of kernel (paged_attention.hpp).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

namespace fpx {
namespace {

constexpr int kCombineThreads = 256;

// One work-group per (sequence, query head) of more than one chunk: the
// chunks' (max, sum) become weights in LDS, then 4-channel vectors of the
// chunks' outputs are summed, 256 / (D / 4) chunks at a time and in a fixed
// order.
template <typename Q, int D>
__global__ __launch_bounds__(kCombineThreads) void combine_chunks_kernel(PagedArgs a) {
  constexpr int kVecs = D / 4;
  constexpr int kLanes = kCombineThreads / kVecs;  // chunks at a time
  __shared__ float weight[kMaxChunks];
  __shared__ float red[kCombineThreads / kWave];
  __shared__ f32x4 sums[kLanes][kVecs];
  const int row = blockIdx.x;
  const int q_heads = a.heads * a.group;
  const int b = row / q_heads, hq = row - b * q_heads;
  const int chunks = chunk_count(key_range(a.lengths[b], a.max_length, a.window), a.chunk);
  if (chunks <= 1) return;  // written by its only work-group

  const float* ml = a.part_ml + (int64_t)row * a.splits * 2;
  const int tid = threadIdx.x;
  const bool has = tid < chunks;
  const float m = has ? ml[2 * tid] : -__builtin_inff();
  const float l = has ? ml[2 * tid + 1] : 0.0f;
  // (a NaN maximum cannot be: a NaN score leaves it out and makes the sum NaN)
  float top = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int w = 1; w < kCombineThreads / kWave; ++w) top = fmaxf(top, red[w]);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  const float w = exp2_fast(m - ref);
  weight[tid] = w;
  __syncthreads();
  const float part = wave_sum(has ? w * l : 0.0f);
  if ((tid & 63) == 0) red[tid >> 6] = part;
  __syncthreads();
  float total = red[0];
#pragma unroll
  for (int i = 1; i < kCombineThreads / kWave; ++i) total += red[i];

  const int vec = tid % kVecs, first = tid / kVecs;
  const f32x4* parts = reinterpret_cast<const f32x4*>(a.part + (int64_t)row * a.splits * D) + vec;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = first; c < chunks; c += kLanes) acc += parts[(int64_t)c * kVecs] * weight[c];
  sums[first][vec] = acc;
  __syncthreads();
  if (first == 0) {
#pragma unroll
    for (int i = 1; i < kLanes; ++i) acc += sums[i][vec];
    Q* out = static_cast<Q*>(a.out) + b * a.o_b + hq * a.o_h + 4 * vec;
    const float scale = 1.0f / total;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (Q)(acc[i] * scale);
  }
  if (tid == 0 && a.lse)
    a.lse[row] = (top + __builtin_amdgcn_logf(total) - a.weight_shift) * 0.69314718055994531f;
}

template <typename Q>
void launch_combine(const PagedArgs& a, unsigned rows, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: combine_chunks_kernel<Q, 32><<<rows, kCombineThreads, 0, stream>>>(a); break;
    case 64: combine_chunks_kernel<Q, 64><<<rows, kCombineThreads, 0, stream>>>(a); break;
    case 128: combine_chunks_kernel<Q, 128><<<rows, kCombineThreads, 0, stream>>>(a); break;
    default: combine_chunks_kernel<Q, 256><<<rows, kCombineThreads, 0, stream>>>(a); break;
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
  const unsigned blocks = (unsigned)((int64_t)a.batch * a.heads * a.qtiles * a.splits);
  hipError_t e;
  switch (a.cache_dtype) {
    case 0: e = launch_paged_f32(a, blocks, stream); break;
    case 1: e = launch_paged_bf16(a, blocks, stream); break;
    case 2: e = launch_paged_f16(a, blocks, stream); break;
    case 3: e = launch_paged_fp8(a, blocks, stream); break;
    default: e = launch_paged_int8(a, blocks, stream); break;
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
