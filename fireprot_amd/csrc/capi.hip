// C-ABI entry points (declared in include/fireprot_amd.h).
//
// Every entry validates sizes and pointers on the host first (status 2 / 3 /
// 4, before any device pointer is touched), then enqueues on the caller's
// stream and returns the launch status.  Nothing here allocates or
// synchronises.
#include "fireprot_amd.h"

#include "common.hpp"
#include "kernels.hpp"
#include "overlap.hpp"

#include <cmath>
#include <mutex>

namespace {

using fpx::round_up;

bool aligned(const void* p, uintptr_t bytes) {
  return p != nullptr && reinterpret_cast<uintptr_t>(p) % bytes == 0;
}
bool aligned_or_null(const void* p, uintptr_t bytes) {
  return p == nullptr || reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

constexpr int kMaxN = 4096;
constexpr int kQueryTile = 128;  // attention query tile: every block extent pads to it

size_t elem_bytes(int dtype) { return dtype == FPX_BF16 ? 2 : 4; }

// Workspace segments of the block, all 256-byte aligned, element size e
// (4 for FPX_F32, 2 for FPX_BF16; the mask bias is always float):
//   qh, kh [n][4][np][32]; vt [n][4][32][np] (BF16: [n][4][np / 32][32][32],
//   tile-major); gs [n][np][128]; og [n][n][128] (BF16: head-major [4][n][n][32]);
//   tri_bias [4][np][np] (FP32: fragment order, twice: as is and scaled by
//   log2(e); BF16: bias_frag_index_bf16, once); mbias [n][np] float;
//   tile flags [n][kTileFlagParts * kTileFlagWords] uint32, then the
//   kMagnitudeWords words of the magnitude record; scales [3][n][4][np / 32]
//   float (the plane layout's per-tile inverse scales of q, k and v^T); FP32
//   only: the constant-mask rows' weights and chunk list (AttnArgs::const_m,
//   const_l, const_p: kConstListWord words, the list in room for twice the
//   ceil(n / kConstRows) chunk indices it may hold, l [4][np] float, the planes
//   [4][np / 32][ceil(n / 32)] x 4 KB).
// FP32 blocks hold q, k and v^T in the fp16 plane layout (ProjArgs), in the
// same bytes as FP32 values.
struct BlockWorkspace {
  size_t qh, kh, vt, gs, og, bias, mbias, flags, scales, cw_m, cw_l, cw_p, total;
};

BlockWorkspace block_workspace(int n, int dtype) {
  const size_t np = (size_t)round_up(n, kQueryTile);
  const size_t e = elem_bytes(dtype);
  auto seg = [](size_t bytes) { return (size_t)round_up((int64_t)bytes, 256); };
  const size_t qkv = seg((size_t)n * fpx::kHeads * np * fpx::kHeadDim * e);
  const size_t g = seg((size_t)n * n * fpx::kHidden * e);
  const size_t gate = seg((size_t)n * np * fpx::kHidden * e);
  const size_t bias = seg((size_t)fpx::kHeads * np * np * e * (dtype == FPX_F32 ? 2 : 1));
  const size_t mb = seg((size_t)n * np * sizeof(float));
  const size_t fl = seg(((size_t)n * fpx::kTileFlagParts * fpx::kTileFlagWords +
                        fpx::kMagnitudeWords) * sizeof(uint32_t));
  BlockWorkspace w{};
  w.qh = 0;
  w.kh = w.qh + qkv;
  w.vt = w.kh + qkv;
  w.gs = w.vt + qkv;
  w.og = w.gs + gate;
  w.bias = w.og + g;
  w.mbias = w.bias + bias;
  w.flags = w.mbias + mb;
  w.scales = w.flags + fl;
  const size_t cw_m = w.scales + seg((size_t)3 * n * fpx::kHeads * (np / 32) * sizeof(float));
  w.cw_m = cw_m;
  if (dtype == FPX_F32) {
    const size_t nkt = (size_t)(n + 31) / 32;
    const size_t chunks = (size_t)(n + fpx::kConstRows - 1) / fpx::kConstRows;
    w.cw_l = cw_m + seg((fpx::kConstListWord + 2 * chunks) * sizeof(uint32_t));
    w.cw_p = w.cw_l + seg((size_t)fpx::kHeads * np * sizeof(float));
    w.total = w.cw_p + (size_t)fpx::kHeads * (np / 32) * nkt * 4096;
  } else {
    w.cw_l = w.cw_p = w.total = cw_m;
  }
  return w;
}

bool block_dims_ok(int n, int c, int heads, int head_dim, int dtype) {
  return (dtype == FPX_F32 || dtype == FPX_BF16) && c == fpx::kChannels &&
         heads == fpx::kHeads && head_dim == fpx::kHeadDim && n >= 1 && n <= kMaxN;
}

int status(hipError_t e) { return e == hipSuccess ? FPX_OK : (int)e; }

struct BlockPointers {
  char *qh, *kh, *vt, *gs, *og, *tri;
  float* mbias;
  uint32_t* flags;
  uint32_t* magnitudes;
  float* scales;
  uint32_t* const_m;  // FP32 only (else null), as const_l and const_p
  float* const_l;
  uint8_t* const_p;
  int np;
};

BlockPointers block_pointers(void* workspace, int n, int dtype) {
  const BlockWorkspace ws = block_workspace(n, dtype);
  char* base = static_cast<char*>(workspace);
  BlockPointers p{};
  p.qh = base + ws.qh;
  p.kh = base + ws.kh;
  p.vt = base + ws.vt;
  p.gs = base + ws.gs;
  p.og = base + ws.og;
  p.tri = base + ws.bias;
  p.mbias = reinterpret_cast<float*>(base + ws.mbias);
  p.flags = reinterpret_cast<uint32_t*>(base + ws.flags);
  p.magnitudes = p.flags + (size_t)n * fpx::kTileFlagParts * fpx::kTileFlagWords;
  p.scales = reinterpret_cast<float*>(base + ws.scales);
  if (dtype == FPX_F32) {
    p.const_m = reinterpret_cast<uint32_t*>(base + ws.cw_m);
    p.const_l = reinterpret_cast<float*>(base + ws.cw_l);
    p.const_p = reinterpret_cast<uint8_t*>(base + ws.cw_p);
  }
  p.np = (int)round_up(n, kQueryTile);
  return p;
}

int check_workspace(int n, int dtype, const void* workspace, size_t workspace_bytes) {
  if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
  if (workspace_bytes < block_workspace(n, dtype).total) return FPX_ERR_WORKSPACE;
  return FPX_OK;
}

template <typename T>
T* as(char* p) {
  return reinterpret_cast<T*>(p);
}

// The FP32 block's attention operands in its workspace.
fpx::AttnArgs block_attention_args(const BlockPointers& w, int n, bool has_mask) {
  fpx::AttnArgs a{};
  a.q = as<float>(w.qh);
  a.k = as<float>(w.kh);
  a.v = as<float>(w.vt);
  a.mbias = w.mbias;
  a.mb_stride = w.np;
  a.bias = as<float>(w.tri);
  a.bias_l2 = as<float>(w.tri) + (size_t)fpx::kHeads * w.np * w.np;
  a.bias_stride = w.np;
  a.bias_rows = w.np;
  a.gate = as<float>(w.gs);
  a.out = as<float>(w.og);
  a.tile_flags = w.flags;
  a.magnitudes = w.magnitudes;
  a.scales = w.scales;
  a.const_m = w.const_m;
  a.const_l = w.const_l;
  a.const_p = w.const_p;
  a.has_mask = has_mask;
  a.batch = n;
  a.n = n;
  a.np = w.np;
  return a;
}

// has_mask = 0: the prepare stage ran without a mask.
int attend_stage(int dtype, int n, int has_mask, void* workspace, size_t workspace_bytes,
                 void* stream) {
  if (!block_dims_ok(n, fpx::kChannels, fpx::kHeads, fpx::kHeadDim, dtype)) return FPX_ERR_DIMS;
  if (int rc = check_workspace(n, dtype, workspace, workspace_bytes)) return rc;
  const BlockPointers w = block_pointers(workspace, n, dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FPX_BF16) {
    fpx::Bf16AttnArgs a{};
    a.q = as<__bf16>(w.qh);
    a.k = as<__bf16>(w.kh);
    a.v = as<__bf16>(w.vt);
    a.mbias = w.mbias;
    a.tile_flags = w.flags;
    a.bias = as<__bf16>(w.tri);
    a.gate = as<__bf16>(w.gs);
    a.out = as<__bf16>(w.og);
    a.batch = n;
    a.n = n;
    a.np = w.np;
    return status(fpx::launch_attention_bf16(a, s));
  }
  return status(fpx::launch_attention_split(fpx::kAttnBlock,
                                            block_attention_args(w, n, has_mask != 0), s));
}

// Output projection into dz, or added to dz (accumulate), in z's frame.
int finish_stage(int dtype, const void* w_o, const void* b_o, int n, int ending, void* dz,
                 int64_t dz_stride0, int64_t dz_stride1, void* workspace, size_t workspace_bytes,
                 void* stream, int accumulate) {
  if (!block_dims_ok(n, fpx::kChannels, fpx::kHeads, fpx::kHeadDim, dtype)) return FPX_ERR_DIMS;
  if (ending != 0 && ending != 1) return FPX_ERR_DIMS;
  if (dz_stride0 < 0 || dz_stride1 < 0) return FPX_ERR_DIMS;
  if (!aligned(w_o, 16) || !aligned(dz, 16) || !aligned_or_null(b_o, 2)) return FPX_ERR_POINTER;
  if (dtype == FPX_F32 && !aligned_or_null(b_o, 4)) return FPX_ERR_POINTER;
  if (int rc = check_workspace(n, dtype, workspace, workspace_bytes)) return rc;
  const BlockPointers w = block_pointers(workspace, n, dtype);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t os_i = ending ? dz_stride1 : dz_stride0;
  const int64_t os_j = ending ? dz_stride0 : dz_stride1;
  if (dtype == FPX_BF16) {
    fpx::Bf16ProjArgs o{};
    o.x = as<__bf16>(w.og);  // head-major [4][n][n][32]
    o.xs_i = (int64_t)n * fpx::kHeadDim;
    o.xs_j = fpx::kHeadDim;
    o.xs_h = (int64_t)n * n * fpx::kHeadDim;
    o.rows_i = n;
    o.rows_j = n;
    o.span_j = n;
    o.w[0] = static_cast<const __bf16*>(w_o);
    o.bias_vec = static_cast<const __bf16*>(b_o);
    o.out = static_cast<__bf16*>(dz);
    o.os_i = os_i;
    o.os_j = os_j;
    o.accumulate = accumulate;
    return status(fpx::launch_projection_bf16(fpx::kProjOut, o, s));
  }
  fpx::ProjArgs o{};
  o.x = as<float>(w.og);
  o.xs_i = (int64_t)n * fpx::kHidden;
  o.xs_j = fpx::kHidden;
  o.rows_i = n;
  o.rows_j = n;
  o.span_j = n;
  o.w[0] = static_cast<const float*>(w_o);
  o.b_g = static_cast<const float*>(b_o);
  o.out = static_cast<float*>(dz);
  o.os_i = os_i;
  o.os_j = os_j;
  o.accumulate = accumulate;
  return status(fpx::launch_projection(fpx::kProjOut, o, s));
}

// The whole block: prepare, attend, then the output projection written to or
// (accumulate) added to dz.
int block_impl(int dtype, const void* z, int64_t z_stride0, int64_t z_stride1, const float* mask,
               int64_t m_stride0, int64_t m_stride1, const void* ln_w, const void* ln_b,
               float eps, const void* w_qkvg, const void* b_g, const void* w_bias,
               const void* w_o, const void* b_o, float mask_inf, int n, int c, int heads,
               int head_dim, int ending, void* dz, int64_t dz_stride0, int64_t dz_stride1,
               void* workspace, size_t workspace_bytes, void* stream, int accumulate) {
  if (!block_dims_ok(n, c, heads, head_dim, dtype)) return FPX_ERR_DIMS;
  if (ending != 0 && ending != 1) return FPX_ERR_DIMS;
  if (dz_stride0 < 0 || dz_stride1 < 0) return FPX_ERR_DIMS;
  if (!aligned(w_o, 16) || !aligned(dz, 16) || !aligned_or_null(b_o, 2)) return FPX_ERR_POINTER;
  if (dtype == FPX_F32 && !aligned_or_null(b_o, 4)) return FPX_ERR_POINTER;
  int rc = fpx_tri_attn_prepare(dtype, z, z_stride0, z_stride1, mask, m_stride0, m_stride1, ln_w,
                                ln_b, eps, w_qkvg, b_g, w_bias, mask_inf, n, ending, workspace,
                                workspace_bytes, stream);
  if (rc) return rc;
  rc = attend_stage(dtype, n, mask != nullptr, workspace, workspace_bytes, stream);
  if (rc) return rc;
  return finish_stage(dtype, w_o, b_o, n, ending, dz, dz_stride0, dz_stride1, workspace,
                      workspace_bytes, stream, accumulate);
}

// Workspace of fpx_attn_strided, 256-byte aligned segments:
//   bias [4][np][np] float in fragment order, twice (as is, scaled by log2(e));
//   mbias [batch][np] float; tile flags [batch][kTileFlagParts * kTileFlagWords] uint32;
//   q, k and v planes [batch][4] slices of np * 128 bytes each; their scales
//   [3][batch][4][np / 32] float; the magnitude record (kMagnitudeWords) and
//   the staging's per-work-group maxima (3 floats per group of 4 tiles).
struct StridedWorkspace {
  size_t bias, bias_l2, mbias, flags, qp, kp, vp, scales, magnitudes, partial, total;
};

StridedWorkspace strided_workspace(int batch, int n) {
  const size_t np = (size_t)round_up(n, kQueryTile);
  auto seg = [](size_t bytes) { return (size_t)round_up((int64_t)bytes, 256); };
  StridedWorkspace w{};
  w.bias = 0;
  w.bias_l2 = seg((size_t)fpx::kHeads * np * np * sizeof(float));
  w.mbias = 2 * w.bias_l2;
  w.flags = w.mbias + seg((size_t)batch * np * sizeof(float));
  w.qp = w.flags + seg((size_t)batch * fpx::kTileFlagParts * fpx::kTileFlagWords *
                        sizeof(uint32_t));
  const size_t planes = seg((size_t)batch * fpx::kHeads * np * 128);
  w.kp = w.qp + planes;
  w.vp = w.kp + planes;
  w.scales = w.vp + planes;
  w.magnitudes = w.scales + seg(3 * (size_t)batch * fpx::kHeads * (np / 32) * sizeof(float));
  w.partial = w.magnitudes + seg(fpx::kMagnitudeWords * sizeof(uint32_t));
  const size_t groups = (3 * (size_t)batch * fpx::kHeads * (np / 32) + 3) / 4;
  w.total = w.partial + seg(3 * groups * sizeof(float));
  return w;
}

// Workspace of fpx_tri_mul, 256-byte aligned segments: a and b, 128 np^2
// floats each (channel-blocked [8][np / 32][np][16][32]); x blocked
// [n][np / 32][128][32] float; the row maxima of a and b [2][128][np] uint32.
struct TriMulWorkspace {
  size_t pa, pb, x, rowmax, total;
};

TriMulWorkspace trimul_workspace(int n) {
  const size_t np = (size_t)round_up(n, kQueryTile);
  auto seg = [](size_t bytes) { return (size_t)round_up((int64_t)bytes, 256); };
  TriMulWorkspace w{};
  w.pa = 0;
  w.pb = seg((size_t)fpx::kChannels * np * np * sizeof(float));
  w.x = 2 * w.pb;
  w.rowmax = w.x + seg((size_t)n * np * fpx::kChannels * sizeof(float));
  w.total = w.rowmax + seg(2 * (size_t)fpx::kChannels * np * sizeof(uint32_t));
  return w;
}

// Workspace of fpx_transition: the fused kernel's weight planes (16 chunks
// of 48 KB), folded biases [2][512] float and its plane exponents (5 KB),
// whatever the number of rows.
constexpr size_t kTransitionPlanesBytes = 16 * 48 * 1024;
constexpr size_t kTransitionFusedBytes = kTransitionPlanesBytes + 2 * 512 * sizeof(float) + 5120;
size_t transition_workspace(int64_t /*rows*/) { return kTransitionFusedBytes; }

// A [batch][4][n][32] operand with channel stride 1 the strided attention
// kernel can read: non-negative strides that keep 16-byte rows aligned, and
// (for K and V) a (b, h) slice that a buffer descriptor covers.
bool strided_operand_ok(const int64_t s[3], int n, bool slice) {
  for (int d = 0; d < 3; ++d)
    if (s[d] < 0 || s[d] % 4 != 0) return false;
  return !slice || ((int64_t)(n - 1) * s[2] + fpx::kHeadDim) * 4 < 0x7fffffffll;
}

// Scratch of fpx_tri_attn_block_noalloc: the block workspace of N <= 128
// (block_workspace(128, FPX_F32).total = 42565888 bytes, every smaller N and
// the BF16 block need less), held by each GPU the library runs on until the
// process ends.  Host code never passes `scratch` itself (its host-side name
// is no device address): it uses the per-device address that
// hipGetSymbolAddress returns.
constexpr int kNoAllocMaxN = 128;
constexpr size_t kNoAllocScratchBytes = 41u << 20;
static __device__ __align__(256) uint8_t scratch[kNoAllocScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex scratch_mutex;
void* scratch_ptr[kMaxDevices] = {};

// The current device's address of `scratch`, looked up once per device with
// that device current; nullptr (and the HIP status in *err) on failure.
void* device_scratch(hipError_t* err) {
  int device = 0;
  *err = hipGetDevice(&device);
  if (*err != hipSuccess) return nullptr;
  if (device < 0 || device >= kMaxDevices) {
    *err = hipErrorInvalidDevice;
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(scratch_mutex);
  if (scratch_ptr[device] == nullptr) {
    void* ptr = nullptr;
    *err = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (*err != hipSuccess) return nullptr;
    scratch_ptr[device] = ptr;
  }
  return scratch_ptr[device];
}

// ---- paged key-value cache: what its entries share

bool is_coded(int dtype) {
  return dtype == FPX_F8E4M3 || dtype == FPX_I8 || dtype == FPX_F4E2M1;
}

uintptr_t type_bytes(int dtype) {
  return dtype == FPX_F32 ? 4 : dtype == FPX_BF16 || dtype == FPX_F16 ? 2 : 1;
}

bool row_type_ok(int dtype) {
  return dtype == FPX_F32 || dtype == FPX_BF16 || dtype == FPX_F16;
}

// Status of a cache's sizes, and its page shift.
int cache_dims(int cache_dtype, int64_t pages, int heads, int page_size, int head_dim,
               int* page_shift) {
  if (!row_type_ok(cache_dtype) && !is_coded(cache_dtype)) return FPX_ERR_DIMS;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return FPX_ERR_DIMS;
  if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1))) return FPX_ERR_DIMS;
  if (heads < 1 || heads > 65535 || pages < 1 || pages > 0x7fffffff) return FPX_ERR_DIMS;
  *page_shift = __builtin_ctz((unsigned)page_size);
  return FPX_OK;
}

bool cache_pointers_ok(int cache_dtype, const void* k, const void* v, const void* k_scale,
                       const void* v_scale) {
  if (!aligned(k, 16) || !aligned(v, 16)) return false;
  return !is_coded(cache_dtype) || (aligned(k_scale, 16) && aligned(v_scale, 16));
}

// A cache's k, v and scales (empty for plain types).
struct CacheBlocks {
  fpx::MemoryBlock block[4];
};

CacheBlocks cache_blocks(int cache_dtype, const void* k, const void* v, const void* k_scale,
                         const void* v_scale, int64_t pages, int heads, int page_size,
                         int head_dim) {
  // (below 2^59; the channels of each row are an axis of their own, as the product of
  // both could pass 2^63)
  const int64_t rows = pages * heads * page_size, e = (int64_t)type_bytes(cache_dtype);
  const bool coded = is_coded(cache_dtype), fp4 = cache_dtype == FPX_F4E2M1;
  const int64_t row = fp4 ? head_dim / 2 : head_dim;  // elements
  const int64_t scale = fp4 ? head_dim / 32 : 4;      // bytes of a row's scales
  return {{{k, e, fpx::MemoryAxis{rows, row}, fpx::MemoryAxis{row, 1}},
           {v, e, fpx::MemoryAxis{rows, row}, fpx::MemoryAxis{row, 1}},
           {coded ? k_scale : nullptr, scale, fpx::MemoryAxis{rows, 1}},
           {coded ? v_scale : nullptr, scale, fpx::MemoryAxis{rows, 1}}}};
}

bool meets_cache(const fpx::MemoryBlock& x, const CacheBlocks& cache) {
  for (const fpx::MemoryBlock& b : cache.block)
    if (fpx::blocks_meet(x, b)) return true;
  return false;
}

int cache_impl(bool read, int row_dtype, int cache_dtype, const void* k, int64_t k_st,
               int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots,
               int64_t tokens, const void* cache_k, const void* cache_v, const void* k_scale,
               const void* v_scale, int64_t pages, int heads, int page_size, int head_dim,
               void* stream) {
  fpx::CacheArgs a{};
  const int rc = cache_dims(cache_dtype, pages, heads, page_size, head_dim, &a.page_shift);
  if (rc != FPX_OK) return rc;
  if (!row_type_ok(row_dtype)) return FPX_ERR_DIMS;
  if (k_st < 0 || k_sh < 0 || v_st < 0 || v_sh < 0) return FPX_ERR_DIMS;
  if (tokens < 0 || tokens > 0x7fffffff || tokens * heads > 0x7fffffff) return FPX_ERR_DIMS;
  if (tokens == 0) return FPX_OK;
  const uintptr_t elem = type_bytes(row_dtype);
  if (!aligned(k, elem) || !aligned(v, elem) || !aligned(slots, 8) ||
      !cache_pointers_ok(cache_dtype, cache_k, cache_v, k_scale, v_scale))
    return FPX_ERR_POINTER;
  {  // what is written meets nothing else
    using fpx::MemoryAxis;
    const CacheBlocks cache = cache_blocks(cache_dtype, cache_k, cache_v, k_scale, v_scale, pages,
                                           heads, page_size, head_dim);
    const fpx::MemoryBlock rows[2] = {
        {k, (int64_t)elem, MemoryAxis{tokens, k_st}, MemoryAxis{heads, k_sh},
         MemoryAxis{head_dim, 1}},
        {v, (int64_t)elem, MemoryAxis{tokens, v_st}, MemoryAxis{heads, v_sh},
         MemoryAxis{head_dim, 1}}};
    const fpx::MemoryBlock where(slots, 8, MemoryAxis{tokens, 1});
    if (meets_cache(rows[0], cache) || meets_cache(rows[1], cache)) return FPX_ERR_DIMS;
    if (read) {
      if (fpx::blocks_meet(rows[0], rows[1])) return FPX_ERR_DIMS;
      for (const fpx::MemoryBlock& r : rows)
        if (fpx::block_meets_itself(r) || fpx::blocks_meet(r, where)) return FPX_ERR_DIMS;
    } else {
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
          if (fpx::blocks_meet(cache.block[i], cache.block[j])) return FPX_ERR_DIMS;
      if (meets_cache(where, cache)) return FPX_ERR_DIMS;
    }
  }
  a.rows[0] = k;
  a.rows[1] = v;
  a.stride_t[0] = k_st;
  a.stride_t[1] = v_st;
  a.stride_h[0] = k_sh;
  a.stride_h[1] = v_sh;
  a.slots = slots;
  a.cache[0] = const_cast<void*>(cache_k);
  a.cache[1] = const_cast<void*>(cache_v);
  a.scale[0] = const_cast<void*>(k_scale);
  a.scale[1] = const_cast<void*>(v_scale);
  a.tokens = tokens;
  a.pages = pages;
  a.heads = heads;
  a.head_dim = head_dim;
  a.row_dtype = row_dtype;
  a.cache_dtype = cache_dtype;
  return status(fpx::launch_cache(a, read, static_cast<hipStream_t>(stream)));
}

constexpr int64_t kPagedMaxRows = 1 << 20;  // (sequence, query head): the join's grid

// The cut of a call's work, groups = 0 for unsupported sizes.
fpx::PagedPlan paged_plan(int dtype, int cache_dtype, int64_t batch, int q_heads, int heads,
                          int head_dim, int64_t max_length, int64_t window) {
  const fpx::PagedPlan none{};
  if (!row_type_ok(cache_dtype) && !is_coded(cache_dtype)) return none;
  if (batch < 0 || batch > kPagedMaxRows || heads < 1 || q_heads < heads || q_heads % heads ||
      q_heads > kPagedMaxRows || batch * q_heads > kPagedMaxRows)
    return none;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return none;
  if (max_length < 0 || max_length >= (1 << 30) || window < 0) return none;
  return fpx::plan_paged(dtype, cache_dtype, batch < 1 ? 1 : batch, heads, q_heads / heads,
                         head_dim, max_length, window < (1 << 30) ? window : 0);
}

// Places of the rows' shares, their (max, sum), and the rows' places.
struct PagedWorkspace {
  size_t ml, info, total;
};

PagedWorkspace paged_workspace(const fpx::PagedPlan& p, int64_t batch, int heads, int head_dim) {
  const int64_t places = (int64_t)p.groups * 2 * p.tile_queries;
  PagedWorkspace w{};
  w.ml = (size_t)round_up(places * head_dim * 4, 256);
  w.info = w.ml + (size_t)round_up(places * 8, 256);
  w.total = w.info + (size_t)(batch * heads * p.qtiles * 8);
  return w;
}

int paged_impl(int dtype, int cache_dtype, const void* q, int64_t q_sb, int64_t q_sh,
               const void* cache_k, const void* cache_v, const void* k_scale, const void* v_scale,
               int64_t pages, int heads, int page_size, int head_dim, const int32_t* block_table,
               int64_t table_sb, int64_t table_sh, int64_t table_pages, const int32_t* lengths,
               int64_t batch, int q_heads, int64_t max_length, int64_t window, float scale,
               void* out, int64_t o_sb, int64_t o_sh, float* lse, void* workspace,
               size_t workspace_bytes, void* stream) {
  fpx::PagedArgs a{};
  const int rc = cache_dims(cache_dtype, pages, heads, page_size, head_dim, &a.page_shift);
  if (rc != FPX_OK) return rc;
  if (!row_type_ok(dtype) || (!is_coded(cache_dtype) && cache_dtype != dtype)) return FPX_ERR_DIMS;
  const fpx::PagedPlan p =
      paged_plan(dtype, cache_dtype, batch, q_heads, heads, head_dim, max_length, window);
  if (p.groups == 0) return FPX_ERR_DIMS;
  const int64_t row = 16 / (int64_t)type_bytes(dtype);
  if (q_sb < 0 || q_sh < 0 || o_sb < 0 || o_sh < 0 || q_sb % row || q_sh % row || o_sb % row ||
      o_sh % row)
    return FPX_ERR_DIMS;
  if (out == q && (o_sb != q_sb || o_sh != q_sh)) return FPX_ERR_DIMS;
  if (table_sb < 0 || table_sh < 0 || table_pages < (max_length + page_size - 1) / page_size)
    return FPX_ERR_DIMS;
  const float scale_log2 = scale * fpx::kLog2e;
  if (!(scale_log2 - scale_log2 == 0.0f)) return FPX_ERR_DIMS;  // infinite or NaN
  if (batch == 0) return FPX_OK;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(lengths, 4) ||
      !aligned_or_null(lse, 4) || (max_length > 0 && !aligned(block_table, 4)) ||
      !cache_pointers_ok(cache_dtype, cache_k, cache_v, k_scale, v_scale))
    return FPX_ERR_POINTER;
  const PagedWorkspace ws = paged_workspace(p, batch, heads, head_dim);
  if (p.split) {
    if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
    if (workspace_bytes < ws.total) return FPX_ERR_WORKSPACE;
    char* base = static_cast<char*>(workspace);
    a.part = as<float>(base);
    a.part_ml = as<float>(base + ws.ml);
    a.row_info = as<int>(base + ws.info);
  }
  {  // what is written meets nothing else, but q in place
    using fpx::MemoryAxis;
    const int64_t e = (int64_t)type_bytes(dtype);
    const fpx::MemoryBlock query(q, e, MemoryAxis{batch, q_sb}, MemoryAxis{q_heads, q_sh},
                                 MemoryAxis{head_dim, 1});
    const fpx::MemoryBlock written[3] = {
        {out, e, MemoryAxis{batch, o_sb}, MemoryAxis{q_heads, o_sh}, MemoryAxis{head_dim, 1}},
        {lse, 4, MemoryAxis{batch * q_heads, 1}},
        {p.split ? workspace : nullptr, 1, MemoryAxis{(int64_t)ws.total, 1}}};
    const fpx::MemoryBlock table(block_table, 4, MemoryAxis{batch, table_sb},
                                 MemoryAxis{table_sh > 0 ? heads : 1, table_sh},
                                 MemoryAxis{(max_length + page_size - 1) / page_size, 1});
    const fpx::MemoryBlock count(lengths, 4, MemoryAxis{batch, 1});
    const CacheBlocks cache = cache_blocks(cache_dtype, cache_k, cache_v, k_scale, v_scale, pages,
                                           heads, page_size, head_dim);
    if (fpx::block_meets_itself(written[0])) return FPX_ERR_DIMS;
    for (int i = 0; i < 3; ++i) {
      if ((!(i == 0 && out == q) && fpx::blocks_meet(written[i], query)) ||
          fpx::blocks_meet(written[i], table) || fpx::blocks_meet(written[i], count) ||
          meets_cache(written[i], cache))
        return FPX_ERR_DIMS;
      for (int j = 0; j < i; ++j)
        if (fpx::blocks_meet(written[i], written[j])) return FPX_ERR_DIMS;
    }
  }
  a.q = q;
  a.q_b = q_sb;
  a.q_h = q_sh;
  a.k = cache_k;
  a.v = cache_v;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.table = block_table;
  a.table_b = table_sb;
  a.table_h = table_sh;
  a.lengths = lengths;
  a.out = out;
  a.o_b = o_sb;
  a.o_h = o_sh;
  a.lse = lse;
  a.scale_log2 = scale_log2;
  a.weight_shift = cache_dtype == FPX_F16 ? fpx::kWeightShiftF16 : 0.0f;
  a.pages = pages;
  a.batch = (int)batch;
  a.heads = heads;
  a.group = q_heads / heads;
  a.head_dim = head_dim;
  a.max_length = (int)max_length;
  a.window = window < (1 << 30) ? (int)window : 0;
  a.dtype = dtype;
  a.cache_dtype = cache_dtype;
  a.groups = p.groups;
  a.split = p.split;
  a.unit = p.unit;
  a.each = p.each;
  a.tile_queries = p.tile_queries;
  a.qtiles = p.qtiles;
  a.query_tiles = p.query_tiles;
  return status(fpx::launch_paged_attention(a, static_cast<hipStream_t>(stream)));
}

}  // namespace

extern "C" {

int fpx_abi_version(void) { return FPX_ABI_VERSION; }

size_t fpx_tri_attn_workspace_bytes(int n, int c, int heads, int head_dim, int dtype) {
  if (!block_dims_ok(n, c, heads, head_dim, dtype)) return 0;
  return block_workspace(n, dtype).total;
}

int fpx_tri_attn_prepare(int dtype, const void* z, int64_t z_stride0, int64_t z_stride1,
                         const float* mask, int64_t m_stride0, int64_t m_stride1,
                         const void* ln_w, const void* ln_b, float eps, const void* w_qkvg,
                         const void* b_g, const void* w_bias, float mask_inf, int n, int ending,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!block_dims_ok(n, fpx::kChannels, fpx::kHeads, fpx::kHeadDim, dtype)) return FPX_ERR_DIMS;
  if (ending != 0 && ending != 1) return FPX_ERR_DIMS;
  // rows must be 16-byte aligned: 4 floats or 8 bf16
  const int64_t row_align = dtype == FPX_BF16 ? 8 : 4;
  if (z_stride0 % row_align || z_stride1 % row_align || z_stride0 < 0 || z_stride1 < 0)
    return FPX_ERR_DIMS;
  if (m_stride0 < 0 || m_stride1 < 0) return FPX_ERR_DIMS;
  if (!(eps >= 0.0f) || !std::isfinite(mask_inf)) return FPX_ERR_DIMS;
  if (!aligned(z, 16) || !aligned(w_qkvg, 16) || !aligned(w_bias, 16)) return FPX_ERR_POINTER;
  if (!aligned_or_null(mask, 4) || !aligned_or_null(ln_w, 8) || !aligned_or_null(ln_b, 8) ||
      !aligned_or_null(b_g, 4))
    return FPX_ERR_POINTER;
  if (int rc = check_workspace(n, dtype, workspace, workspace_bytes)) return rc;

  const hipStream_t s = static_cast<hipStream_t>(stream);
  const BlockPointers w = block_pointers(workspace, n, dtype);
  // x-frame strides: the ending node reads x[i][j] = z[j][i] (and the mask alike).
  const int64_t xs_i = ending ? z_stride1 : z_stride0;
  const int64_t xs_j = ending ? z_stride0 : z_stride1;
  const int64_t ms_i = ending ? m_stride1 : m_stride0;
  const int64_t ms_j = ending ? m_stride0 : m_stride1;

  hipError_t e = fpx::launch_mask_bias(mask, ms_i, ms_j, n, w.np, mask_inf, w.mbias, w.flags,
                                       w.tri, dtype == FPX_BF16, w.magnitudes, s);
  if (e != hipSuccess) return status(e);

  const float q_scale = 1.0f / std::sqrt((float)fpx::kHeadDim);
  const int64_t wstride = (int64_t)fpx::kHidden * fpx::kChannels;
  if (dtype == FPX_BF16) {
    const __bf16* wq = static_cast<const __bf16*>(w_qkvg);
    fpx::Bf16ProjArgs p{};
    p.x = static_cast<const __bf16*>(z);
    p.xs_i = xs_i;
    p.xs_j = xs_j;
    p.rows_i = n;
    p.rows_j = n;
    p.span_j = (int)round_up(n, 32);  // as the FP32 block's, below
    p.ln_w = static_cast<const __bf16*>(ln_w);
    p.ln_b = static_cast<const __bf16*>(ln_b);
    p.eps = eps;
    for (int g = 0; g < 4; ++g) p.w[g] = wq + g * wstride;
    p.bias_vec = static_cast<const __bf16*>(b_g);
    p.w_bias = static_cast<const __bf16*>(w_bias);
    // BF16 attention logits come out of the matrix cores in log2 units: q
    // and the triangle bias are stored scaled by log2(e).
    p.q_scale = q_scale * fpx::kLog2e;
    p.qh = as<__bf16>(w.qh);
    p.kh = as<__bf16>(w.kh);
    p.vt = as<__bf16>(w.vt);
    p.gs = as<__bf16>(w.gs);
    p.tri_bias = as<__bf16>(w.tri);
    p.np = w.np;
    return status(fpx::launch_projection_bf16(fpx::kProjBlock, p, s));
  }
  const float* wq = static_cast<const float*>(w_qkvg);
  fpx::ProjArgs p{};
  p.x = static_cast<const float*>(z);
  p.xs_i = xs_i;
  p.xs_j = xs_j;
  p.rows_i = n;
  p.rows_j = n;
  // key and query tiles that hold a row; the attention reads none past them
  // but for the queries of its last work-group, whose results it drops
  p.span_j = (int)round_up(n, 32);
  p.ln_w = static_cast<const float*>(ln_w);
  p.ln_b = static_cast<const float*>(ln_b);
  p.eps = eps;
  for (int g = 0; g < 4; ++g) p.w[g] = wq + g * wstride;
  p.b_g = static_cast<const float*>(b_g);
  p.w_bias = static_cast<const float*>(w_bias);
  p.q_scale = q_scale;
  p.qh = as<float>(w.qh);
  p.kh = as<float>(w.kh);
  p.vt = as<float>(w.vt);
  p.gs = as<float>(w.gs);
  p.tri_bias = as<float>(w.tri);
  p.tri_bias_l2 = as<float>(w.tri) + (size_t)fpx::kHeads * w.np * w.np;
  p.magnitudes = w.magnitudes;
  p.scales = w.scales;
  p.np = w.np;
  e = fpx::launch_projection(fpx::kProjBlock, p, s);
  if (e != hipSuccess) return status(e);
  // the fast softmax reads the log2 bias relative to each query's reference,
  // constant-mask rows their shared weights
  return status(fpx::launch_pair_bias(block_attention_args(w, n, mask != nullptr), p.tri_bias_l2,
                                      w.magnitudes, w.flags, s));
}

int fpx_tri_attn_attend(int dtype, int n, void* workspace, size_t workspace_bytes, void* stream) {
  return attend_stage(dtype, n, 1, workspace, workspace_bytes, stream);
}

int fpx_tri_attn_finish(int dtype, const void* w_o, const void* b_o, int n, int ending, void* dz,
                        int64_t dz_stride0, int64_t dz_stride1, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return finish_stage(dtype, w_o, b_o, n, ending, dz, dz_stride0, dz_stride1, workspace,
                      workspace_bytes, stream, 0);
}

int fpx_tri_attn_block(int dtype, const void* z, int64_t z_stride0, int64_t z_stride1,
                       const float* mask, int64_t m_stride0, int64_t m_stride1,
                       const void* ln_w, const void* ln_b, float eps, const void* w_qkvg,
                       const void* b_g, const void* w_bias, const void* w_o, const void* b_o,
                       float mask_inf, int n, int c, int heads, int head_dim, int ending,
                       void* dz, int64_t dz_stride0, int64_t dz_stride1, void* workspace,
                       size_t workspace_bytes, void* stream) {
  return block_impl(dtype, z, z_stride0, z_stride1, mask, m_stride0, m_stride1, ln_w, ln_b, eps,
                    w_qkvg, b_g, w_bias, w_o, b_o, mask_inf, n, c, heads, head_dim, ending, dz,
                    dz_stride0, dz_stride1, workspace, workspace_bytes, stream, 0);
}

int fpx_tri_attn_block_noalloc(int dtype, const void* z, int64_t z_stride0, int64_t z_stride1,
                               const float* mask, int64_t m_stride0, int64_t m_stride1,
                               const void* ln_w, const void* ln_b, float eps, const void* w_qkvg,
                               const void* b_g, const void* w_bias, const void* w_o,
                               const void* b_o, float mask_inf, int n, int c, int heads,
                               int head_dim, int ending, void* dz, int64_t dz_stride0,
                               int64_t dz_stride1, void* stream) {
  if (!block_dims_ok(n, c, heads, head_dim, dtype) || n > kNoAllocMaxN) return FPX_ERR_DIMS;
  if (block_workspace(n, dtype).total > kNoAllocScratchBytes) return FPX_ERR_DIMS;
  hipError_t err = hipSuccess;
  void* ws = device_scratch(&err);
  if (ws == nullptr) return status(err);
  return block_impl(dtype, z, z_stride0, z_stride1, mask, m_stride0, m_stride1, ln_w, ln_b, eps,
                    w_qkvg, b_g, w_bias, w_o, b_o, mask_inf, n, c, heads, head_dim, ending, dz,
                    dz_stride0, dz_stride1, ws, kNoAllocScratchBytes, stream, 0);
}

int fpx_tri_attn_block_residual(int dtype, const void* z, int64_t z_stride0, int64_t z_stride1,
                                const float* mask, int64_t m_stride0, int64_t m_stride1,
                                const void* ln_w, const void* ln_b, float eps,
                                const void* w_qkvg, const void* b_g, const void* w_bias,
                                const void* w_o, const void* b_o, float mask_inf, int n, int c,
                                int heads, int head_dim, int ending, void* z_out,
                                int64_t out_stride0, int64_t out_stride1, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if (z_out == z && (out_stride0 != z_stride0 || out_stride1 != z_stride1)) return FPX_ERR_DIMS;
  return block_impl(dtype, z, z_stride0, z_stride1, mask, m_stride0, m_stride1, ln_w, ln_b, eps,
                    w_qkvg, b_g, w_bias, w_o, b_o, mask_inf, n, c, heads, head_dim, ending, z_out,
                    out_stride0, out_stride1, workspace, workspace_bytes, stream, 1);
}

int fpx_attn_core_masked(const float* q, const float* k, const float* v, const float* mask_bias,
                         int64_t mask_bias_stride, const float* bias, int64_t bias_row_stride,
                         float* out, int batch, int n, void* stream) {
  if (batch < 1 || n < 1 || n % 4 != 0 || n > 65536) return FPX_ERR_DIMS;
  if (bias_row_stride < n || bias_row_stride % 4 != 0) return FPX_ERR_DIMS;
  if (mask_bias != nullptr && mask_bias_stride < 0) return FPX_ERR_DIMS;
  if ((int64_t)batch * fpx::kHeads * (round_up(n, kQueryTile) / kQueryTile) > 0x7fffffffll)
    return FPX_ERR_DIMS;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(bias, 16) ||
      !aligned(out, 16))
    return FPX_ERR_POINTER;
  if (!aligned_or_null(mask_bias, 4)) return FPX_ERR_POINTER;
  fpx::AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.mbias = mask_bias;
  a.mb_stride = mask_bias_stride;
  a.bias = bias;
  a.bias_stride = bias_row_stride;
  a.bias_rows = n;
  a.gate = nullptr;
  a.out = out;
  a.batch = batch;
  a.n = n;
  a.np = n;
  return status(fpx::launch_attention(fpx::kAttnHeadLast, a, static_cast<hipStream_t>(stream)));
}

int fpx_attn_core(float* q, float* k, float* v, float* bias, float* out, int batch, int n,
                  void* stream) {
  return fpx_attn_core_masked(q, k, v, nullptr, 0, bias, n, out, batch, n, stream);
}

int ck_attention(float* q, float* k, float* v, float* bias, float* out, int batch, int n,
                 void* stream) {
  if (!((batch == 1000 && n == 1000) || (batch == 512 && n == 1536))) return FPX_ERR_DIMS;
  // the reference's physical bias row stride (fireprot_ck_attention.cpp:37)
  return fpx_attn_core_masked(q, k, v, nullptr, 0, bias, n == 1536 ? n + 16 : n, out, batch, n,
                              stream);
}

int ck_attention_exact1536(float* q, float* k, float* v, float* bias, float* out, int batch,
                           int n, void* stream) {
  if (batch != 512 || n != 1536) return FPX_ERR_DIMS;
  return fpx_attn_core_masked(q, k, v, nullptr, 0, bias, 1552, out, batch, n, stream);
}

int ck_attention_vector_bias1000(float* q, float* k, float* v, float* bias, float* out,
                                 int batch, int n, void* stream) {
  if (batch != 1000 || n != 1000) return FPX_ERR_DIMS;
  return fpx_attn_core_masked(q, k, v, nullptr, 0, bias, 1000, out, batch, n, stream);
}

size_t fpx_attn_strided_workspace_bytes(int batch, int n) {
  if (batch < 1 || n < 1 || n > kMaxN) return 0;
  return strided_workspace(batch, n).total;
}

int fpx_attn_strided(const float* q, int64_t q_sb, int64_t q_sh, int64_t q_sn, const float* k,
                     int64_t k_sb, int64_t k_sh, int64_t k_sn, const float* v, int64_t v_sb,
                     int64_t v_sh, int64_t v_sn, const float* mask_bias, int64_t m_sb,
                     int64_t m_sk, const float* bias, int64_t b_sh, int64_t b_sq, int64_t b_sk,
                     float* out, int64_t o_sb, int64_t o_sh, int64_t o_sn, int batch, int n,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 1 || n < 1 || n > kMaxN) return FPX_ERR_DIMS;
  const int np = (int)round_up(n, kQueryTile);
  if ((int64_t)batch * fpx::kHeads * (np / kQueryTile) > 0x7fffffffll) return FPX_ERR_DIMS;
  fpx::AttnArgs a{};
  const int64_t qs[3] = {q_sb, q_sh, q_sn}, ks[3] = {k_sb, k_sh, k_sn};
  const int64_t vs[3] = {v_sb, v_sh, v_sn}, os[3] = {o_sb, o_sh, o_sn};
  if (!strided_operand_ok(qs, n, false) || !strided_operand_ok(ks, n, true) ||
      !strided_operand_ok(vs, n, true) || !strided_operand_ok(os, n, false))
    return FPX_ERR_DIMS;
  if (m_sb < 0 || m_sk < 0 || b_sh < 0 || b_sq < 0 || b_sk < 0) return FPX_ERR_DIMS;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return FPX_ERR_POINTER;
  if (!aligned_or_null(mask_bias, 4) || !aligned_or_null(bias, 4)) return FPX_ERR_POINTER;
  if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
  const StridedWorkspace ws = strided_workspace(batch, n);
  if (workspace_bytes < ws.total) return FPX_ERR_WORKSPACE;
  char* base = static_cast<char*>(workspace);
  float* frag = as<float>(base + ws.bias);
  float* frag_l2 = as<float>(base + ws.bias_l2);
  float* mbias = as<float>(base + ws.mbias);
  uint32_t* flags = as<uint32_t>(base + ws.flags);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  uint32_t* mag = as<uint32_t>(base + ws.magnitudes);
  hipError_t e =
      fpx::launch_mask_rows(mask_bias, m_sb, m_sk, batch, n, np, mbias, flags, mag, st);
  if (e != hipSuccess) return status(e);
  e = fpx::launch_stage_bias(bias, b_sh, b_sq, b_sk, n, np, frag, frag_l2, mag, st);
  if (e != hipSuccess) return status(e);
  a.q = q;
  a.k = k;
  a.v = v;
  a.mbias = mbias;
  a.mb_stride = np;
  a.bias = frag;
  a.bias_l2 = frag_l2;
  a.out = out;
  a.tile_flags = flags;
  for (int d = 0; d < 3; ++d) {
    a.qs[d] = qs[d];
    a.ks[d] = ks[d];
    a.vs[d] = vs[d];
    a.os[d] = os[d];
  }
  a.batch = batch;
  a.n = n;
  a.np = np;
  // q, k, v into the plane layout, then the block attention's kernel on it;
  // the magnitude record enables its trailing masked-tile skip
  void* qp = base + ws.qp;
  void* kp = base + ws.kp;
  void* vp = base + ws.vp;
  float* scales = as<float>(base + ws.scales);
  e = fpx::launch_stage_planes(a, qp, kp, vp, scales, as<float>(base + ws.partial), mag, flags,
                               st);
  if (e != hipSuccess) return status(e);
  a.q = static_cast<const float*>(qp);
  a.k = static_cast<const float*>(kp);
  a.v = static_cast<const float*>(vp);
  a.scales = scales;
  a.magnitudes = mag;
  return status(fpx::launch_attention_split(fpx::kAttnStaged, a, st));
}

size_t fpx_tri_mul_workspace_bytes(int n, int c_z, int c_hidden) {
  if (n < 1 || n > kMaxN || c_z != fpx::kChannels || c_hidden != fpx::kHidden) return 0;
  return trimul_workspace(n).total;
}

int fpx_tri_mul(const float* z, int64_t z_stride0, int64_t z_stride1, const float* mask,
                int64_t m_stride0, int64_t m_stride1, const float* ln_in_w, const float* ln_in_b,
                float eps_in, const float* w_abpg, const float* b_abpg, const float* ln_out_w,
                const float* ln_out_b, float eps_out, const float* w_z, const float* b_z,
                const float* w_g, const float* b_g, int n, int c_z, int c_hidden, int outgoing,
                int accumulate, float* out, int64_t out_stride0, int64_t out_stride1,
                void* workspace, size_t workspace_bytes, void* stream) {
  if (n < 1 || n > kMaxN || c_z != fpx::kChannels || c_hidden != fpx::kHidden) return FPX_ERR_DIMS;
  if ((outgoing != 0 && outgoing != 1) || (accumulate != 0 && accumulate != 1)) return FPX_ERR_DIMS;
  if (z_stride0 < 0 || z_stride1 < 0 || z_stride0 % 4 || z_stride1 % 4) return FPX_ERR_DIMS;
  if (out_stride0 < 0 || out_stride1 < 0) return FPX_ERR_DIMS;
  if (mask != nullptr && (m_stride0 < 0 || m_stride1 < 0)) return FPX_ERR_DIMS;
  if (!(eps_in >= 0.0f) || !(eps_out >= 0.0f)) return FPX_ERR_DIMS;
  // out may be z itself (same strides: each pair row is read before it is
  // written, by the same tile); any other overlap is unsupported.
  if (out == z && (out_stride0 != z_stride0 || out_stride1 != z_stride1)) return FPX_ERR_DIMS;
  if (!aligned(z, 16) || !aligned(w_abpg, 16) || !aligned(w_z, 16) || !aligned(w_g, 16) ||
      !aligned(out, 4))
    return FPX_ERR_POINTER;
  if (!aligned_or_null(mask, 4) || !aligned_or_null(b_abpg, 4) || !aligned_or_null(ln_in_w, 8) ||
      !aligned_or_null(ln_in_b, 8) || !aligned_or_null(ln_out_w, 8) ||
      !aligned_or_null(ln_out_b, 8) || !aligned_or_null(b_z, 4) || !aligned_or_null(b_g, 4))
    return FPX_ERR_POINTER;
  if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
  const TriMulWorkspace ws = trimul_workspace(n);
  if (workspace_bytes < ws.total) return FPX_ERR_WORKSPACE;
  char* base = static_cast<char*>(workspace);
  fpx::TriMulArgs a{};
  a.z = static_cast<const float*>(z);
  a.zs_i = z_stride0;
  a.zs_j = z_stride1;
  a.mask = mask;
  a.ms_i = m_stride0;
  a.ms_j = m_stride1;
  a.ln_in_w = ln_in_w;
  a.ln_in_b = ln_in_b;
  a.eps_in = eps_in;
  for (int g = 0; g < 4; ++g) {
    a.w_ab[g] = w_abpg + (int64_t)g * fpx::kHidden * fpx::kChannels;
    a.b_ab[g] = b_abpg ? b_abpg + (int64_t)g * fpx::kHidden : nullptr;
  }
  a.ln_out_w = ln_out_w;
  a.ln_out_b = ln_out_b;
  a.eps_out = eps_out;
  a.w_z = w_z;
  a.b_z = b_z;
  a.w_g = w_g;
  a.b_g = b_g;
  a.pa = as<float>(base + ws.pa);
  a.pb = as<float>(base + ws.pb);
  a.x = as<float>(base + ws.x);
  a.rowmax = as<uint32_t>(base + ws.rowmax);
  a.out = out;
  a.os_i = out_stride0;
  a.os_j = out_stride1;
  a.n = n;
  a.np = (int)round_up(n, kQueryTile);
  a.outgoing = outgoing;
  a.accumulate = accumulate;
  return status(fpx::launch_trimul(a, static_cast<hipStream_t>(stream)));
}

size_t fpx_transition_workspace_bytes(int64_t rows_i, int64_t rows_j, int c, int expansion) {
  if (rows_i < 0 || rows_j < 0 || rows_i > 0x7fffffff || rows_j > 0x7fffffff ||
      c != fpx::kChannels || expansion * c != fpx::kTransitionHidden)
    return 0;
  const int64_t rows = rows_i * rows_j;
  if (rows < 1 || (rows_j + 31) / 32 * rows_i > 0x7fffffffll) return 0;
  return transition_workspace(rows);
}

int fpx_transition(const float* x, int64_t rows_i, int64_t rows_j, int64_t x_stride_i,
                   int64_t x_stride_j, const float* ln_w, const float* ln_b, float eps,
                   const float* w_a, const float* w_b, const float* w_o, int c, int expansion,
                   int accumulate, float* out, int64_t out_stride_i, int64_t out_stride_j,
                   void* workspace, size_t workspace_bytes, void* stream) {
  const size_t need = fpx_transition_workspace_bytes(rows_i, rows_j, c, expansion);
  if (need == 0) return FPX_ERR_DIMS;
  if (accumulate != 0 && accumulate != 1) return FPX_ERR_DIMS;
  // x rows are read as 16-byte vectors: strides in multiples of 4 floats
  if (x_stride_i < 0 || x_stride_j < 0 || x_stride_i % 4 || x_stride_j % 4) return FPX_ERR_DIMS;
  if (out_stride_i < 0 || out_stride_j < 0) return FPX_ERR_DIMS;
  if (!(eps >= 0.0f)) return FPX_ERR_DIMS;
  if (out == x && (out_stride_i != x_stride_i || out_stride_j != x_stride_j)) return FPX_ERR_DIMS;
  if (!aligned(x, 16) || !aligned(w_a, 16) || !aligned(w_b, 16) || !aligned(w_o, 16) ||
      !aligned(out, 4) || !aligned_or_null(ln_w, 8) || !aligned_or_null(ln_b, 8))
    return FPX_ERR_POINTER;
  if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
  if (workspace_bytes < need) return FPX_ERR_WORKSPACE;
  fpx::TransitionArgs a{};
  a.x = x;
  a.xs_i = x_stride_i;
  a.xs_j = x_stride_j;
  a.rows_i = (int)rows_i;
  a.rows_j = (int)rows_j;
  a.ln_w = ln_w;
  a.ln_b = ln_b;
  a.eps = eps;
  a.w_a = w_a;
  a.w_b = w_b;
  a.w_o = w_o;
  a.planes = static_cast<__bf16*>(workspace);
  a.fbias = as<float>(static_cast<char*>(workspace) + kTransitionPlanesBytes);
  a.exps = as<int>(static_cast<char*>(workspace) + kTransitionPlanesBytes + 2 * 512 * sizeof(float));
  a.out = out;
  a.os_i = out_stride_i;
  a.os_j = out_stride_j;
  a.accumulate = accumulate;
  return status(fpx::launch_transition(a, static_cast<hipStream_t>(stream)));
}

int fpx_layer_norm_c128(const float* x, int64_t rows_i, int64_t rows_j, int64_t stride_i,
                        int64_t stride_j, const float* w, const float* b, float eps, float* y,
                        void* stream) {
  if (rows_i < 0 || rows_j < 0 || stride_i < 0 || stride_j < 0) return FPX_ERR_DIMS;
  if (stride_i % 2 || stride_j % 2 || !(eps >= 0.0f)) return FPX_ERR_DIMS;
  if (!aligned(x, 8) || !aligned(y, 8) || !aligned_or_null(w, 8) || !aligned_or_null(b, 8))
    return FPX_ERR_POINTER;
  return status(fpx::launch_layer_norm(x, rows_i, rows_j, stride_i, stride_j, w, b, eps, y,
                                       static_cast<hipStream_t>(stream)));
}

int fpx_qkv_projection(const float* x, int64_t rows, const float* wq, const float* wk,
                       const float* wv, float* out, void* stream) {
  if (rows < 0 || rows > 0x7fffffffll) return FPX_ERR_DIMS;
  if (!aligned(x, 16) || !aligned(wq, 16) || !aligned(wk, 16) || !aligned(wv, 16) ||
      !aligned(out, 16))
    return FPX_ERR_POINTER;
  fpx::ProjArgs p{};
  p.x = x;
  p.xs_i = 0;
  p.xs_j = fpx::kChannels;
  p.rows_i = 1;
  p.rows_j = (int)rows;
  p.span_j = (int)rows;
  p.w[0] = wq;
  p.w[1] = wk;
  p.w[2] = wv;
  p.w[3] = wv;
  p.q_scale = 1.0f / std::sqrt((float)fpx::kHeadDim);
  p.out = out;
  return status(fpx::launch_projection(fpx::kProjQkv, p, static_cast<hipStream_t>(stream)));
}

int fpx_sigmoid_mul_out(const float* gate, const float* value, float* out, int64_t count,
                        void* stream) {
  if (count < 0 || count % 4 != 0) return FPX_ERR_DIMS;
  if (!aligned(gate, 16) || !aligned(value, 16) || !aligned(out, 16)) return FPX_ERR_POINTER;
  return status(fpx::launch_sigmoid_mul(gate, value, out, count / 4,
                                        static_cast<hipStream_t>(stream)));
}

int fpx_split_planes(const float* x, int64_t count, uint16_t* planes, void* stream) {
  if (count < 0 || count % 8 != 0) return FPX_ERR_DIMS;
  if (!aligned(x, 16) || !aligned(planes, 16)) return FPX_ERR_POINTER;
  return status(fpx::launch_split_planes(x, planes, count / 8, static_cast<hipStream_t>(stream)));
}

int fpx_rotary(int dtype, int layout, const void* q, int64_t q_sb, int64_t q_sn, int64_t q_sh,
               void* q_out, int64_t qo_sb, int64_t qo_sn, int64_t qo_sh, int q_heads,
               const void* k, int64_t k_sb, int64_t k_sn, int64_t k_sh, void* k_out,
               int64_t ko_sb, int64_t ko_sn, int64_t ko_sh, int k_heads, const void* positions,
               int positions_64, int64_t p_sb, int64_t p_sn, const double* inv_freq, float scale,
               int inverse, int64_t batch, int64_t tokens, int head_dim, int rotary_dim,
               void* stream) {
  if (dtype != FPX_F32 && dtype != FPX_BF16 && dtype != FPX_F16) return FPX_ERR_DIMS;
  if (layout != FPX_ROTARY_HALF && layout != FPX_ROTARY_INTERLEAVED) return FPX_ERR_DIMS;
  if (positions_64 != 0 && positions_64 != 1) return FPX_ERR_DIMS;
  if (inverse != 0 && inverse != 1) return FPX_ERR_DIMS;
  if (head_dim < 2 || head_dim > fpx::kRotaryMaxDim || rotary_dim < 2 || rotary_dim > head_dim ||
      rotary_dim % 2)
    return FPX_ERR_DIMS;
  if (q_heads < 1 || k_heads < 0 || q_heads > 8192 || k_heads > 8192 - q_heads)
    return FPX_ERR_DIMS;
  if (batch < 0 || tokens < 0 || batch > 0x7fffffff || tokens > 0x7fffffff ||
      batch * tokens > 0x7fffffff)
    return FPX_ERR_DIMS;
  if (q_sb < 0 || q_sn < 0 || q_sh < 0 || qo_sb < 0 || qo_sn < 0 || qo_sh < 0 || p_sb < 0 ||
      p_sn < 0)
    return FPX_ERR_DIMS;
  if (q == q_out && (q_sb != qo_sb || q_sn != qo_sn || q_sh != qo_sh)) return FPX_ERR_DIMS;
  if (k_heads > 0) {
    if (k_sb < 0 || k_sn < 0 || k_sh < 0 || ko_sb < 0 || ko_sn < 0 || ko_sh < 0)
      return FPX_ERR_DIMS;
    if (k == k_out && (k_sb != ko_sb || k_sn != ko_sn || k_sh != ko_sh)) return FPX_ERR_DIMS;
  }
  if (batch == 0 || tokens == 0) return FPX_OK;
  const uintptr_t elem = type_bytes(dtype);
  if (!aligned(q, elem) || !aligned(q_out, elem) || !aligned(positions, positions_64 ? 8 : 4) ||
      !aligned(inv_freq, 8))
    return FPX_ERR_POINTER;
  if (k_heads > 0 && (!aligned(k, elem) || !aligned(k_out, elem))) return FPX_ERR_POINTER;
  {  // what is written meets nothing else, but an input in place
    using fpx::MemoryAxis;
    auto rows = [&](const void* p, int64_t sb, int64_t sn, int64_t sh, int heads) {
      return fpx::MemoryBlock(heads > 0 ? p : nullptr, (int64_t)elem, MemoryAxis{batch, sb},
                              MemoryAxis{tokens, sn}, MemoryAxis{heads, sh},
                              MemoryAxis{head_dim, 1});
    };
    const fpx::MemoryBlock in[2] = {rows(q, q_sb, q_sn, q_sh, q_heads),
                                    rows(k, k_sb, k_sn, k_sh, k_heads)};
    const fpx::MemoryBlock out[2] = {rows(q_out, qo_sb, qo_sn, qo_sh, q_heads),
                                     rows(k_out, ko_sb, ko_sn, ko_sh, k_heads)};
    const fpx::MemoryBlock place(positions, positions_64 ? 8 : 4, MemoryAxis{batch, p_sb},
                                 MemoryAxis{tokens, p_sn});
    const fpx::MemoryBlock freq(inv_freq, 8, MemoryAxis{rotary_dim / 2, 1});
    const bool in_place[2] = {q_out == q, k_out == k};
    for (int i = 0; i < 2; ++i)
      if (fpx::block_meets_itself(out[i]) || (!in_place[i] && fpx::blocks_meet(out[i], in[i])) ||
          fpx::blocks_meet(out[i], in[1 - i]) || fpx::blocks_meet(out[i], place) ||
          fpx::blocks_meet(out[i], freq))
        return FPX_ERR_DIMS;
    if (fpx::blocks_meet(out[0], out[1])) return FPX_ERR_DIMS;
  }
  fpx::RotaryArgs a{};
  a.x[0] = {q, q_out, q_sb, q_sn, q_sh, qo_sb, qo_sn, qo_sh, q_heads};
  if (k_heads > 0) a.x[1] = {k, k_out, k_sb, k_sn, k_sh, ko_sb, ko_sn, ko_sh, k_heads};
  a.pos = positions;
  a.pos_b = p_sb;
  a.pos_n = p_sn;
  a.pos64 = positions_64;
  a.freq = inv_freq;
  a.scale = scale;
  a.inverse = inverse;
  a.dtype = dtype;
  a.interleaved = layout == FPX_ROTARY_INTERLEAVED;
  a.tokens = (int)tokens;
  a.total = (int)(batch * tokens);
  a.head_dim = head_dim;
  a.rot = rotary_dim;
  return status(fpx::launch_rotary(a, static_cast<hipStream_t>(stream)));
}

int fpx_cache_write(int row_dtype, int cache_dtype, const void* k, int64_t k_st, int64_t k_sh,
                    const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots,
                    int64_t tokens, void* cache_k, void* cache_v, void* k_scale, void* v_scale,
                    int64_t pages, int heads, int page_size, int head_dim, void* stream) {
  return cache_impl(false, row_dtype, cache_dtype, k, k_st, k_sh, v, v_st, v_sh, slots, tokens,
                    cache_k, cache_v, k_scale, v_scale, pages, heads, page_size, head_dim, stream);
}

int fpx_cache_read(int row_dtype, int cache_dtype, void* k, int64_t k_st, int64_t k_sh, void* v,
                   int64_t v_st, int64_t v_sh, const int64_t* slots, int64_t tokens,
                   const void* cache_k, const void* cache_v, const void* k_scale,
                   const void* v_scale, int64_t pages, int heads, int page_size, int head_dim,
                   void* stream) {
  return cache_impl(true, row_dtype, cache_dtype, k, k_st, k_sh, v, v_st, v_sh, slots, tokens,
                    cache_k, cache_v, k_scale, v_scale, pages, heads, page_size, head_dim, stream);
}

int fpx_cache_append(int dtype, int cache_dtype, int layout, const void* q, int64_t q_sb,
                     int64_t q_sn, int64_t q_sh, void* q_out, int64_t qo_sb, int64_t qo_sn,
                     int64_t qo_sh, int q_heads, const void* k, int64_t k_sb, int64_t k_sn,
                     int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                     const void* positions, int positions_64, int64_t p_sb, int64_t p_sn,
                     const double* inv_freq, float scale, int rotary_dim, const int64_t* slots,
                     const int32_t* block_table, int64_t table_sb, int64_t table_pages,
                     int64_t batch, int64_t tokens, void* cache_k, void* cache_v, void* k_scale,
                     void* v_scale, int64_t pages, int heads, int page_size, int head_dim,
                     void* stream) {
  fpx::AppendArgs a{};
  const int rc = cache_dims(cache_dtype, pages, heads, page_size, head_dim, &a.page_shift);
  if (rc != FPX_OK) return rc;
  if (!row_type_ok(dtype)) return FPX_ERR_DIMS;
  if (layout != FPX_ROTARY_HALF && layout != FPX_ROTARY_INTERLEAVED) return FPX_ERR_DIMS;
  if (positions_64 != 0 && positions_64 != 1) return FPX_ERR_DIMS;
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2) return FPX_ERR_DIMS;
  if (q_heads < 0 || q_heads > 8192 || heads > 4096 || q_heads + 2 * heads > 8192)
    return FPX_ERR_DIMS;
  if (batch < 0 || tokens < 0 || batch > 0x7fffffff || tokens > 0x7fffffff ||
      batch * tokens > 0x7fffffff)
    return FPX_ERR_DIMS;
  if (k_sb < 0 || k_sn < 0 || k_sh < 0 || v_sb < 0 || v_sn < 0 || v_sh < 0 || p_sb < 0 || p_sn < 0)
    return FPX_ERR_DIMS;
  if (q_heads > 0) {
    if (q_sb < 0 || q_sn < 0 || q_sh < 0 || qo_sb < 0 || qo_sn < 0 || qo_sh < 0)
      return FPX_ERR_DIMS;
    if (q == q_out && (q_sb != qo_sb || q_sn != qo_sn || q_sh != qo_sh)) return FPX_ERR_DIMS;
  }
  if ((slots == nullptr) == (block_table == nullptr)) return FPX_ERR_DIMS;
  if (!slots && (table_sb < 0 || table_pages < 0)) return FPX_ERR_DIMS;
  if (batch == 0 || tokens == 0) return FPX_OK;
  const uintptr_t elem = type_bytes(dtype);
  if (!aligned(k, elem) || !aligned(v, elem) || !aligned(positions, positions_64 ? 8 : 4) ||
      !aligned(inv_freq, 8) || (slots ? !aligned(slots, 8) : !aligned(block_table, 4)) ||
      !cache_pointers_ok(cache_dtype, cache_k, cache_v, k_scale, v_scale))
    return FPX_ERR_POINTER;
  if (q_heads > 0 && (!aligned(q, elem) || !aligned(q_out, elem))) return FPX_ERR_POINTER;
  {  // what is written meets nothing else, but q in place
    using fpx::MemoryAxis;
    auto rows = [&](const void* p, int64_t sb, int64_t sn, int64_t sh, int n) {
      return fpx::MemoryBlock(n > 0 ? p : nullptr, (int64_t)elem, MemoryAxis{batch, sb},
                              MemoryAxis{tokens, sn}, MemoryAxis{n, sh}, MemoryAxis{head_dim, 1});
    };
    const fpx::MemoryBlock out = rows(q_out, qo_sb, qo_sn, qo_sh, q_heads);
    const fpx::MemoryBlock in[6] = {
        rows(q, q_sb, q_sn, q_sh, q_heads), rows(k, k_sb, k_sn, k_sh, heads),
        rows(v, v_sb, v_sn, v_sh, heads),
        {positions, positions_64 ? 8 : 4, MemoryAxis{batch, p_sb}, MemoryAxis{tokens, p_sn}},
        {inv_freq, 8, MemoryAxis{rotary_dim / 2, 1}},
        slots ? fpx::MemoryBlock(slots, 8, MemoryAxis{batch * tokens, 1})
              : fpx::MemoryBlock(block_table, 4, MemoryAxis{batch, table_sb},
                                 MemoryAxis{table_pages, 1})};
    const CacheBlocks cache = cache_blocks(cache_dtype, cache_k, cache_v, k_scale, v_scale, pages,
                                           heads, page_size, head_dim);
    if (fpx::block_meets_itself(out) || meets_cache(out, cache)) return FPX_ERR_DIMS;
    for (int i = 0; i < 6; ++i)
      if ((!(i == 0 && q_out == q) && fpx::blocks_meet(out, in[i])) || meets_cache(in[i], cache))
        return FPX_ERR_DIMS;
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < i; ++j)
        if (fpx::blocks_meet(cache.block[i], cache.block[j])) return FPX_ERR_DIMS;
  }
  const void* in[3] = {q, k, v};
  const int64_t strides[3][3] = {{q_sb, q_sn, q_sh}, {k_sb, k_sn, k_sh}, {v_sb, v_sn, v_sh}};
  for (int w = 0; w < 3; ++w) {
    a.in[w] = in[w];
    a.in_b[w] = strides[w][0];
    a.in_n[w] = strides[w][1];
    a.in_h[w] = strides[w][2];
  }
  a.q_out = q_out;
  a.out_b = qo_sb;
  a.out_n = qo_sn;
  a.out_h = qo_sh;
  a.pos = positions;
  a.pos_b = p_sb;
  a.pos_n = p_sn;
  a.pos64 = positions_64;
  a.freq = inv_freq;
  a.scale = scale;
  a.interleaved = layout == FPX_ROTARY_INTERLEAVED;
  a.rot = rotary_dim;
  a.slots = slots;
  a.table = block_table;
  a.table_b = table_sb;
  a.table_pages = table_pages;
  a.cache[0] = cache_k;
  a.cache[1] = cache_v;
  a.cache_scale[0] = k_scale;
  a.cache_scale[1] = v_scale;
  a.pages = pages;
  a.total = batch * tokens;
  a.tokens = (int)tokens;
  a.q_heads = q_heads;
  a.heads = heads;
  a.head_dim = head_dim;
  a.row_dtype = dtype;
  a.cache_dtype = cache_dtype;
  return status(fpx::launch_cache_append(a, static_cast<hipStream_t>(stream)));
}

size_t fpx_paged_attention_workspace_bytes(int cache_dtype, int64_t batch, int q_heads, int heads,
                                           int head_dim, int64_t max_length, int64_t window) {
  // (of the queries that a cache of this type takes BF16 ones have most shares)
  const fpx::PagedPlan p = paged_plan(is_coded(cache_dtype) ? FPX_BF16 : cache_dtype, cache_dtype,
                                      batch, q_heads, heads, head_dim, max_length, window);
  if (p.groups == 0) return 0;
  return p.split ? paged_workspace(p, batch, heads, head_dim).total : 256;
}

int fpx_paged_attention(int dtype, int cache_dtype, const void* q, int64_t q_sb, int64_t q_sh,
                        const void* cache_k, const void* cache_v, const void* k_scale,
                        const void* v_scale, int64_t pages, int heads, int page_size,
                        int head_dim, const int32_t* block_table, int64_t table_sb,
                        int64_t table_pages, const int32_t* lengths, int64_t batch, int q_heads,
                        int64_t max_length, int64_t window, float scale, void* out, int64_t o_sb,
                        int64_t o_sh, float* lse, void* workspace, size_t workspace_bytes,
                        void* stream) {
  return paged_impl(dtype, cache_dtype, q, q_sb, q_sh, cache_k, cache_v, k_scale, v_scale, pages,
                    heads, page_size, head_dim, block_table, table_sb, 0, table_pages, lengths,
                    batch, q_heads, max_length, window, scale, out, o_sb, o_sh, lse, workspace,
                    workspace_bytes, stream);
}

int fpx_paged_attention_lists(int dtype, int cache_dtype, const void* q, int64_t q_sb, int64_t q_sh,
                              const void* cache_k, const void* cache_v, const void* k_scale,
                              const void* v_scale, int64_t pages, int heads, int page_size,
                              int head_dim, const int32_t* block_table, int64_t table_sb,
                              int64_t table_sh, int64_t table_pages, const int32_t* lengths,
                              int64_t batch, int q_heads, int64_t max_length, float scale,
                              void* out, int64_t o_sb, int64_t o_sh, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return paged_impl(dtype, cache_dtype, q, q_sb, q_sh, cache_k, cache_v, k_scale, v_scale, pages,
                    heads, page_size, head_dim, block_table, table_sb, table_sh, table_pages,
                    lengths, batch, q_heads, max_length, 0, scale, out, o_sb, o_sh, lse, workspace,
                    workspace_bytes, stream);
}

size_t fpx_select_pages_workspace_bytes(int64_t batch, int heads, int page_size,
                                        int64_t max_length, int count) {
  // (each factor is bounded before the next product is formed)
  if (batch < 0 || batch > kPagedMaxRows || heads < 1 || heads > 65535 ||
      batch * heads > kPagedMaxRows || page_size < 16 || page_size > 4096 ||
      (page_size & (page_size - 1)) || max_length < 0 || max_length >= (1 << 30) || count < 1 ||
      count > ((1 << 30) - 1) / page_size)
    return 0;
  const int64_t pages = (max_length + page_size - 1) / page_size;
  if (batch * heads * ((pages + 63) / 64) > 0x7fffffff) return 0;
  if (pages <= count || pages <= fpx::kFewPages) return 256;
  // (never the 256 that stand for none)
  return (size_t)round_up((batch < 1 ? 1 : batch) * heads * pages * 4, 512);
}

int fpx_page_bounds(int cache_dtype, const void* cache_k, const void* k_scale, int64_t pages,
                    int heads, int page_size, int head_dim, const int32_t* block_table,
                    int64_t table_sb, int64_t table_pages, const int32_t* lengths, int64_t batch,
                    int64_t max_length, int64_t fresh, void* bounds, void* stream) {
  fpx::BoundsArgs a{};
  const int rc = cache_dims(cache_dtype, pages, heads, page_size, head_dim, &a.page_shift);
  if (rc != FPX_OK) return rc;
  if (batch < 0 || batch > kPagedMaxRows || max_length < 0 || max_length >= (1 << 30) || fresh < 1)
    return FPX_ERR_DIMS;
  const int64_t most = (max_length + page_size - 1) / page_size;
  if (table_sb < 0 || table_pages < most) return FPX_ERR_DIMS;
  // (so many consecutive tokens touch at most)
  const int64_t each = fresh >= max_length ? most : (fresh + page_size - 2) / page_size + 1;
  a.each = (int)(each < most ? each : most);
  if (batch * heads * a.each > 0x7fffffff) return FPX_ERR_DIMS;
  if (batch == 0 || a.each == 0) return FPX_OK;
  if (!aligned(bounds, 16) || !aligned(lengths, 4) || !aligned(block_table, 4) ||
      !cache_pointers_ok(cache_dtype, cache_k, cache_k, k_scale, k_scale))
    return FPX_ERR_POINTER;
  {  // the bounds meet nothing else
    using fpx::MemoryAxis;
    const int64_t e = (int64_t)type_bytes(is_coded(cache_dtype) ? FPX_BF16 : cache_dtype);
    const fpx::MemoryBlock out(bounds, e, MemoryAxis{pages * heads, 2 * head_dim},
                               MemoryAxis{2 * head_dim, 1});
    const CacheBlocks cache = cache_blocks(cache_dtype, cache_k, cache_k, k_scale, k_scale, pages,
                                           heads, page_size, head_dim);
    const fpx::MemoryBlock table(block_table, 4, MemoryAxis{batch, table_sb}, MemoryAxis{most, 1});
    const fpx::MemoryBlock count(lengths, 4, MemoryAxis{batch, 1});
    if (meets_cache(out, cache) || fpx::blocks_meet(out, table) || fpx::blocks_meet(out, count))
      return FPX_ERR_DIMS;
  }
  a.k = cache_k;
  a.k_scale = k_scale;
  a.bounds = bounds;
  a.table = block_table;
  a.table_b = table_sb;
  a.lengths = lengths;
  a.pages = pages;
  a.batch = (int)batch;
  a.heads = heads;
  a.head_dim = head_dim;
  a.max_length = (int)max_length;
  a.fresh = (int)(fresh < (1 << 30) ? fresh : (1 << 30));
  a.cache_dtype = cache_dtype;
  return status(fpx::launch_page_bounds(a, static_cast<hipStream_t>(stream)));
}

int fpx_select_pages(int dtype, int bounds_dtype, const void* q, int64_t q_sb, int64_t q_sh,
                     int q_heads, const void* bounds, int64_t pages, int heads, int page_size,
                     int head_dim, const int32_t* block_table, int64_t table_sb,
                     int64_t table_pages, const int32_t* lengths, int64_t batch,
                     int64_t max_length, int count, int sinks, int recent, int32_t* index,
                     int32_t* table_out, int32_t* lengths_out, void* workspace,
                     size_t workspace_bytes, void* stream) {
  fpx::SelectArgs a{};
  if (!row_type_ok(dtype) || !row_type_ok(bounds_dtype)) return FPX_ERR_DIMS;
  const int rc = cache_dims(bounds_dtype, pages, heads, page_size, head_dim, &a.page_shift);
  if (rc != FPX_OK) return rc;
  const size_t need =
      fpx_select_pages_workspace_bytes(batch, heads, page_size, max_length, count);
  if (need == 0 || q_heads < heads || q_heads % heads || q_heads > kPagedMaxRows ||
      batch * q_heads > kPagedMaxRows)
    return FPX_ERR_DIMS;
  if (sinks < 0 || recent < 1 || sinks > count - recent) return FPX_ERR_DIMS;
  const int64_t row = 16 / (int64_t)type_bytes(dtype);
  if (q_sb < 0 || q_sh < 0 || q_sb % row || q_sh % row) return FPX_ERR_DIMS;
  const int64_t most = (max_length + page_size - 1) / page_size;
  if (table_sb < 0 || table_pages < most) return FPX_ERR_DIMS;
  if (batch == 0) return FPX_OK;
  if (!aligned(q, 16) || !aligned(bounds, 16) || !aligned(lengths, 4) || !aligned(index, 4) ||
      !aligned(table_out, 4) || !aligned(lengths_out, 4) ||
      (max_length > 0 && !aligned(block_table, 4)))
    return FPX_ERR_POINTER;
  if (need > 256) {
    if (!aligned(workspace, 256)) return FPX_ERR_POINTER;
    if (workspace_bytes < need) return FPX_ERR_WORKSPACE;
  }
  {  // what is written meets nothing else
    using fpx::MemoryAxis;
    const int64_t e = (int64_t)type_bytes(dtype), f = (int64_t)type_bytes(bounds_dtype);
    const int64_t chosen = batch * heads * (int64_t)count;
    const fpx::MemoryBlock written[4] = {
        {index, 4, MemoryAxis{chosen, 1}},
        {table_out, 4, MemoryAxis{chosen, 1}},
        {lengths_out, 4, MemoryAxis{batch, 1}},
        {need > 256 ? workspace : nullptr, 1, MemoryAxis{(int64_t)need, 1}}};
    const fpx::MemoryBlock read[4] = {
        {q, e, MemoryAxis{batch, q_sb}, MemoryAxis{q_heads, q_sh}, MemoryAxis{head_dim, 1}},
        {bounds, f, MemoryAxis{pages * heads, 2 * head_dim}, MemoryAxis{2 * head_dim, 1}},
        {block_table, 4, MemoryAxis{batch, table_sb}, MemoryAxis{most, 1}},
        {lengths, 4, MemoryAxis{batch, 1}}};
    for (int i = 0; i < 4; ++i) {
      for (const fpx::MemoryBlock& r : read)
        if (fpx::blocks_meet(written[i], r)) return FPX_ERR_DIMS;
      for (int j = 0; j < i; ++j)
        if (fpx::blocks_meet(written[i], written[j])) return FPX_ERR_DIMS;
    }
  }
  a.q = q;
  a.q_b = q_sb;
  a.q_h = q_sh;
  a.bounds = bounds;
  a.table = block_table;
  a.table_b = table_sb;
  a.lengths = lengths;
  a.ranks = static_cast<uint32_t*>(workspace);
  a.index = index;
  a.table_out = table_out;
  a.lengths_out = lengths_out;
  a.pages = pages;
  a.max_pages = most;
  a.batch = (int)batch;
  a.heads = heads;
  a.group = q_heads / heads;
  a.head_dim = head_dim;
  a.max_length = (int)max_length;
  a.count = count;
  a.sinks = sinks;
  a.recent = recent;
  a.dtype = dtype;
  a.bounds_dtype = bounds_dtype;
  return status(fpx::launch_select_pages(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
