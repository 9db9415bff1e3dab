// Attention of one new token per sequence over a paged key-value cache: the
// kernel, instantiated per cache type by the paged_attention_*.hip files.
//
//   o[b][h] = sum_j w_j v_j,  w = softmax_j(scale q[b][h] . k_j),
//   j over the sequence's keys [first, length), query head h reading cache
//   head h / group.
//
// A row of the work is one sequence's keys for one cache head and up to 16 QT of the
// query heads that share it, so every key and value is read from memory once for 32
// query heads (16 at 256 channels, whose registers hold one tile of queries): 16
// sequences of 2001 to 8192 BF16 keys, 4 heads of 128, 43 us with 32 queries to a
// head, 63 with 40; of 256, 67 with 16, 108 with 24.  The rows of all sequences, cut
// into units of 128 keys (FP32: 64), form one line of units, of which each of as many
// work-groups as fit the card at once takes an equal share, whatever the sequences'
// lengths: cutting every sequence into chunks of one size instead took 62 us at best
// where this takes 53 (32 sequences of 1 to 4097 BF16 keys, 8 heads of 128), since few
// large chunks leave CUs idle and many small ones are mostly start and join.  (Small
// calls keep to one unit of a row for each work-group: see plan_paged.)  In a row the
// four waves take its tiles in turn, each with an online softmax of its own, and
// join at its end.  Rows that two shares meet in leave (max, sum, o) of each to
// join_shares_kernel.
//
// The bound is memory: 2 D bytes-of-type per key against 4 D group flop.  So
// all products run on the matrix cores with the queries padded to 16 (at one
// query head a 16th of their rate, still several times what the reads need),
// nothing goes through LDS in the loop, and no operand is transposed there:
//   * S^T = K Q^T: a lane holds 8 channels of one key, as they lie in memory.
//     The channels may be contracted in any order, so a lane takes 16
//     consecutive bytes and the queries are loaded in the same order.
//   * the scores of key 4g + r of a 16-key half come out in register r of lane
//     group g (= lane / 16), one query per lane % 16, which is already the B
//     operand of O^T = V^T P^T with its keys in that order: P needs no move.
//   * a lane reads V's rows for its group's eight keys, a 16-byte piece of each
//     row; 4 v_perm per two channels pair the keys up into A operands.
// K of the next tile is in flight during the softmax and the second product,
// V of the next during the first.
//
// Measured, in one call with its join, against the 6.3 TB/s of a plain read: one
// sequence of 131071 BF16 keys, 8 heads of 128: 89 us, 6.0 TB/s; 16 of 20001 to
// 65536 FP8 keys: 235 us, 6.1 TB/s; the ragged 32 above: 5.1 TB/s, of which the
// start and the join are 8 us.  FP32 rows of 256 channels: 7 sequences of 513 to 8190
// keys, 2 heads, 33 us, 3.8 TB/s (four tiles of 128 KB to a work-group, so the start
// and the join are a third of it); 32 of 16384 keys 324 to 339 us, 6.3 to 6.6 TB/s.
// In 4 bits, 8 heads of 128: 16 of 20001 to 131071 keys, 64 queries, 235 us, 5.6 TB/s;
// 32 of 4096, 32 queries, 36.6 us, 3.9, where each further 4096 keys take 25 (5.7): the
// start, the join and the launches between are 11 us.  4 heads of 256, FP16, 24 sequences
// of 4096 keys 34.8 us, of 16384 84.7, 5.1 TB/s: 18 us are fixed, with two work-groups to
// a CU, and the rest runs at 6.1 to 6.6.
//
// Rounding: scores, softmax and accumulators are FP32.  The weights (times the
// value's scale in an 8-bit cache) enter the second product as 16-bit terms whose
// sum has 16 bits of each (two BF16 terms, off by at most 2^-16 of the weight:
// outputs of 8 bits), 22 (two FP16 terms, those weights scaled by 2^14 so that
// small ones keep their bits) or all 24 (three BF16 terms: FP32 queries, and so
// outputs, over 8-bit caches).  Queries of another type than the operands' are
// split likewise into two or three terms (exactly).  8-bit codes are exact in
// BF16, 4-bit codes times their scales as well: those are treated as BF16 values,
// with the terms of an 8-bit cache.
#pragma once

#include "common.hpp"
#include "kernels.hpp"
#include "paged_layout.hpp"

#include <type_traits>

namespace fpx {

struct Fp8Cache {};
struct Int8Cache {};
struct Fp4Cache {};  // codes of 4 bits, a scale to 32 channels

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / kWave;
constexpr float kLn2 = 0.69314718055994531f;

// Sum and maximum over the four lane groups l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float groups_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v),
                                                  __builtin_bit_cast(unsigned, v), false, false);
  v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v),
                                                  __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
}

__device__ __forceinline__ float groups_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v),
                                                  __builtin_bit_cast(unsigned, v), false, false);
  v = fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v),
                                                  __builtin_bit_cast(unsigned, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)s[0]),
               __builtin_bit_cast(float, (unsigned)s[1]));
}

// kBytes (1, 2, 4, 8 or 16) bytes into 32-bit words, the first in the low bits.
// kOnce: non-temporal loads, for whole lines that are read once (V): a plain
// stream of them reaches 7.1 TB/s on an MI355X where ordinary ones reach 6.3
// (4 GB in 32 KB work-groups).  K's lines are read in halves, by two loads, and
// must last from one to the next.
template <int kBytes, bool kOnce>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  using Words = std::conditional_t<
      kBytes <= 2, std::conditional_t<kBytes == 1, uint8_t, uint16_t>,
      std::conditional_t<kBytes == 4, uint32_t,
                         uint32_t __attribute__((ext_vector_type(kBytes < 8 ? 2 : kBytes / 4)))>>;
  const Words* q = reinterpret_cast<const Words*>(p);
  const Words x = kOnce ? __builtin_nontemporal_load(q) : *q;
  if constexpr (kBytes <= 4) {
    w[0] = x;
  } else {
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) w[i] = x[i];
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// Two weights as hi + lo 16-bit words.  hi is cut, not rounded, so that lo is
// never negative, and where values may be infinite (kInfinite) lo is kept above
// zero: then a value of infinity times a weight comes out infinite, and not as
// the NaN of a product with zero or of opposite infinities.  What that adds is
// at most 2^-40 of a weight (FP16: 2^-38 of the largest).
template <bool kF16, bool kInfinite>
__device__ __forceinline__ void split_weights(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  if constexpr (kF16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    float e0 = x0 - (float)h[0], e1 = x1 - (float)h[1];
    if constexpr (kInfinite) {
      e0 = fmaxf(e0, fminf(x0, 0x1p-24f));
      e1 = fmaxf(e1, fminf(x1, 0x1p-24f));
    }
    const f16x2 e = {(_Float16)e0, (_Float16)e1};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, e);
  } else {
    const uint32_t b0 = __builtin_bit_cast(uint32_t, x0), b1 = __builtin_bit_cast(uint32_t, x1);
    hi = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
    float e0 = x0 - __builtin_bit_cast(float, b0 & 0xffff0000u);
    float e1 = x1 - __builtin_bit_cast(float, b1 & 0xffff0000u);
    if constexpr (kInfinite) {
      e0 = fmaxf(e0, x0 * 0x1p-40f);
      e1 = fmaxf(e1, x1 * 0x1p-40f);
    }
    lo = pack_bf16(e0, e1);
  }
}

// Two weights as three BF16 words whose sum is the weight itself: the first two
// cut, so what is left of 24 bits fits the third.
__device__ __forceinline__ void split_weights_exactly(float x0, float x1, uint32_t* terms) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t b0 = __builtin_bit_cast(uint32_t, x0), b1 = __builtin_bit_cast(uint32_t, x1);
    terms[i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
    x0 -= __builtin_bit_cast(float, b0 & 0xffff0000u);
    x1 -= __builtin_bit_cast(float, b1 & 0xffff0000u);
  }
  terms[2] = pack_bf16(x0, x1);
}

// Two 8-bit codes (bytes 2 kHalf and 2 kHalf + 1 of w) as a word of BF16.
template <typename C, int kHalf>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  if constexpr (std::is_same_v<C, Fp8Cache>)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHalf != 0));
  else
    return pack_bf16((float)(int8_t)(w >> (16 * kHalf)), (float)(int8_t)(w >> (16 * kHalf + 8)));
}

// Two 4-bit codes (byte i of w) times their block's scale (its byte) as a word of BF16:
// exact, and NaN where the scale is.
__device__ __forceinline__ uint32_t codes4_bf16(uint32_t w, uint32_t scale, int i) {
  const float s = __builtin_bit_cast(float, scale << 23);
  bf16x2 x;
  switch (i) {
    case 0: x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0); break;
    case 1: x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1); break;
    case 2: x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2); break;
    default: x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  }
  return __builtin_bit_cast(uint32_t, x);
}

// Lanes 8 to 15 of each row of 16 take x, from 8 lanes below, the others keep own; and the
// lower eight from 8 lanes above.
template <typename X>
__device__ __forceinline__ X upper_from(X own, X x) {
  return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, own),
                                                           __builtin_bit_cast(int, x), 0x118, 0xF,
                                                           0xC, false));
}
template <typename X>
__device__ __forceinline__ X lower_from(X own, X x) {
  return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, own),
                                                           __builtin_bit_cast(int, x), 0x108, 0xF,
                                                           0x3, false));
}
__device__ __forceinline__ float halves_sum(float v) { return v + dpp<0x128>(v); }  // row_ror:8
__device__ __forceinline__ float halves_max(float v) { return fmaxf(v, dpp<0x128>(v)); }

// kColumns: of the products, to a query.  Up to eight query heads leave half of the 16
// columns idle, and half of what the softmax computes unused.  A 4-bit cache, whose codes
// take as many instructions to decode as 8 bits and half the time to read, gives each
// query two: in the first product the second column has the query's second term, in the
// second one the weights' second term, and in between its lanes have the other 16 of a
// tile's 32 keys.
template <typename Q, typename C, int D, int QT, int kColumns_>
struct PagedTraits {
  static constexpr int kColumns = kColumns_;
  static constexpr bool kF32 = std::is_same_v<C, float>;
  static constexpr bool kFp4 = std::is_same_v<C, Fp4Cache>;
  // a scale to each row, which its score and its weight are multiplied by
  static constexpr bool kScaled = std::is_same_v<C, Fp8Cache> || std::is_same_v<C, Int8Cache>;
  static constexpr bool kCoded = kScaled || kFp4;
  static constexpr bool kF16 = std::is_same_v<C, _Float16>;
  // channels of `bytes` of a cached row, and bytes of the row
  static constexpr int channels(int bytes) {
    return kFp4 ? 2 * bytes : bytes / (kF32 ? 4 : kCoded ? 1 : 2);
  }
  static constexpr int kRow = D / 2 * (kF32 ? 8 : kFp4 ? 1 : kCoded ? 2 : 4);
  // 16-key parts of a tile
  static constexpr int kHalves =
      kF32 ? 1 : kColumns == 2 && wide_tile4(!std::is_same_v<Q, __bf16>, D) ? 4 : 2;
  static constexpr int kTile = 16 * kHalves;
  // terms a query is split into: all of its bits in BF16, 8 to a term
  static constexpr int kTerms = !kCoded ? 1 : std::is_same_v<Q, __bf16> ? 1
                                          : std::is_same_v<Q, _Float16> ? 2 : 3;
  // terms a weight is split into: what the output's type needs
  static constexpr int kWeightTerms = kCoded && std::is_same_v<Q, float> ? 3 : 2;
  // products for them
  static constexpr int kTermColumns = (kTerms + kColumns - 1) / kColumns;
  static constexpr int kWeightColumns = (kWeightTerms + kColumns - 1) / kColumns;
  static constexpr int kSlots = 4 * kHalves / kColumns;  // keys of a lane in the softmax
  // K: pieces of kPiece bytes a lane holds of its key's row (16 where a
  // quarter of the row has them)
  static constexpr int kPiece = kRow / 4 < 16 ? kRow / 4 : 16;
  static constexpr int kPieces = kRow / 4 / kPiece;
  static constexpr int kPieceChannels = channels(kPiece);
  static constexpr int kPieceSteps = kF32 ? 1 : kPieceChannels / 8;
  static constexpr int kSteps = kF32 ? D / 4 : D / 32;         // of the first product
  static constexpr int kQuerySteps = kF32 ? D / 16 : kSteps;   // 16 bytes of a term each
  // V: channels a lane holds of a row, in pieces
  static constexpr int kChannels = D / 16;
  static constexpr int kPart = kRow / 16 < 16 ? kRow / 16 : 16;  // bytes
  static constexpr int kParts = kRow / 16 / kPart;
  static constexpr int kPartChannels = channels(kPart);
  static constexpr int kPartWords = (kPart + 3) / 4;
  // 4-bit rows of 32 bytes and less: four and more to a line, read by as many loads (of
  // 64 bytes non-temporal loads are still ahead: 237 us and 247 where of 32 it is 100
  // and 93, 16 sequences of 20001 keys and more, 8 heads)
  static constexpr bool kVOnce = !kFp4 || kRow >= 64;
  static constexpr int kVec = kChannels < 4 ? kChannels : 4;   // for the waves' join
  static constexpr int kVecs = kChannels / kVec;
  static constexpr int kPassVecs = kVecs < 2 ? kVecs : 2;      // 32 KB of LDS at most
  // Registers of a lane: its queries, the tile of K and V in flight, the
  // accumulators, and what codes are decoded to.  Where they would spill (256
  // channels, split queries of two tiles) the queries stay in LDS, which the four
  // waves share.  With that, and one step's queries at a time read for both halves of
  // a tile, no kernel here spills (253 registers at most at 256 channels, 226 at most
  // below).  Halves one after the other, which kept all steps' queries from one to the
  // next, spilled up to 217: 16 sequences of 2001 to 16384 keys, 8 heads of 256, FP32
  // queries over INT8, 195 us, 125 now; BF16, 8192 keys, 122 and 113.
  static constexpr int kQueryWords = QT * kQuerySteps * kTermColumns * 4;
  static constexpr int kTileWords = kHalves * (kRow / 16 + 4 * kParts * kPartWords);
  static constexpr bool kQueryLds =
      kQueryWords + kTileWords + QT * kChannels * 4 + (kFp4 ? 32 : kCoded ? 16 : 0) > 160;
  static constexpr float kShift = kF16 ? kWeightShiftF16 : 0.0f;
};

// Units [unit0, unit1) of the row_units of a row: one sequence's keys for one
// cache head and one tile of its query heads.
struct Segment {
  int seq, head, qtile, unit0, unit1, row_units;
  KeyRange range;
};

template <typename Q, typename C, int D, int QT, int kColumns>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_attention_kernel(PagedArgs a) {
  using T = PagedTraits<Q, C, D, QT, kColumns>;
  static_assert(kColumns == 1 || (T::kFp4 && QT == 1), "two columns: 4-bit caches");
  constexpr int kHalves = T::kHalves;
  __shared__ u32x4_t query_lds[T::kQueryLds ? T::kQueryWords / 4 : 1][kWave];
  typedef float Vec __attribute__((ext_vector_type(T::kVec)));
  __shared__ Vec joined[kPagedWaves][4][T::kPassVecs][kWave];
  __shared__ float wave_m[kPagedWaves][QT * 16], wave_l[kPagedWaves][QT * 16];
  __shared__ int wave_units[kPagedWaves];
  __shared__ int found[2];

  // (scalar, so that tile counts and the pages' rows are)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = a.heads * a.qtiles;  // of a sequence
  const int group = ((int)blockIdx.y * rows + (int)blockIdx.x) * (int)gridDim.z + (int)blockIdx.z;
  // (scalar: the compiler cannot know that no store changes the lengths)
  auto range_of = [&](int seq) {
    return key_range(__builtin_amdgcn_readfirstlane(a.lengths[seq]), a.max_length, a.window);
  };
  auto units_of = [&](int seq) {  // each thread's own sequence
    return unit_count(key_range(a.lengths[seq], a.max_length, a.window), a.unit);
  };

  // ---- this work-group's share of the units: one unit of one row, each row
  // having places for a.each of them, or an equal part of them all
  Segment cur;
  Shares shares = {1, 0};
  int share_first, share_end;
  int early_pages = 0, early_key = 0;  // looked up before the length is known
  const bool fixed = a.each > 0;
  if (fixed) {
    cur.seq = blockIdx.y;
    cur.head = blockIdx.x;
    cur.unit0 = blockIdx.z;
    cur.unit1 = cur.unit0 + 1;
    share_first = group;
    share_end = group + 1;
    // without a window the unit's keys are known, and the table has entries up
    // to max_length
    const int lane = threadIdx.x & 63;
    early_key = cur.unit0 * a.unit + (wave + kPagedWaves * (lane / kHalves)) * T::kTile +
                16 * (lane % kHalves);
    if (a.window <= 0 && early_key < a.max_length)
      early_pages = a.table[cur.seq * a.table_b + cur.head / a.qtiles * a.table_h +
                            (early_key >> a.page_shift)];
  } else {
    // The scan over the sequences' units: one to a lane where they fit, in each
    // wave for itself (0.4 us sooner), a run of them to a thread otherwise.
    const int lane = threadIdx.x & 63;
    const bool few = a.batch <= kWave;
    const int per = few ? 1 : (a.batch + kPagedThreads - 1) / kPagedThreads;
    const int thread_first = (few ? lane : (int)threadIdx.x) * per;
    const int last = min(a.batch, thread_first + per);
    int sum = 0, length = 0;
    for (int i = thread_first; i < last; ++i) {
      length = a.lengths[i];
      sum += unit_count(key_range(length, a.max_length, a.window), a.unit);
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int below = __shfl_up(upto, d);
      upto += lane >= d ? below : 0;
    }
    int total = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (!few) {
      if (lane == 0) wave_units[wave] = total;
      if (threadIdx.x == 0) found[0] = found[1] = 0;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) {
        upto += w < wave ? wave_units[w] : 0;
        total += wave_units[w];
      }
      total = __builtin_amdgcn_readfirstlane(total);
    }
    shares = make_shares(total * rows, a.groups);
    share_first = share_start(shares, group);
    share_end = share_start(shares, group + 1);
    if (share_first >= share_end) return;
    const int target = share_first / rows;
    int base;  // units before the sequence, of one row per sequence
    if (few) {
      cur.seq = __popcll(__ballot(upto <= target));
      base = __builtin_amdgcn_readlane(upto - sum, cur.seq);
      cur.range = key_range(__builtin_amdgcn_readlane(length, cur.seq), a.max_length, a.window);
    } else {
      if (target >= upto - sum && target < upto) {
        int seq = thread_first, before = upto - sum;
        for (int n = units_of(seq); target >= before + n && seq + 1 < last; n = units_of(++seq))
          before += n;
        found[0] = seq;
        found[1] = before;
      }
      __syncthreads();
      cur.seq = __builtin_amdgcn_readfirstlane(found[0]);
      base = __builtin_amdgcn_readfirstlane(found[1]);
      cur.range = range_of(cur.seq);
    }
    cur.row_units = unit_count(cur.range, a.unit);
    // (in bounds also where another stream changes the lengths meanwhile)
    const int in_seq = max(share_first - rows * base, 0);
    cur.head = min(in_seq / cur.row_units, rows - 1);
    cur.unit0 = min(in_seq - cur.head * cur.row_units, cur.row_units - 1);
    cur.unit1 = min(cur.row_units, cur.unit0 + share_end - share_first);
  }
  // (so far the row of the sequence)
  cur.qtile = 0;
  if (a.qtiles > 1) {
    const int row = cur.head;
    cur.head = row / a.qtiles;
    cur.qtile = row - cur.head * a.qtiles;
  }
  int unit = share_first;  // the segment's first

  const int page_mask = (1 << a.page_shift) - 1;
  const char* kbase = static_cast<const char*>(a.k);
  const char* vbase = static_cast<const char*>(a.v);
  constexpr int kAhead = kWave / kHalves;  // tiles that 64 pages serve

  uint32_t kw[kHalves][T::kPieces * T::kPiece / 4];
  uint32_t vw[kHalves * 4][T::kParts * T::kPartWords];
  // scales: a row's, or of a block (K: the lane's of each piece; V: of the lane's
  // channels in each of its four rows) as bytes
  f32x4 ks[T::kScaled ? kHalves : 1], vs[T::kScaled ? kHalves : 1];
  uint32_t kb[T::kFp4 ? kHalves : 1][T::kPieces], vb[T::kFp4 ? kHalves * 4 : 1];
  constexpr int kBlocks = D / 32;  // of a row
  // The next 64 halves' pages, one to a lane; a page outside the cache is never
  // read: page 0 stands in and the row comes out NaN.
  int pages_ahead = 0;
  bool bad = false;

  int lane = threadIdx.x & 63;
  auto start_of = [&](const Segment& x) { return first_key(x.range) + x.unit0 * a.unit; };
  auto tiles_of = [&](const Segment& x) {
    const int keys = min(x.range.end, first_key(x.range) + x.unit1 * a.unit) - start_of(x);
    const int tiles = keys > 0 ? (keys + T::kTile - 1) / T::kTile : 0;
    return tiles > wave ? (tiles - wave + kPagedWaves - 1) / kPagedWaves : 0;
  };
  auto look_up = [&](const Segment& x, int n) -> int {
    const int key = start_of(x) + (wave + kPagedWaves * (n + lane / kHalves)) * T::kTile +
                    16 * (lane % kHalves);
    return a.table[x.seq * a.table_b + x.head * a.table_h +
                   table_entry(key, x.range, a.page_shift)];
  };
  auto take_pages = [&](int pages) {
    const bool ok = page_valid(pages, a.pages);
    bad |= !ok;
    pages_ahead = ok ? pages : 0;
  };
  auto row_of = [&](const Segment& x, int n, int u) -> int64_t {
    const int page = __builtin_amdgcn_readlane(pages_ahead, (n % kAhead) * kHalves + u);
    const int key = start_of(x) + (wave + kPagedWaves * n) * T::kTile + 16 * u;
    return (((int64_t)page * a.heads + x.head) << a.page_shift) + (key & page_mask);
  };
  auto load_k = [&](const Segment& x, int n) {
    const int at = (lane & 15) * T::kRow + (lane >> 4) * T::kPiece;
#pragma unroll
    for (int u = 0; u < kHalves; ++u) {
      const int64_t row = row_of(x, n, u);
      const char* p = kbase + row * T::kRow + at;
#pragma unroll
      for (int c = 0; c < T::kPieces; ++c)
        load_words<T::kPiece, false>(p + c * 64, &kw[u][c * T::kPiece / 4]);
      if constexpr (T::kScaled)
        ks[u] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.k_scale) + row +
                                                4 * (lane >> 4));
      if constexpr (T::kFp4) {
        const uint8_t* s = static_cast<const uint8_t*>(a.k_scale) + (row + (lane & 15)) * kBlocks +
                           (lane >> 4) * T::kPieceChannels / 32;
#pragma unroll
        for (int c = 0; c < T::kPieces; ++c) kb[u][c] = s[4 * c];
      }
    }
  };
  auto load_v = [&](const Segment& x, int n) {
    const int at = 4 * (lane >> 4) * T::kRow + (lane & 15) * T::kPart;
#pragma unroll
    for (int u = 0; u < kHalves; ++u) {
      const int64_t row = row_of(x, n, u);
      const char* p = vbase + row * T::kRow + at;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < T::kParts; ++c)
          load_words<T::kPart, T::kVOnce>(p + r * T::kRow + c * 256,
                                          &vw[u * 4 + r][c * T::kPartWords]);
      if constexpr (T::kScaled)
        vs[u] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.v_scale) + row +
                                                4 * (lane >> 4));
      if constexpr (T::kFp4) {
        const uint8_t* s = static_cast<const uint8_t*>(a.v_scale) +
                           (row + 4 * (lane >> 4)) * kBlocks + (lane & 15) * T::kChannels / 32;
#pragma unroll
        for (int r = 0; r < 4; ++r) vb[u * 4 + r] = s[r * kBlocks];
      }
    }
  };
  // the segment after x, where the share goes on
  auto after = [&](const Segment& x) {
    Segment y = x;
    y.unit0 = 0;
    if (++y.qtile == a.qtiles) {
      y.qtile = 0;
      ++y.head;
    }
    if (y.head == a.heads) {
      y.head = 0;
      y.seq = min(y.seq + 1, a.batch - 1);
      y.range = range_of(y.seq);
      y.row_units = unit_count(y.range, a.unit);
    }
    y.unit1 = min(y.row_units, share_end - (unit + x.unit1 - x.unit0));
    return y;
  };

  // ---- the B operand of S^T = K Q^T: the channels of query `col` in K's order,
  // a step at a time, as they lie in memory and split into terms.  (Lanes past
  // the head's last query compute its first one again; their columns are not
  // stored.)
  constexpr int kRaw = T::kF32 ? 1 : (int)sizeof(Q) / 2;  // 16-byte words of a step
  constexpr int kQuads = T::kQuerySteps * T::kTermColumns;  // of a query tile, term by term
  auto load_step = [&](const Segment& x, int t, int st, u32x4_t* raw) {
    const int g = lane >> 4;
    const int qi = (x.qtile * QT + t) * 16 + (lane & (16 / kColumns - 1));
    const Q* q = static_cast<const Q*>(a.q) + x.seq * a.q_b +
                 (int64_t)(x.head * a.group + (qi < a.group ? qi : 0)) * a.q_h;
    const int d = T::kPieceChannels * (4 * (st / T::kPieceSteps) + g) + 8 * (st % T::kPieceSteps);
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = *reinterpret_cast<const u32x4_t*>(q + d + 4 * i);
  };
  auto split_step = [&](const u32x4_t* raw, u32x4_t* terms) {
    if constexpr (T::kTerms == 1) {
      terms[0] = raw[0];
    } else {
      typedef Q Eight __attribute__((ext_vector_type(8)));
      Eight v;
      __builtin_memcpy(&v, raw, sizeof(v));
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
#pragma unroll
      for (int p = 0; p < T::kTerms; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // cut, not rounded: a value near the largest would round to infinity
          const uint32_t w = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[2 * i + 1]),
                                                   __builtin_bit_cast(uint32_t, x[2 * i]),
                                                   0x07060302u);
          terms[p][i] = w;
          // what is left of an infinite value is NaN, which its product with a
          // key would not be: the first term carries it alone
          const float r0 = x[2 * i] - __builtin_bit_cast(float, w << 16);
          const float r1 = x[2 * i + 1] - __builtin_bit_cast(float, w & 0xffff0000u);
          x[2 * i] = __builtin_isinf(x[2 * i]) ? 0.0f : r0;
          x[2 * i + 1] = __builtin_isinf(x[2 * i + 1]) ? 0.0f : r1;
        }
      }
    }
  };
  // (with the queries in LDS the waves share the steps)
  constexpr int kAllSteps = QT * T::kQuerySteps;
  constexpr int kMySteps =
      T::kQueryLds ? (kAllSteps + kPagedWaves - 1) / kPagedWaves : kAllSteps;
  auto step_of = [&](int i) { return T::kQueryLds ? wave + kPagedWaves * i : i; };
  u32x4_t raw[kMySteps][kRaw];
  auto load_queries = [&](const Segment& x) {
#pragma unroll
    for (int i = 0; i < kMySteps; ++i)
      if (step_of(i) < kAllSteps)
        load_step(x, step_of(i) / T::kQuerySteps, step_of(i) % T::kQuerySteps, raw[i]);
  };

  // ---- the rows of the share, one after another.  What the next one begins with
  // is asked for before this one is joined: its pages at this one's start, its
  // first tile (and queries) after this one's last.
  load_queries(cur);
  if (fixed) {
    cur.range = range_of(cur.seq);
    cur.row_units = unit_count(cur.range, a.unit);
    if (cur.unit0 >= cur.row_units) return;
  }
  int mine = tiles_of(cur);
  if (mine > 0) {
    int pages;
    if (fixed && a.window <= 0) {
      // past the sequence's last key its first page here stands in, which
      // holds keys as the wave has a tile
      const int lead = __builtin_amdgcn_readfirstlane(early_pages);
      pages = early_key < cur.range.end ? early_pages : lead;
    } else {
      pages = look_up(cur, 0);
    }
    take_pages(pages);
    load_k(cur, 0);
    load_v(cur, 0);
  }
  while (true) {
    // (not known to be the same for every row: what is derived from the lane is
    // formed again for each, not kept in registers through the loop on its keys)
    asm volatile("" : "+v"(lane));
    const int col = lane & 15, g = lane >> 4;
    const KeyRange range = cur.range;
    const int start = start_of(cur);
    const int next_unit = unit + cur.unit1 - cur.unit0;
    const bool more = next_unit < share_end;
    Segment next = cur;
    int next_pages = 0, next_mine = 0;
    if (more) {
      next = after(cur);
      next_mine = tiles_of(next);
      if (next_mine > 0) next_pages = look_up(next, 0);
    }

    float m[QT], l[QT];
    f32x4 o[QT][T::kChannels];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
#pragma unroll
      for (int c = 0; c < T::kChannels; ++c) o[t][c] = {0.0f, 0.0f, 0.0f, 0.0f};
    }
    u32x4_t qw[T::kQueryLds ? 1 : QT * kQuads];
#pragma unroll
    for (int i = 0; i < kMySteps; ++i) {
      const int t = step_of(i) / T::kQuerySteps, st = step_of(i) % T::kQuerySteps;
      u32x4_t terms[T::kTerms];
      split_step(raw[i], terms);
      if constexpr (kColumns == 2 && T::kTerms > 1) {
#pragma unroll
        for (int p = 0; p < T::kTermColumns; ++p)
          terms[p] = col < 8                  ? terms[2 * p]
                     : 2 * p + 1 < T::kTerms ? terms[2 * p + 1 < T::kTerms ? 2 * p + 1 : 0]
                                             : u32x4_t{0, 0, 0, 0};
      }
#pragma unroll
      for (int p = 0; p < T::kTermColumns; ++p) {
        if constexpr (!T::kQueryLds)
          qw[t * kQuads + p * T::kQuerySteps + st] = terms[p];
        else if (t < QT)
          query_lds[t * kQuads + p * T::kQuerySteps + st][lane] = terms[p];
      }
    }
    if constexpr (T::kQueryLds) {
      // (what was loaded ends here: the compiler keeps it through the loop on the keys
      // otherwise, and spills)
#pragma unroll
      for (int i = 0; i < kMySteps; ++i)
#pragma unroll
        for (int j = 0; j < kRaw; ++j) raw[i][j] = u32x4_t{0, 0, 0, 0};
      __syncthreads();
    }
    int query_lane = lane;
    auto query = [&](int i) -> u32x4_t {
      if constexpr (T::kQueryLds)
        return query_lds[i][query_lane];
      else
        return qw[i];
    };

    for (int n = 0; n < mine; ++n) {
      const int key0 = start + (wave + kPagedWaves * n) * T::kTile;
      // (not known to be the same in every tile, so the reads stay in the loop)
      if constexpr (T::kQueryLds) asm volatile("" : "+v"(query_lane));
      // ---- S^T = K Q^T.  FP32: four sums of a quarter of the channels, which
      // halves the rounding of one long sum
      f32x4 s[QT][kHalves];
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < kHalves; ++u) s[t][u] = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (T::kF32) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          f32x4 sum[4] = {};
#pragma unroll
          for (int c = 0; c < T::kPieces; ++c) {
            const f32x4 y = __builtin_bit_cast(f32x4, query(t * kQuads + c));
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sum[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __builtin_bit_cast(float, kw[0][4 * c + i]), y[i], sum[i], 0, 0, 0);
          }
          s[t][0] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
      } else {
#pragma unroll
        for (int st = 0; st < T::kSteps; ++st) {
          u32x4_t x[kHalves];
#pragma unroll
          for (int u = 0; u < kHalves; ++u) {
            if constexpr (T::kFp4) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                x[u][i] = codes4_bf16(kw[u][st], kb[u][st / T::kPieceSteps], i);
            } else if constexpr (T::kCoded) {
              x[u][0] = codes_bf16<C, 0>(kw[u][2 * st]);
              x[u][1] = codes_bf16<C, 1>(kw[u][2 * st]);
              x[u][2] = codes_bf16<C, 0>(kw[u][2 * st + 1]);
              x[u][3] = codes_bf16<C, 1>(kw[u][2 * st + 1]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) x[u][i] = kw[u][4 * st + i];
            }
          }
#pragma unroll
          for (int t = 0; t < QT; ++t) {
#pragma unroll
            for (int p = T::kTermColumns - 1; p >= 0; --p) {  // the smallest term first
              const u32x4_t y = query(t * kQuads + p * T::kQuerySteps + st);
#pragma unroll
              for (int u = 0; u < kHalves; ++u) {
                if constexpr (T::kF16)
                  s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                      __builtin_bit_cast(f16x8, x[u]), __builtin_bit_cast(f16x8, y), s[t][u], 0, 0,
                      0);
                else
                  s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      __builtin_bit_cast(bf16x8, x[u]), __builtin_bit_cast(bf16x8, y), s[t][u], 0,
                      0, 0);
              }
            }
          }
        }
      }
      // ---- factors of the scores in log2 units; keys outside the range left out
      const bool edge = key0 < range.first || key0 + T::kTile > range.end;
      float f[kHalves][T::kScaled ? 4 : 1];
      uint32_t unseen = 0;  // a bit to a slot
#pragma unroll
      for (int u = 0; u < kHalves; ++u)
#pragma unroll
        for (int r = 0; r < (T::kScaled ? 4 : 1); ++r) {
          if constexpr (T::kScaled)
            f[u][r] = a.scale_log2 * ks[u][r];
          else
            f[u][r] = a.scale_log2;
        }
      if (edge) {
#pragma unroll
        for (int u = 0; u < kHalves; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = key0 + 16 * u + 4 * g + r;
            if (key >= range.first && key < range.end) continue;
            if constexpr (kColumns == 1)
              unseen |= 1u << (4 * u + r);
            else if (u % 2 == (col >> 3))  // (the lane's half of each 32 keys)
              unseen |= 1u << (4 * (u / 2) + r);
            // what the page holds there may be NaN: it must not meet a weight
            // of zero
            if constexpr (T::kScaled) vs[u][r] = 0.0f;
            if constexpr (T::kFp4) vb[u * 4 + r] = 0u;
#pragma unroll
            for (int i = 0; i < T::kParts * T::kPartWords; ++i) vw[u * 4 + r][i] = 0u;
          }
      }
      if (n + 1 < mine) {
        if ((n + 1) % kAhead == 0) take_pages(look_up(cur, n + 1));
        load_k(cur, n + 1);
      }
      // ---- two columns: the terms' scores added up, and of each 32 keys 16 to a column
      if constexpr (kColumns == 2) {
#pragma unroll
        for (int u = 0; u < kHalves; u += 2)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (T::kTerms == 1) {
              s[0][u / 2][r] = upper_from(s[0][u][r], s[0][u + 1][r]);
            } else {
              // (both formed by all lanes, whose neighbours read them)
              const float first = halves_sum(s[0][u][r]), second = halves_sum(s[0][u + 1][r]);
              s[0][u / 2][r] = col < 8 ? first : second;
            }
          }
      }
      // ---- online softmax; a lane's l covers its own keys
      float p[QT][T::kSlots];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < T::kSlots / 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = s[t][u][r] * f[u][T::kScaled ? r : 0];
            top = fmaxf(top, unseen & (1u << (4 * u + r)) ? -__builtin_inff() : x);
          }
        top = groups_max(top);
        if constexpr (kColumns == 2) top = halves_max(top);
        const float next = fmaxf(m[t], top);
        const float ref = next == -__builtin_inff() ? 0.0f : next;
        if (__any(next > m[t])) {
          const float alpha = exp2_fast(m[t] - ref);
          l[t] *= alpha;
#pragma unroll
          for (int c = 0; c < T::kChannels; ++c) o[t][c] *= alpha;
        }
        m[t] = next;
#pragma unroll
        for (int u = 0; u < T::kSlots / 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // one rounding from the product to the exponent
            const float e = __builtin_fmaf(s[t][u][r], f[u][T::kScaled ? r : 0], -ref);
            float w = exp2_fast(T::kShift == 0.0f ? e : e + T::kShift);
            w = unseen & (1u << (4 * u + r)) ? 0.0f : w;
            l[t] += w;
            if constexpr (T::kScaled)
              p[t][u * 4 + r] = w * vs[u][r];
            else
              p[t][u * 4 + r] = w;
          }
      }
      // ---- O^T += V^T P^T
      if constexpr (T::kF32) {
#pragma unroll
        for (int c = 0; c < T::kChannels; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              o[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __builtin_bit_cast(float, vw[r][c]), p[t][r], o[t][c], 0, 0, 0);
      } else {
#pragma unroll
        for (int k0 = 0; k0 < kHalves * 4; k0 += 8) {  // the lane's eight of 32 keys
          u32x4_t weights[QT][T::kWeightColumns];
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < 4 / kColumns; ++i) {
              uint32_t terms[T::kWeightTerms];
              const int slot = k0 / kColumns + 2 * i;
              const float p0 = p[t][slot], p1 = p[t][slot + 1];
              if constexpr (T::kWeightTerms == 3)
                split_weights_exactly(p0, p1, terms);
              else
                split_weights<T::kF16, !T::kCoded>(p0, p1, terms[0], terms[1]);
              if constexpr (kColumns == 1) {
#pragma unroll
                for (int w = 0; w < T::kWeightTerms; ++w) weights[t][w][i] = terms[w];
              } else {
                // the lower lanes have the first 16 keys' weights, the upper the others':
                // the first column gets the first term of both, the second the second
                weights[t][0][i] = upper_from(terms[0], terms[1]);
                weights[t][0][2 + i] = lower_from(terms[1], terms[0]);
                if constexpr (T::kWeightTerms == 3) {
                  const uint32_t none = 0;
                  weights[t][1][i] = col < 8 ? terms[2] : none;
                  weights[t][1][2 + i] = lower_from(none, terms[2]);
                }
              }
            }
          uint32_t pair[8];  // two channels of them
#pragma unroll
          for (int c = 0; c < T::kChannels; ++c) {
            if (c % 2 == 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if constexpr (!T::kCoded)
                  pair[j] = vw[k0 + j][c / 2];
                else if constexpr (T::kFp4)
                  pair[j] = codes4_bf16(vw[k0 + j][c / 8], vb[k0 + j], c % 8 / 2);
                else
                  pair[j] = c % 4 == 0 ? codes_bf16<C, 0>(vw[k0 + j][c / 4])
                                       : codes_bf16<C, 1>(vw[k0 + j][c / 4]);
              }
            }
            u32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i],
                                           c % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
#pragma unroll
              for (int w = T::kWeightColumns - 1; w >= 0; --w) {  // the smallest term first
                if constexpr (T::kF16)
                  o[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                      __builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, weights[t][w]),
                      o[t][c], 0, 0, 0);
                else
                  o[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                      __builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, weights[t][w]),
                      o[t][c], 0, 0, 0);
              }
            }
          }
        }
      }
      if (n + 1 < mine) load_v(cur, n + 1);
    }

    const bool any_bad = __any(bad) || !range.valid;
    bad = false;
    if (more) {
      if constexpr (!T::kQueryLds) load_queries(next);
      if (next_mine > 0) {
        take_pages(next_pages);
        load_k(next, 0);
        load_v(next, 0);
      }
    }

    // ---- the four waves joined, in their order.  Each leaves its maximum, sum and
    // O^T in LDS, and takes one of the four registers r of all of them: a quarter of
    // the row's channels, which it scales, sums and stores.  (Two exchanges between
    // pairs of waves, and one wave's stores, took 0.3 us longer a row of 128
    // channels, 1 us of 256.)
    __syncthreads();  // (the last row's are read)
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      l[t] = any_bad ? __builtin_nanf("") : groups_sum(l[t]);
      if constexpr (kColumns == 2) {
        l[t] = halves_sum(l[t]);
#pragma unroll
        for (int c = 0; c < T::kChannels; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][c][r] = halves_sum(o[t][c][r]);
      }
      if (g == 0) {
        wave_m[wave][t * 16 + col] = m[t];
        wave_l[wave][t * 16 + col] = l[t];
      }
    }
    const int b = cur.seq, head = cur.head;
    const bool direct = cur.unit0 == 0 && cur.unit1 == cur.row_units;
    const bool empty = range.valid && range.end <= range.first;
    const int place = group * 2 + (unit == share_first ? 0 : 1);
    if (cur.unit0 == 0 && a.split && threadIdx.x == 0) {
      int* info = a.row_info + ((int64_t)b * rows + head * a.qtiles + cur.qtile) * 2;
      info[0] = place;
      info[1] = fixed ? cur.row_units
                      : share_of(shares, unit + cur.row_units - 1) - group + 1;
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float factor[kPagedWaves], sum[T::kChannels] = {};
      float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
      for (int v0 = 0; v0 < T::kVecs; v0 += T::kPassVecs) {
        if (t > 0 || v0 > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int v = 0; v < T::kPassVecs; ++v) {
            Vec x;
#pragma unroll
            for (int c = 0; c < T::kVec; ++c) x[c] = o[t][(v0 + v) * T::kVec + c][r];
            joined[wave][r][v][lane] = x;
          }
        __syncthreads();
        if (v0 == 0) {
#pragma unroll
          for (int w = 0; w < kPagedWaves; ++w) top = fmaxf(top, wave_m[w][t * 16 + col]);
          const float ref = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
          for (int w = 0; w < kPagedWaves; ++w) {
            factor[w] = exp2_fast(wave_m[w][t * 16 + col] - ref);
            total += wave_l[w][t * 16 + col] * factor[w];
          }
        }
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w)
#pragma unroll
          for (int v = 0; v < T::kPassVecs; ++v) {
            const Vec x = joined[w][wave][v][lane];
#pragma unroll
            for (int c = 0; c < T::kVec; ++c) sum[(v0 + v) * T::kVec + c] += x[c] * factor[w];
          }
      }
      const int qi = (cur.qtile * QT + t) * 16 + col;  // of the cache head's query heads
      if (qi >= a.group) continue;
      // O^T: lane (query col, group g), register r of channel c of a part: channel
      // (4g + r) * kPartChannels + c of the part's 16 * kPartChannels
      const int hq = head * a.group + qi;
      const float scale = direct ? (empty ? 0.0f : 1.0f / total) : 1.0f;
      const int64_t part_row = (int64_t)place * a.tile_queries + t * 16 + col;
      // (rows of out are 16-byte aligned)
      char* to = direct ? reinterpret_cast<char*>(static_cast<Q*>(a.out) + b * a.o_b + hq * a.o_h)
                        : reinterpret_cast<char*>(a.part + part_row * D);
      typedef float Piece __attribute__((ext_vector_type(T::kPartChannels)));
      typedef Q OutPiece __attribute__((ext_vector_type(T::kPartChannels)));
#pragma unroll
      for (int pt = 0; pt < T::kParts; ++pt) {
        const int d = (16 * pt + 4 * g + wave) * T::kPartChannels;
        Piece x;
#pragma unroll
        for (int c = 0; c < T::kPartChannels; ++c) x[c] = sum[pt * T::kPartChannels + c] * scale;
        if (std::is_same_v<Q, float> || !direct)
          *reinterpret_cast<Piece*>(to + d * 4) = x;
        else
          *reinterpret_cast<OutPiece*>(to + d * sizeof(Q)) = __builtin_convertvector(x, OutPiece);
      }
      if (threadIdx.x < 16) {
        if (!direct) {
          a.part_ml[part_row * 2] = top;
          a.part_ml[part_row * 2 + 1] = total;
        } else if (a.lse) {
          a.lse[(int64_t)b * a.heads * a.group + hq] =
              empty ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total) - T::kShift) * kLn2;
        }
      }
    }

    if (!more) break;
    if constexpr (T::kQueryLds) load_queries(next);  // (no registers for them before)
    unit = next_unit;
    cur = next;
    mine = next_mine;
  }
}

template <typename Q, typename C, int D>
hipError_t launch_paged_dim(const PagedArgs& a, hipStream_t stream) {
  // a unit of a row to a work-group, the units slowest (work-groups go to the
  // XCDs in turn: with the units fastest those that shorter sequences lack would
  // all be missing on the same XCDs), or equal shares
  const dim3 groups = a.each > 0 ? dim3(a.heads * a.qtiles, a.batch, a.each) : dim3(a.groups);
  if (a.query_tiles == 1) {
    if constexpr (std::is_same_v<C, Fp4Cache>) {
      if (a.group <= 8) {
        paged_attention_kernel<Q, C, D, 1, 2><<<groups, kPagedThreads, 0, stream>>>(a);
        return hipGetLastError();
      }
    }
    paged_attention_kernel<Q, C, D, 1, 1><<<groups, kPagedThreads, 0, stream>>>(a);
  } else {
    if constexpr (D <= 128)
      paged_attention_kernel<Q, C, D, 2, 1><<<groups, kPagedThreads, 0, stream>>>(a);
    else
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <typename Q, typename C>
hipError_t launch_paged_type(const PagedArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 32: return launch_paged_dim<Q, C, 32>(a, stream);
    case 64: return launch_paged_dim<Q, C, 64>(a, stream);
    case 128: return launch_paged_dim<Q, C, 128>(a, stream);
    default: return launch_paged_dim<Q, C, 256>(a, stream);
  }
}

}  // namespace fpx
