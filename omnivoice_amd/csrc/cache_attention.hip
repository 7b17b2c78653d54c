// Attention over the 8-bit key/value cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j that a query sees
//
// The rows of a kv head are its query heads' queries, row r of a sequence
// being query r / group of head r % group: the whole group shares every key
// and value that is loaded. Scores are formed transposed, S^T = K Q^T, so a
// lane owns one row's column, and so is the output, O^T = V^T P^T, whose P^T
// operand is the scores' accumulator itself. e4m3 codes are exact in fp16 and
// bf16, so the products see the queries and codes as they are: the keys' scale
// joins the softmax's in the float32 scores, the values' is a power of two. The
// one rounding on the way is that of the probabilities to the queries' type, and
// the row's sum takes the rounded ones, so that the weights still add up to one.
//
// A work-group takes 16 or 32 rows of one sequence and kv head and one split of
// its keys; each of its four waves takes a quarter of those in steps of 32, with a
// softmax of its own that runs along (maximum m, sum l, output o), and the four are
// joined in LDS at the end. Where there are rows enough, each wave takes 32 of them
// and all their keys instead, and nothing is joined. The pool's order is that of the matrix operands: the
// codes go from memory straight into registers, a step ahead, and are converted
// there, with no LDS and no barrier on the way. A version in which 128 rows shared
// tiles that were converted once and left in LDS was slower at every size (two
// causal prompts of 2500 tokens 104 us and 81 here, four chunks of 375 frames over
// 2000 keys 61 and 39): its waves wait for each other at every tile, and a tile of
// 128 rows leaves CUs idle where there are few.
//
// Bound: memory where rows are few, 48 sequences of up to 8192 tokens (474 MB) in
// 96.0 us, 4.9 TB/s. With many the issue of matrix and vector instructions: two causal
// prompts of up to 5000 tokens (198 GFLOP) in 230 us on one card and 240 on another, 860
// and 828 TFLOP/s, the matrix cores busy 46 % and vector instructions 38 % of the time;
// of the largest library product 1174. A third work-group to a CU, its queries in LDS,
// did not raise that. A short call is a chain of trips to memory: one token over 430
// takes the kernel 7 us.
#include <algorithm>

#include "cache.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Types;
template <>
struct Types<_Float16> {
  typedef f16x2 x2;
  typedef f16x8 x8;
  static __device__ __forceinline__ x2 Low(unsigned w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), s, false);
  }
  static __device__ __forceinline__ x2 High(unsigned w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), s, true);
  }
  // To the type, nearest even.
  static __device__ __forceinline__ x2 Round(float a, float b) {
    return x2{static_cast<_Float16>(a), static_cast<_Float16>(b)};
  }
  static __device__ __forceinline__ float AddPair(x2 pair, float sum) {
    return __builtin_amdgcn_fdot2(pair, x2{1, 1}, sum, false);
  }
  static __device__ __forceinline__ floatx4 Mfma16(x8 a, x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx16 Mfma32(x8 a, x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Types<__bf16> {
  typedef bf16x2 x2;
  typedef bf16x8 x8;
  static __device__ __forceinline__ x2 Low(unsigned w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), s, false);
  }
  static __device__ __forceinline__ x2 High(unsigned w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), s, true);
  }
  // To the type, nearest even.
  static __device__ __forceinline__ x2 Round(float a, float b) {
    return x2{static_cast<__bf16>(a), static_cast<__bf16>(b)};
  }
  static __device__ __forceinline__ float AddPair(x2 pair, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(pair, x2{static_cast<__bf16>(1.0F), static_cast<__bf16>(1.0F)}, sum, false);
  }
  static __device__ __forceinline__ floatx4 Mfma16(x8 a, x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx16 Mfma32(x8 a, x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Eight codes in two words, times the power of two `scale`, as one operand.
template <typename T>
__device__ __forceinline__ typename Types<T>::x8 Operand(unsigned lo, unsigned hi, float scale) {
  typedef Types<T> X;
  const typename X::x2 a = X::Low(lo, scale), b = X::High(lo, scale);
  const typename X::x2 c = X::Low(hi, scale), d = X::High(hi, scale);
  return typename X::x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48, and their sum: two swaps of
// rows between registers instead of trips through LDS.
__device__ __forceinline__ float Partner32(float v, float* other) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  *other = __uint_as_float(r[1]);
  return __uint_as_float(r[0]);
}
__device__ __forceinline__ float Partner16(float v, float* other) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  *other = __uint_as_float(r[1]);
  return __uint_as_float(r[0]);
}
__device__ __forceinline__ float Max32(float v) {
  float b;
  const float a = Partner32(v, &b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float Sum32(float v) {
  float b;
  const float a = Partner32(v, &b);
  return a + b;
}
__device__ __forceinline__ float Max16(float v) {
  float b;
  const float a = Partner16(v, &b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float Sum16(float v) {
  float b;
  const float a = Partner16(v, &b);
  return a + b;
}

// Over the lanes of a row: lane, lane ^ 32 and with 16 rows lane ^ 16, ^ 48.
template <int ROWS>
__device__ __forceinline__ float RowMax(float v) {
  return Max32(ROWS == 16 ? Max16(v) : v);
}
template <int ROWS>
__device__ __forceinline__ float RowSum(float v) {
  return Sum32(ROWS == 16 ? Sum16(v) : v);
}

__device__ __forceinline__ float Lane(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// The values' loudness: the scale that the sums are held at, a power of two
// that only grows. A block's codes are multiplied by its own scale over this one
// as they are converted, at most 1, so that no fp16 operand overflows however
// loud a block is; a block quieter than the loudest by 2^15 or more loses the
// bits under fp16's 2^-24, 2^-33 of that loudest block's largest value.
constexpr float kQuietest = 7.52316385e-37F;  // 2^-120
__device__ __forceinline__ float InversePower(float p) {
  return __uint_as_float((254u << 23) - __float_as_uint(p));
}
// The power of two above a row's sum of weights (0, or from 1 to 2^38). Outputs are
// taken over that much before they meet their loudness: averages of the type's largest
// values are finite where their sums are not, and powers of two round nothing.
__device__ __forceinline__ float PowerAbove(float sum) {
  return __uint_as_float((__float_as_uint(fmaxf(sum, 1.0F)) & 0x7F800000u) + (1u << 23));
}
// 0 for a block without a (numeric) scale.
__device__ __forceinline__ float Loudness(float scale) { return scale == scale ? scale : 0.0F; }

// The query and head of a tile's rows, by products with the host's 2^36 / group
// (for the tile's first row, below 2^24 group) and 2^16 / group (for the fewer than
// 128 + 64 rows behind the start of its query), both rounded up and exact there.
struct RowSplit {
  int query, left, group, inverse;
  __device__ __forceinline__ RowSplit(const CacheAttentionParams& p, int first_row) {
    group = p.group;
    inverse = p.group_inverse;
    query = static_cast<int>(static_cast<unsigned long long>(first_row) * p.group_magic >> 36);
    left = first_row - query * group;
  }
  __device__ __forceinline__ int Of(int behind, int* of_group) const {
    const int more = ((left + behind) * inverse) >> 16;
    *of_group = left + behind - more * group;
    return query + more;
  }
  __device__ __forceinline__ int At(int row) const {  // the query of a row of the tile
    return query + (((row - query * group) * inverse) >> 16);
  }
};

// How far a row's maximum may rise before its sums are scaled again: their
// probabilities are then at most 2^8, far inside fp16, and most steps of a long
// row leave the sums alone. Each row goes by its own maximum: what the others
// hold changes none of its bits. (The values' loudness is that of all the sequence's
// blocks so far, also of those that a row does not see; a power of two, it rounds
// only what lies 2^-33 under it in fp16.)
constexpr float kSlack = 8.0F;

// A weight's exponent is one fused step from the score's product, score * factor - maximum,
// whose maximum was rounded: by 2^-8 at most below 2^16 in size, which every weight of the
// row shares, but by more than the weights' range from 2^28 on. Rows whose maximum is
// larger than this round their products first, as the maximum is.
constexpr float kLarge = 65536.0F;

constexpr int kWaves = 4;

// A wave's window of the block table: lane i holds, of the i-th block, where the
// head's part begins, the scores' factor, and the values' scale over `loud`, the
// loudest of this window's blocks and all before. The steps wait for the table and
// the scales once per 64 blocks and not one after the other. Where a block is not there
// (no name in the table, or behind the keys) a step reads the window's first one that
// is: its rows have no weight, but only a block that was written holds nothing but
// numbers, and 0 times a NaN code would be NaN.
struct Window {
  unsigned offset_low, offset_high;
  float factor, unit;
  float loud;                // the same in every lane
  unsigned long long there;  // a bit for each block that there is
  __device__ __forceinline__ void LoadPages(const CacheView& c, int sequence, int head, int first,
                                            int stop, int lane) {
    const int block = first + lane;
    const int page = (block << c.block_shift) < stop ? PageOf(c, sequence, block) : -1;
    there = __ballot(page >= 0);
    if (there == 0)
      return;  // nothing to read
    const int some = __builtin_amdgcn_readlane(page, __ffsll(there) - 1);
    scale_at = ScaleIndex(c, page >= 0 ? page : some, head, 0);
    const std::size_t offset = scale_at * (static_cast<std::size_t>(c.dim) << c.block_shift);
    offset_low = static_cast<unsigned>(offset);
    offset_high = static_cast<unsigned>(offset >> 32);
  }
  __device__ __forceinline__ void LoadScales(const CacheAttentionParams& p, int lane) {
    const float k_scale = p.cache.scales[scale_at], v_scale = p.cache.scales[scale_at + 1];
    const bool here = (there >> lane & 1) != 0;
    // A NaN scale, of keys or values, makes the block's scores NaN.
    factor = here ? p.scale_log2 * k_scale + 0.0F * v_scale : 0.0F;
    const float level = here ? Loudness(v_scale) : 0.0F;
    loud = fmaxf(loud, WaveMaxFast(level));
    unit = fmaxf(level * InversePower(loud), kQuietest);
  }
  __device__ __forceinline__ const unsigned char* Base(const unsigned char* data, int i) const {
    const std::size_t low = __builtin_amdgcn_readlane(offset_low, i);
    const std::size_t high = __builtin_amdgcn_readlane(offset_high, i);
    return data + (high << 32 | (low & 0xFFFFFFFFu));
  }

 private:
  std::size_t scale_at;
};

// The first of the four dims of a lane's j-th run of output: of rows 8 (j % 4) + 4 part
// .. + 3 of tile j / 4, or 4 part .. + 3 of tile j.
template <int DIM, int ROWS>
__device__ __forceinline__ int DimOf(int j, int part) {
  const int t = j / 4, high = j % 4 / 2, d = 8 * (j % 2) + 4 * part;
  return ROWS == 16   ? 16 * j + 4 * part
         : DIM == 128 ? 64 * high + 16 * t + d
                      : 32 * high + 16 * t + d;
}

// ROWS rows (16 or 32) on v_mfma_f32_16x16x32 or v_mfma_f32_32x32x16: lane l holds
// row l % ROWS and is part l / ROWS of it. Of every 16 keys a part holds four in a
// row at 4 part (and with two parts the four at 8 more). A lane's 16 bytes of a key
// are 16 dims, the next part's the next 16; which dim meets which is the same for the
// queries. A lane's bytes of the values are four keys of dims 16 apart: with 16 rows
// the output's tile t is dims 16 t .. + 15; with 32 its two halves of rows stand for
// dims 64 apart (128 dims) or 32 apart (64).
// ONE: 32 keys are of one block (blocks of 32 or 64 tokens), else of two of 16.
// OWN: a wave takes a tile of its own with all its keys, the work-group's four one
// after the other, instead of a quarter of one tile's keys: nothing is joined, and
// the four read the same codes at about the same time, three of them out of the L1.
template <typename T, int DIM, int ROWS, bool ONE, bool OWN>
__global__ __launch_bounds__(kWaves* kWave, 2) void CacheAttentionKernel(
    CacheAttentionParams p) {
  typedef Types<T> X;
  typedef typename X::x8 x8;
  constexpr int kParts = kWave / ROWS;
  constexpr int kSteps = DIM / 16 / kParts;  // 16-byte loads of a key's codes in a lane
  constexpr int kOfGroup = 16 / kParts;      // a lane's keys of 16
  constexpr int kTiles = DIM / ROWS;         // of the output
  constexpr int kFours = ROWS * ROWS / 256;  // a lane's runs of four rows of a tile
  typedef float acc_t __attribute__((ext_vector_type(4 * kFours)));
  // A lane's codes of the values of 16 keys: loads, and the bytes of one.
  constexpr int kValueLoads = ROWS == 16 ? DIM / 64 : 2;
  constexpr int kValueWords = ROWS == 16 ? 4 : DIM / 32;
  typedef unsigned value_t __attribute__((ext_vector_type(kValueWords)));
  const CacheView& c = p.cache;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane % ROWS, part = lane / ROWS;
  const int head = blockIdx.x;

  // The last rows of a causal sequence see the most keys: they start first.
  const int item = p.items - 1 - p.first_item - static_cast<int>(blockIdx.y);
  const Found found = FindItem(c, p.group, ROWS == 16 ? 4 : OWN ? 7 : 5, 1, item);
  const int sequence = found.sequence;
  const int tile = OWN ? found.item * kWaves + wave : found.item;
  const Span span = found.span;
  const int rows = span.count * p.group;
  if (tile < 0 || tile * ROWS >= rows)
    return;
  const int length = min(span.length, c.table_width << c.block_shift);
  // Keys that any row of the tile sees, those of this split, and those every row sees.
  const RowSplit split(p, tile * ROWS);
  const int last = min(tile * ROWS + ROWS, rows) - 1;
  const int end = p.causal ? min(span.start + split.At(last) + 1, length) : length;
  const int chunk = ChunkOf(length, p.splits);
  const int begin = blockIdx.z * chunk;
  const int stop = min(begin + chunk, end);
  const int all_see = p.causal ? min(span.start + split.query + 1, length) : length;

  // Rows past the last one repeat it; nothing of theirs is stored.
  const int row = tile * ROWS + column;
  int of_group;
  const int query = split.Of(min(row, rows - 1) - tile * ROWS, &of_group);
  const int seen = p.causal ? min(span.start + query + 1, length) : length;
  x8 q[kSteps][2];
  {
    const T* from = static_cast<const T*>(p.q) +
                    static_cast<std::int64_t>(span.first + query) * p.q_stride +
                    static_cast<std::int64_t>(head * p.group + of_group) * DIM + 16 * part;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      __builtin_memcpy(&q[i][0], from + 16 * kParts * i, sizeof(x8));
      __builtin_memcpy(&q[i][1], from + 16 * kParts * i + 8, sizeof(x8));
    }
    if (p.negate) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        q[i][0] = -q[i][0];
        q[i][1] = -q[i][1];
      }
    }
  }

  float m = -__builtin_inff(), l[2] = {0.0F, 0.0F};
  acc_t o[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
    o[t] = acc_t(0.0F);
  float loud = kQuietest;
  bool large = false;  // some row's maximum is

  const int quarter = ((stop - begin + kWaves * 32 - 1) / (kWaves * 32)) * 32;
  const int wave_begin = OWN ? begin : begin + wave * quarter;
  const int wave_stop = OWN ? stop : min(wave_begin + quarter, stop);
  const int in_block = (1 << c.block_shift) - 1;
  const std::size_t half_bytes = static_cast<std::size_t>(DIM) << c.block_shift;
  // With 32 rows a lane's key is of the first or the second 16, and its values of
  // the tiles' first or second 16 rows.
  const int second = ROWS == 16 ? 0 : (lane >> 4) & 1;
  const int key_at = part * 256 + (lane & 15) * 16;
  const int value_at = key_at + second * (DIM == 128 ? 1024 : 8);

  Window w;
  w.loud = kQuietest;
  for (int window = wave_begin; window < wave_stop;) {
    const int first_block = window >> c.block_shift;
    w.LoadPages(c, sequence, head, first_block, wave_stop, lane);
    const int window_stop = min((first_block + kWave) << c.block_shift, wave_stop);
    if (w.there == 0) {
      window = window_stop;
      continue;
    }
    const int last_step = window + ((window_stop - 1 - window) & ~31);

    struct Codes {
      u32x4 k[32 / ROWS][kSteps];  // with 16 rows of two groups, else of the lane's own
      value_t v[2][kValueLoads];
    };
    const auto load = [&](int key, Codes* d) {
      const int at = min(key, last_step);
      const int block = (at >> c.block_shift) - first_block;
      const unsigned char* group[2];
      group[0] = w.Base(c.data, block) + (ONE ? at & in_block : 0) * DIM;
      group[1] = ONE ? group[0] + 16 * DIM : w.Base(c.data, block + 1);
#pragma unroll
      for (int g = 0; g < 32 / ROWS; ++g) {
        const unsigned char* from = ROWS == 16 ? group[g] : second == 0 ? group[0] : group[1];
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          d->k[g][i] = *reinterpret_cast<const u32x4*>(from + key_at + 256 * kParts * i);
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i)
          d->v[g][i] = *reinterpret_cast<const value_t*>(group[g] + half_bytes + value_at +
                                                         (ROWS == 16 ? 1024 : 512) * i);
    };
    const auto step = [&](int key, const Codes& d) {
      const int block = (key >> c.block_shift) - first_block;
      float factor[2], unit[2];
      bool there[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int at = ONE ? block : block + g;
        factor[g] = Lane(w.factor, at);
        unit[g] = Lane(w.unit, at);
        there[g] = (w.there >> at & 1) != 0;
      }
      float s[2][kOfGroup];
      if constexpr (ROWS == 16) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          floatx4 acc = {};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            acc = X::Mfma16(Operand<T>(d.k[g][i][0], d.k[g][i][1], 1.0F), q[i][0], acc);
            acc = X::Mfma16(Operand<T>(d.k[g][i][2], d.k[g][i][3], 1.0F), q[i][1], acc);
          }
#pragma unroll
          for (int r = 0; r < kOfGroup; ++r)
            s[g][r] = acc[r];
        }
      } else {
        floatx16 acc = {};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          acc = X::Mfma32(Operand<T>(d.k[0][i][0], d.k[0][i][1], 1.0F), q[i][0], acc);
          acc = X::Mfma32(Operand<T>(d.k[0][i][2], d.k[0][i][3], 1.0F), q[i][1], acc);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r / 8][r % 8] = acc[r];
      }
      // Where some row does not see all of the step, what it does not is -inf and the
      // factors have been taken.
      if (!(there[0] && there[1]) || key + 32 > all_see) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
          for (int r = 0; r < kOfGroup; ++r) {
            const int at = key + 16 * g + 4 * (part + kParts * (r / 4)) + r % 4;
            s[g][r] = there[g] && at < seen ? s[g][r] * factor[g] : -__builtin_inff();
          }
          factor[g] = 1.0F;
        }
      }
      float peak = -__builtin_inff();
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float most = s[g][0];
#pragma unroll
        for (int r = 1; r < kOfGroup; ++r)
          most = fmaxf(most, s[g][r]);
        peak = fmaxf(peak, factor[g] * most);
      }
      peak = RowMax<ROWS>(peak);
      if (__any(peak > m + kSlack)) {
        const float top = peak > m + kSlack ? peak : m;
        const float shrink = top == -__builtin_inff() ? 1.0F : __builtin_amdgcn_exp2f(m - top);
        m = top;
        large = __any(fabsf(m) > kLarge && m > -__builtin_inff());
        l[0] *= shrink;
        l[1] *= shrink;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
          o[t] *= shrink;
      }
      const float from = m == -__builtin_inff() ? 0.0F : m;
      if (__builtin_expect(large, 0)) {
        // Row by row, and the exponents at once: no row's bits depend on another's size.
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < kOfGroup; ++r)
            s[g][r] = fabsf(from) > kLarge ? s[g][r] * factor[g] - from
                                           : __builtin_fmaf(s[g][r], factor[g], -from);
        factor[0] = factor[1] = 1.0F;
      }
      const float less = large ? 0.0F : from;
      typename X::x2 w2[2][kOfGroup / 2];  // the weights
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < kOfGroup; r += 2) {
          w2[g][r / 2] = X::Round(
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[g][r], factor[g], -less)),
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[g][r + 1], factor[g], -less)));
          l[r / 2 % 2] = X::AddPair(w2[g][r / 2], l[r / 2 % 2]);
        }
      if constexpr (ROWS == 16) {
        const x8 weights = {w2[0][0][0], w2[0][0][1], w2[0][1][0], w2[0][1][1],
                            w2[1][0][0], w2[1][0][1], w2[1][1][0], w2[1][1][1]};
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const unsigned lo = d.v[0][t / 4][t % 4], hi = d.v[1][t / 4][t % 4];
          const typename X::x2 a = X::Low(lo, unit[0]), b = X::High(lo, unit[0]);
          const typename X::x2 e = X::Low(hi, unit[1]), f = X::High(hi, unit[1]);
          const x8 operand{a[0], a[1], b[0], b[1], e[0], e[1], f[0], f[1]};
          o[t] = X::Mfma16(operand, weights, o[t]);
        }
      } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const x8 weights = {w2[g][0][0], w2[g][0][1], w2[g][1][0], w2[g][1][1],
                              w2[g][2][0], w2[g][2][1], w2[g][3][0], w2[g][3][1]};
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            o[t] = X::Mfma32(Operand<T>(d.v[g][0][t], d.v[g][1][t], unit[g]), weights, o[t]);
        }
      }
    };

    // A step's codes are on their way while the one before is worked on. With 16 rows
    // the loop is kept small and not unrolled: a short call runs it a few times only,
    // from an instruction cache that has not seen it (430 keys: 7.0 us of the kernel,
    // 8.2 unrolled four times); with 32 rows two steps save the copies of the codes
    // (two causal prompts of up to 5000 tokens 238 -> 231 us). The load past the end
    // fetches the last step again, under no condition, so that the waits stay exact.
    Codes now;
    load(window, &now);
    w.LoadScales(p, lane);  // behind the first codes, which only wait for the pages
    if (w.loud > loud) {
      const float shrink = loud * InversePower(w.loud);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        o[t] *= shrink;
      loud = w.loud;
    }
    if constexpr (ROWS == 16) {
#pragma unroll 1
      for (int key = window; key < window_stop; key += 32) {
        Codes next;
        load(key + 32, &next);
        step(key, now);
        now = next;
      }
    } else {
#pragma unroll 1
      for (int key = window; key < window_stop; key += 64) {
        Codes next;
        load(key + 32, &next);
        step(key, now);
        if (key + 32 >= window_stop)
          break;
        load(key + 64, &now);
        step(key + 32, next);
      }
    }
    window = window_stop;
  }

  if constexpr (OWN) {
    const float sum = RowSum<ROWS>(l[0] + l[1]);
    if (row >= rows)
      return;
    const float above = PowerAbove(sum);
    const float held = loud * InversePower(above);
    const float scale = sum == 0.0F ? 0.0F : above / sum;
    T* to = static_cast<T*>(p.out) + static_cast<std::int64_t>(span.first + query) * p.out_stride +
            static_cast<std::int64_t>(head * p.group + of_group) * DIM;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < kFours; ++i) {
        T rounded[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          rounded[r] = static_cast<T>(o[t][4 * i + r] * held * scale);
        __builtin_memcpy(to + DimOf<DIM, ROWS>(t * kFours + i, part), rounded, sizeof(rounded));
      }
    return;
  }
  __shared__ float shared_m[kWaves][ROWS], shared_l[kWaves][ROWS];
  __shared__ floatx4 shared_o[kWaves][kTiles * kFours][64];
  const float sum = RowSum<ROWS>(l[0] + l[1]);
  if (part == 0) {
    shared_m[wave][column] = m;
    shared_l[wave][column] = sum;
  }
  const float held = loud * InversePower(PowerAbove(sum));
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < kFours; ++i)
      shared_o[wave][t * kFours + i][lane] =
          floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]} * held;
  __syncthreads();
  float top = -__builtin_inff(), total = 0.0F;
  float weight[kWaves];
#pragma unroll
  for (int i = 0; i < kWaves; ++i)
    top = fmaxf(top, shared_m[i][column]);
  const float from = top == -__builtin_inff() ? 0.0F : top;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    weight[i] = __builtin_amdgcn_exp2f(shared_m[i][column] - from);
    total += shared_l[i][column] * weight[i];
  }
  if (row >= rows)
    return;
  const float above = PowerAbove(total);
#pragma unroll
  for (int i = 0; i < kWaves; ++i)
    weight[i] *= PowerAbove(shared_l[i][column]) * InversePower(above);
  const std::size_t slot =
      p.splits == 1
          ? 0
          : ((static_cast<std::size_t>(item) * c.kv_heads + head) * p.splits + blockIdx.z) * ROWS +
                column;
  if (p.splits > 1 && wave == 0 && part == 0) {
    p.partial_m[2 * slot] = top;
    p.partial_m[2 * slot + 1] = total;
  }
  // Nothing seen: zero.
  const float scale = total == 0.0F ? 0.0F : above / total;
  T* to = static_cast<T*>(p.out) + static_cast<std::int64_t>(span.first + query) * p.out_stride +
          static_cast<std::int64_t>(head * p.group + of_group) * DIM;
#pragma unroll
  for (int j = wave; j < kTiles * kFours; j += kWaves) {
    floatx4 sum = {};
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      sum += shared_o[i][j][lane] * weight[i];
    const int dim = DimOf<DIM, ROWS>(j, part);
    if (p.splits > 1) {
      *reinterpret_cast<floatx4*>(p.partial_o + slot * DIM + dim) = sum;
    } else {
      T rounded[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        rounded[r] = static_cast<T>(sum[r] * scale);
      __builtin_memcpy(to + dim, rounded, sizeof(rounded));
    }
  }
}

// A split has left its row's maximum and sum of weights, and its output over the power
// of two above that sum.
// Joins the splits of one row: DIM / 4 lanes hold four of its dims each, and the
// work-group's 256 / (DIM / 4) such groups take its splits in turn.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void JoinKernel(CacheAttentionParams p) {
  constexpr int kLanes = DIM / 4, kGroups = 256 / kLanes;
  const CacheView& c = p.cache;
  const int item = p.first_item + static_cast<int>(blockIdx.y);
  const Found found = FindItem(c, p.group, p.tile_shift, 1, item);
  const int tile = found.item;
  const Span span = found.span;
  const int rows = span.count * p.group;
  const int in_tile = blockIdx.z;
  const int row = (tile << p.tile_shift) + in_tile;
  if (tile < 0 || row >= rows)
    return;
  const int head = blockIdx.x;
  const int tid = threadIdx.x, group = tid / kLanes, part = tid % kLanes;
  const std::size_t first =
      (((static_cast<std::size_t>(item) * c.kv_heads + head) * p.splits) << p.tile_shift) +
      in_tile;
  __shared__ float weights[kMostSplits];
  __shared__ float wave_top[4];
  __shared__ float totals[4];
  __shared__ floatx4 sums[kGroups][kLanes];
  float m = -__builtin_inff(), l = 0.0F;
  if (tid < p.splits) {
    const std::size_t slot = first + (static_cast<std::size_t>(tid) << p.tile_shift);
    m = p.partial_m[2 * slot];
    l = p.partial_m[2 * slot + 1];
  }
  float top = WaveMax(m);
  if ((tid & 63) == 0)
    wave_top[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
  const float from = top == -__builtin_inff() ? 0.0F : top;
  const float weight = __builtin_amdgcn_exp2f(m - from);
  if (tid < kMostSplits)
    weights[tid] = weight * PowerAbove(l);
  const float part_total = WaveSum(l * weight);
  if ((tid & 63) == 0)
    totals[tid >> 6] = part_total;
  __syncthreads();
  const float total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
  const float above = PowerAbove(total), held = InversePower(above);
  // Eight loads at a time, none under a condition: a split that saw nothing has
  // left zeros.
  constexpr int kAhead = 8;
  floatx4 sum = {};
  for (int s0 = group; s0 < p.splits; s0 += kAhead * kGroups) {
    floatx4 o[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int s = min(s0 + a * kGroups, p.splits - 1);
      const std::size_t slot = first + (static_cast<std::size_t>(s) << p.tile_shift);
      o[a] = *reinterpret_cast<const floatx4*>(p.partial_o + slot * DIM + 4 * part);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (s0 + a * kGroups < p.splits)
        sum += o[a] * (weights[s0 + a * kGroups] * held);
  }
  sums[group][part] = sum;
  __syncthreads();
  if (group != 0)
    return;
#pragma unroll
  for (int g = 1; g < kGroups; ++g)
    sum += sums[g][part];
  const float scale = total == 0.0F ? 0.0F : above / total;
  int of_group;
  const int query = RowSplit(p, row).Of(0, &of_group);
  T rounded[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    rounded[r] = static_cast<T>(sum[r] * scale);
  __builtin_memcpy(static_cast<T*>(p.out) +
                       static_cast<std::int64_t>(span.first + query) * p.out_stride +
                       static_cast<std::int64_t>(head * p.group + of_group) * DIM + 4 * part,
                   rounded, sizeof(rounded));
}

// Few splits: each group of DIM / 4 lanes joins a row of its own.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void JoinFewKernel(CacheAttentionParams p) {
  constexpr int kLanes = DIM / 4, kGroups = 256 / kLanes;
  const CacheView& c = p.cache;
  const int item = p.first_item + static_cast<int>(blockIdx.y);
  const Found found = FindItem(c, p.group, p.tile_shift, 1, item);
  const int tile = found.item;
  const Span span = found.span;
  const int rows = span.count * p.group;
  const int tid = threadIdx.x, part = tid % kLanes;
  const int in_tile = blockIdx.z * kGroups + tid / kLanes;
  const int row = (tile << p.tile_shift) + in_tile;
  if (tile < 0 || row >= rows)
    return;
  const int head = blockIdx.x;
  const std::size_t first =
      (((static_cast<std::size_t>(item) * c.kv_heads + head) * p.splits) << p.tile_shift) +
      in_tile;
  float m[kFewSplits], l[kFewSplits];
  floatx4 o[kFewSplits];
  float top = -__builtin_inff();
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const std::size_t slot =
        first + (static_cast<std::size_t>(min(s, p.splits - 1)) << p.tile_shift);
    m[s] = p.partial_m[2 * slot];
    l[s] = s < p.splits ? p.partial_m[2 * slot + 1] : 0.0F;
    o[s] = *reinterpret_cast<const floatx4*>(p.partial_o + slot * DIM + 4 * part);
    top = fmaxf(top, m[s]);
  }
  const float from = top == -__builtin_inff() ? 0.0F : top;
  float total = 0.0F;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    m[s] = __builtin_amdgcn_exp2f(m[s] - from);
    total += l[s] * m[s];
  }
  const float above = PowerAbove(total), held = InversePower(above);
  floatx4 sum = {};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s)
    if (s < p.splits)
      sum += o[s] * (m[s] * (PowerAbove(l[s]) * held));
  const float scale = total == 0.0F ? 0.0F : above / total;
  int of_group;
  const int query = RowSplit(p, row).Of(0, &of_group);
  T rounded[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    rounded[r] = static_cast<T>(sum[r] * scale);
  __builtin_memcpy(static_cast<T*>(p.out) +
                       static_cast<std::int64_t>(span.first + query) * p.out_stride +
                       static_cast<std::int64_t>(head * p.group + of_group) * DIM + 4 * part,
                   rounded, sizeof(rounded));
}

constexpr int kMostItems = 65535;  // of a grid's second dimension

template <typename T, int DIM>
void Launch(const CacheAttentionParams& p, hipStream_t stream) {
  const bool one = p.cache.block_shift > 4, last = p.splits == 1;
  const auto kernel = p.tile_shift == 4 ? one ? CacheAttentionKernel<T, DIM, 16, true, false>
                                              : CacheAttentionKernel<T, DIM, 16, false, false>
                      : p.own_shift > 0
                          ? one ? CacheAttentionKernel<T, DIM, 32, true, true>
                                : CacheAttentionKernel<T, DIM, 32, false, true>
                      : one ? CacheAttentionKernel<T, DIM, 32, true, false>
                            : CacheAttentionKernel<T, DIM, 32, false, false>;
  constexpr int kJoined = 256 / (DIM / 4);  // rows of a work-group with few splits
  const int in_tile = 1 << p.tile_shift;
  CacheAttentionParams part = p;
  part.items = ItemBound(p.cache, p.group, p.tile_shift + p.own_shift, 1);
  // A launch holds 65535 items; the heads come first, so that with 8 of them the
  // tiles of a head share their XCD's L2.
  for (part.first_item = 0; part.first_item < part.items; part.first_item += kMostItems) {
    const int items = std::min(part.items - part.first_item, kMostItems);
    const bool first = part.first_item == 0, end = part.first_item + items == part.items;
    Dispatch(kernel, dim3(p.cache.kv_heads, items, p.splits), dim3(kWaves * kWave), 0, stream,
             first, end && last, part);
    if (last)
      continue;
    // The items that this launch took, counted from the last one.
    CacheAttentionParams join = part;
    join.first_item = part.items - part.first_item - items;
    if (p.splits <= kFewSplits)
      Dispatch(JoinFewKernel<T, DIM>,
               dim3(p.cache.kv_heads, items, (in_tile + kJoined - 1) / kJoined), dim3(256), 0,
               stream, false, end, join);
    else
      Dispatch(JoinKernel<T, DIM>, dim3(p.cache.kv_heads, items, in_tile), dim3(256), 0, stream,
               false, end, join);
  }
}

}  // namespace

CacheAttentionPlan PlanCacheAttention(const CacheView& c, int group) {
  CacheAttentionPlan plan;
  if (c.rows == 0)
    return plan;
  // Rows of a sequence on average: 16 columns of the matrix operand where they
  // suffice, else 32.
  const std::int64_t all = static_cast<std::int64_t>(c.rows) * group;
  const bool few = all <= 16ll * c.count;
  plan.tile_shift = few ? 4 : 5;
  const int items = ItemBound(c, group, plan.tile_shift, 1);
  const std::int64_t groups = static_cast<std::int64_t>(items) * c.kv_heads;
  const std::int64_t capacity = static_cast<std::int64_t>(c.table_width) << c.block_shift;
  std::int64_t wanted = kSplitGroups / groups, least = kLeastTileChunk;
  if (few && groups < kFullGroups) {
    wanted = capacity < kLeastSplit ? 1 : kFullGroups / groups;
    least = kLeastChunk;
  } else if (few) {
    wanted = kRaggedGroups / groups;
  }
  plan.splits = static_cast<int>(std::max<std::int64_t>(
      1, std::min({wanted, capacity / least, std::int64_t{kMostSplits}})));
  const std::int64_t fill = kOwnTiles * 128 / c.dim;
  if (plan.splits == 1 && !few &&
      (capacity <= kOwnKeys ? groups >= fill : c.dim == 128 && groups >= 2 * fill))
    plan.own_shift = 2;
  if (plan.splits > 1)
    plan.slots = (static_cast<std::size_t>(groups) * plan.splits) << plan.tile_shift;
  return plan;
}

void LaunchCacheAttention(const CacheAttentionParams& p, DType type, hipStream_t stream) {
  if (p.cache.rows == 0)
    return;
  if (type == DType::kF16)
    p.cache.dim == 64 ? Launch<_Float16, 64>(p, stream) : Launch<_Float16, 128>(p, stream);
  else
    p.cache.dim == 64 ? Launch<__bf16, 64>(p, stream) : Launch<__bf16, 128>(p, stream);
  Check(hipGetLastError(), "cache attention launch");
}

}  // namespace ovg
