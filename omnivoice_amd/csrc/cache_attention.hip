// Attention over the 8-bit key/value cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j that a query sees
//
// The rows of a kv head are its query heads' queries, row r of a sequence
// being query r / group of head r % group: the whole group shares every key
// and value that is loaded. Scores are formed transposed, S^T = K Q^T, so a
// lane owns one row's column, and so is the output, O^T = V^T P^T, whose P^T
// operand is the scores' accumulator itself (v_mfma_f32_16x16x32: lane l
// holds row l % 16 and, of every 16 keys, keys 4 (l / 16) .. + 3). e4m3 codes
// are exact in fp16 and bf16, so the products see the queries and codes as
// they are: the keys' scale joins the softmax's in the float32 scores, the
// values' the float32 sums. The one rounding on the way is that of the
// probabilities to the queries' type, and the row's sum takes the rounded
// ones, so that the weights still add up to one.
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
// 0 for a block without a (numeric) scale.
__device__ __forceinline__ float Loudness(float scale) { return scale == scale ? scale : 0.0F; }

// How far a row's maximum may rise before its sums are scaled again: their
// probabilities are then at most 2^8, far inside fp16, and most steps of a long
// row leave the sums alone. Each row goes by its own maximum: what the others
// hold changes none of its bits.
constexpr float kSlack = 8.0F;

constexpr int kFewWaves = 4;

// A wave's window of the block table: lane i holds the page and scales of the
// i-th block, so that the steps wait for the table once per 64 blocks and not
// one after the other.
struct Window {
  int page;
  float factor;  // of the scores, to the exponent of two; NaN where the block is
  float level;   // the values' loudness
  __device__ __forceinline__ void Load(const CacheAttentionParams& p, int sequence, int head,
                                       int first, int stop, int lane) {
    const CacheView& c = p.cache;
    const int block = first + lane;
    page = (block << c.block_shift) < stop ? PageOf(c, sequence, block) : -1;
    const std::size_t at = ScaleIndex(c, max(page, 0), head, 0);
    const float k_scale = c.scales[at], v_scale = c.scales[at + 1];
    // A NaN scale, of keys or values, makes the block's scores NaN.
    factor = page < 0 ? 0.0F : p.scale_log2 * k_scale + 0.0F * v_scale;
    level = page < 0 ? 0.0F : Loudness(v_scale);
  }
};

// Few rows: a work-group takes 16 NT rows of one sequence and kv head and one
// split of its keys; each of its four waves takes a quarter of them in steps of
// 32, with a softmax of its own that runs along (maximum m, sum l, output o), and
// the four are joined in LDS at the end. The codes go from memory straight into
// registers, a step ahead, and are converted there: with few rows nothing is
// gained by sharing them, and what bounds the kernel is the stream of codes.
template <typename T, int DIM, int NT>
__global__ __launch_bounds__(kFewWaves* kWave) void FewRowsKernel(CacheAttentionParams p) {
  typedef Types<T> X;
  typedef typename X::x8 x8;
  constexpr int kSteps = DIM / 64;  // 16-byte loads of a key's codes in a lane
  constexpr int kTiles = DIM / 16;
  constexpr int kRows = 16 * NT;
  const CacheView& c = p.cache;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15, quad = lane >> 4;
  const int head = blockIdx.x;

  int tile = blockIdx.y;
  const int sequence =
      __builtin_amdgcn_readfirstlane(SequenceOfItem(c, p.group, NT == 1 ? 4 : 5, 1, &tile));
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Span span = SpanOf(c, sequence);
  const int rows = span.count * p.group;
  if (tile < 0 || tile * kRows >= rows)
    return;
  const int length = min(span.length, c.table_width << c.block_shift);
  // Keys that any row of the tile sees, and those of this split.
  const int last = min(tile * kRows + kRows, rows) - 1;
  const int end = p.causal ? min(span.start + last / p.group + 1, length) : length;
  const int chunk = ChunkOf(length, p.splits);
  const int begin = blockIdx.z * chunk;
  const int stop = min(begin + chunk, end);

  int query[NT], of_group[NT], seen[NT];
  x8 q[NT][kSteps][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = tile * kRows + 16 * n + column;
    query[n] = min(row, rows - 1) / p.group;
    of_group[n] = min(row, rows - 1) - query[n] * p.group;
    seen[n] = row >= rows ? 0 : p.causal ? min(span.start + query[n] + 1, length) : length;
    const T* from = static_cast<const T*>(p.q) +
                    static_cast<std::int64_t>(span.first + query[n]) * p.q_stride +
                    static_cast<std::int64_t>(head * p.group + of_group[n]) * DIM + 16 * quad;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      __builtin_memcpy(&q[n][i][0], from + 64 * i, sizeof(x8));
      __builtin_memcpy(&q[n][i][1], from + 64 * i + 8, sizeof(x8));
    }
    if (p.negate) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        q[n][i][0] = -q[n][i][0];
        q[n][i][1] = -q[n][i][1];
      }
    }
  }

  float m[NT], l[NT];
  floatx4 o[NT][kTiles];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -__builtin_inff();
    l[n] = 0.0F;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      o[n][t] = floatx4{0.0F, 0.0F, 0.0F, 0.0F};
  }
  float loud = kQuietest;

  const int quarter = ((stop - begin + kFewWaves * 32 - 1) / (kFewWaves * 32)) * 32;
  const int wave_begin = begin + wave * quarter;
  const int wave_stop = min(wave_begin + quarter, stop);
  const int in_block = (1 << c.block_shift) - 1;
  const std::size_t half_bytes = static_cast<std::size_t>(DIM) << c.block_shift;

  for (int window = wave_begin; window < wave_stop;) {
    Window w;
    const int first_block = window >> c.block_shift;
    w.Load(p, sequence, head, first_block, wave_stop, lane);
    const int window_stop = min((first_block + kWave) << c.block_shift, wave_stop);

    struct Codes {
      u32x4 k[2][kSteps], v[2][kSteps];
    };
    const auto load = [&](int key, Codes* d) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int at = min(key, window_stop - 1) + 16 * g;
        const int block = min((at >> c.block_shift) - first_block, kWave - 1);
        const int page = max(__builtin_amdgcn_readlane(w.page, block), 0);
        const unsigned char* from =
            c.data + (static_cast<std::size_t>(page) * c.kv_heads + head) * 2 * half_bytes +
            static_cast<std::size_t>(at & in_block & ~15) * DIM;
        const u32x4* kc = reinterpret_cast<const u32x4*>(from);
        const u32x4* vc = reinterpret_cast<const u32x4*>(from + half_bytes);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          d->k[g][i] = kc[i * 64 + lane];
          d->v[g][i] = vc[i * 64 + lane];
        }
      }
    };
    const auto step = [&](int key, const Codes& d) {
      float factor[2], level[2];
      bool there[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int block = ((key + 16 * g) >> c.block_shift) - first_block;
        factor[g] = Lane(w.factor, block);
        level[g] = Lane(w.level, block);
        there[g] = __builtin_amdgcn_readlane(w.page, block) >= 0;
      }
      const float louder = fmaxf(loud, fmaxf(level[0], level[1]));
      if (louder > loud) {
        const float shrink = loud * InversePower(louder);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            o[n][t] *= shrink;
        loud = louder;
      }
      const float unit = InversePower(loud);
      x8 weights[NT];
      floatx4 acc[NT][2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          acc[n][g] = floatx4{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const x8 a = Operand<T>(d.k[g][i][0], d.k[g][i][1], 1.0F);
          const x8 b = Operand<T>(d.k[g][i][2], d.k[g][i][3], 1.0F);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n][g] = X::Mfma16(a, q[n][i][0], acc[n][g]);
            acc[n][g] = X::Mfma16(b, q[n][i][1], acc[n][g]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float s[2][4];
        float peak = -__builtin_inff();
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool visible = there[g] && key + 16 * g + 4 * quad + r < seen[n];
            s[g][r] = visible ? acc[n][g][r] * factor[g] : -__builtin_inff();
            peak = fmaxf(peak, s[g][r]);
          }
        peak = Max32(Max16(peak));
        if (__any(peak > m[n] + kSlack)) {
          const float top = peak > m[n] + kSlack ? peak : m[n];
          const float shrink =
              top == -__builtin_inff() ? 1.0F : __builtin_amdgcn_exp2f(m[n] - top);
          m[n] = top;
          l[n] *= shrink;
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            o[n][t] *= shrink;
        }
        const float from = m[n] == -__builtin_inff() ? 0.0F : m[n];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const typename X::x2 pair = X::Round(__builtin_amdgcn_exp2f(s[g][r] - from),
                                                 __builtin_amdgcn_exp2f(s[g][r + 1] - from));
            weights[n][4 * g + r] = pair[0];
            weights[n][4 * g + r + 1] = pair[1];
            l[n] = X::AddPair(pair, l[n]);
          }
      }
      const float v0 = fmaxf(level[0] * unit, kQuietest), v1 = fmaxf(level[1] * unit, kQuietest);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const unsigned lo = d.v[0][t / 4][t % 4], hi = d.v[1][t / 4][t % 4];
        const typename X::x2 a = X::Low(lo, v0), b = X::High(lo, v0);
        const typename X::x2 e = X::Low(hi, v1), f = X::High(hi, v1);
        const x8 operand{a[0], a[1], b[0], b[1], e[0], e[1], f[0], f[1]};
#pragma unroll
        for (int n = 0; n < NT; ++n)
          o[n][t] = X::Mfma16(operand, weights[n], o[n][t]);
      }
    };

    Codes even, odd;
    load(window, &even);
    for (int key = window; key < window_stop; key += 64) {
      load(key + 32, &odd);
      step(key, even);
      if (key + 32 < window_stop) {
        load(key + 64, &even);
        step(key + 32, odd);
      }
    }
    window = window_stop;
  }

  __shared__ float shared_m[kFewWaves][kRows], shared_l[kFewWaves][kRows];
  __shared__ floatx4 shared_o[kFewWaves][NT * kTiles][64];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = Sum32(Sum16(l[n]));
    if (quad == 0) {
      shared_m[wave][16 * n + column] = m[n];
      shared_l[wave][16 * n + column] = l[n];
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      shared_o[wave][n * kTiles + t][lane] = o[n][t] * loud;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int in_tile = 16 * n + column;
    const int row = tile * kRows + in_tile;
    float top = -__builtin_inff(), total = 0.0F;
    float weight[kFewWaves];
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
      top = fmaxf(top, shared_m[w][in_tile]);
    const float from = top == -__builtin_inff() ? 0.0F : top;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      weight[w] = __builtin_amdgcn_exp2f(shared_m[w][in_tile] - from);
      total += shared_l[w][in_tile] * weight[w];
    }
    if (row >= rows)
      continue;
    const std::size_t slot =
        p.splits == 1
            ? 0
            : ((static_cast<std::size_t>(blockIdx.y) * c.kv_heads + head) * p.splits +
               blockIdx.z) * kRows + in_tile;
    if (p.splits > 1 && wave == 0 && quad == 0) {
      p.partial_m[2 * slot] = top;
      p.partial_m[2 * slot + 1] = total;
    }
    // Nothing seen: zero.
    const float scale = total == 0.0F ? 0.0F : 1.0F / total;
    T* to = static_cast<T*>(p.out) +
            static_cast<std::int64_t>(span.first + query[n]) * p.out_stride +
            static_cast<std::int64_t>(head * p.group + of_group[n]) * DIM + 4 * quad;
    for (int t = wave; t < kTiles; t += kFewWaves) {
      floatx4 sum = {};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w)
        sum += shared_o[w][n * kTiles + t][lane] * weight[w];
      if (p.splits > 1) {
        *reinterpret_cast<floatx4*>(p.partial_o + slot * DIM + 16 * t + 4 * quad) = sum;
      } else {
        T rounded[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          rounded[r] = static_cast<T>(sum[r] * scale);
        __builtin_memcpy(to + 16 * t, rounded, sizeof(rounded));
      }
    }
  }
}

constexpr int kManyWaves = 4;
constexpr int kManyRows = 32 * kManyWaves;

// The same for tiles of many rows, whose values are converted for all at once:
// lane i holds where its block's head begins, the scores' factor, and the
// values' scale over `loud`, the loudest of this window's blocks and all before.
struct TileWindow {
  unsigned offset_low, offset_high;
  float factor, unit;
  float loud;                // the same in every lane
  unsigned long long there;  // a bit for each block that there is
  __device__ __forceinline__ void Load(const CacheAttentionParams& p, int sequence, int head,
                                       int first, int stop, int lane) {
    const CacheView& c = p.cache;
    const int block = first + lane;
    const int page = (block << c.block_shift) < stop ? PageOf(c, sequence, block) : -1;
    there = __ballot(page >= 0);
    const std::size_t at = ScaleIndex(c, max(page, 0), head, 0);
    const float k_scale = c.scales[at], v_scale = c.scales[at + 1];
    const std::size_t offset = at * (static_cast<std::size_t>(c.dim) << c.block_shift);
    offset_low = static_cast<unsigned>(offset);
    offset_high = static_cast<unsigned>(offset >> 32);
    // A NaN scale, of keys or values, makes the block's scores NaN.
    factor = page < 0 ? 0.0F : p.scale_log2 * k_scale + 0.0F * v_scale;
    const float level = page < 0 ? 0.0F : Loudness(v_scale);
    loud = fmaxf(loud, WaveMax(level));
    unit = fmaxf(level * InversePower(loud), kQuietest);
  }
  __device__ __forceinline__ const unsigned char* Base(const unsigned char* data, int i) const {
    const std::size_t low = __builtin_amdgcn_readlane(offset_low, i);
    const std::size_t high = __builtin_amdgcn_readlane(offset_high, i);
    return data + (high << 32 | (low & 0xFFFFFFFFu));
  }
};

// What a tile needs beside its codes: a factor for each of its blocks.
template <int BLOCKS>
struct TileScales {
  typedef float vec __attribute__((ext_vector_type(BLOCKS)));
  vec factor;
  float loud;      // that its values are converted at
  float unit;      // of the values that this thread converts
  unsigned there;  // a bit for each block
};

// Many rows: a work-group of four waves takes 128 rows of one sequence and kv
// head, 32 a wave, and goes over the keys in tiles of 64 (128 at 64 dims) that
// the waves share. The threads fetch a tile's codes ahead, convert them once and
// leave them in LDS in the order of the operands of v_mfma_f32_32x32x16 (64 lanes
// of 16 bytes in a row, so every write and read is a conflict-free 16 bytes a
// lane), in two buffers of 16 KB each for keys and values. The softmax runs in
// registers, a row in a lane and its partner lane ^ 32. While a tile's
// probabilities are formed, on the vector unit, the matrix cores form the next
// tile's scores, which depend on nothing of it; so in iteration i the waves read
// keys i + 1 and values i and write keys i + 2 and values i + 1, and one barrier
// an iteration suffices.
template <typename T, int DIM, int SHIFT>
__global__ __launch_bounds__(kManyWaves* kWave, 2) void ManyRowsKernel(CacheAttentionParams p) {
  typedef Types<T> X;
  typedef typename X::x8 x8;
  constexpr int kKeys = 8192 / DIM;          // of a tile
  constexpr int kGroups = kKeys / 16, kBlocks = kKeys / 32;
  constexpr int kK = DIM / 16;               // contraction steps of the scores
  constexpr int kDims = DIM / 32;            // blocks of 32 dims
  constexpr int kChunks = DIM;               // 16-byte chunks of a group's keys or values
  constexpr int kSums = 4;                   // of a row in a lane, to be added at the end
  constexpr int kPages = kKeys >> SHIFT;     // blocks of the pool in a tile: 1 to 8
  constexpr std::size_t kHalf = static_cast<std::size_t>(DIM) << SHIFT;  // bytes
  typedef TileScales<kPages> Scales;
  __shared__ x8 key_tiles[2][kKeys * DIM / 8];
  __shared__ x8 value_tiles[2][kKeys * DIM / 8];
  const CacheView& c = p.cache;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int column = lane & 31, half = lane >> 5;
  const int head = blockIdx.x;

  // The last rows of a causal sequence see the most keys: they start first.
  const int item = gridDim.y - 1 - blockIdx.y;
  int tile = item;
  const int sequence = __builtin_amdgcn_readfirstlane(SequenceOfItem(c, p.group, 7, 1, &tile));
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Span span = SpanOf(c, sequence);
  const int rows = span.count * p.group;
  if (tile < 0 || tile * kManyRows >= rows)
    return;
  const int length = min(span.length, c.table_width << c.block_shift);
  const int last = min(tile * kManyRows + kManyRows, rows) - 1;
  const int end = p.causal ? min(span.start + last / p.group + 1, length) : length;
  const int chunk = ChunkOf(length, p.splits);
  const int begin = blockIdx.z * chunk;
  const int stop = min(begin + chunk, end);

  const int first_row = tile * kManyRows + 32 * wave;
  const int row = first_row + column;
  const int query = min(row, rows - 1) / p.group;
  const int of_group = min(row, rows - 1) - query * p.group;
  const int seen = row >= rows ? 0 : p.causal ? min(span.start + query + 1, length) : length;
  // Keys that every row of the wave sees, and that any does.
  const int all_see = first_row + 31 >= rows ? 0
                      : p.causal             ? min(span.start + first_row / p.group + 1, length)
                                             : length;
  const int wave_end =
      first_row >= rows ? 0
      : p.causal ? min(span.start + min(first_row + 31, rows - 1) / p.group + 1, length)
                 : length;

  x8 q[kK];
  {
    const T* from = static_cast<const T*>(p.q) +
                    static_cast<std::int64_t>(span.first + query) * p.q_stride +
                    static_cast<std::int64_t>(head * p.group + of_group) * DIM + 8 * half;
#pragma unroll
    for (int i = 0; i < kK; ++i)
      __builtin_memcpy(&q[i], from + 16 * i, sizeof(x8));
    if (p.negate) {
#pragma unroll
      for (int i = 0; i < kK; ++i)
        q[i] = -q[i];
    }
  }

  float m = -__builtin_inff();
  float l[kSums] = {};
  floatx16 o[kDims];
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      o[t][r] = 0.0F;
  float loud = kQuietest;

  TileWindow window;
  window.loud = kQuietest;
  int window_first = 0, window_stop = begin;  // block, key

  // A thread's chunks of a tile: two of keys (chunk tid + 256 i: group, dims / 16,
  // token) and a pair of values (group, dims / 64, quad and quad + 2, dim % 16), whose
  // eight tokens make one lane's operand.
  const int value_group = tid / (DIM / 2), value_at = tid % (DIM / 2);
  const int value_chunk = (value_at >> 5) * 64 + (value_at & 31);
  u32x4 k_codes[2], v_codes[2];
  // The tile's scales, the codes of its keys on their way, and where its values are.
  // A tile begins with a block or with a whole part of one.
  const auto fetch_keys = [&](int key, const u32x4** values) {
    if (key >= window_stop) {  // never in the middle of a tile: 64 blocks are whole ones
      window_first = key >> SHIFT;
      window.Load(p, sequence, head, window_first, stop, lane);
      window_stop = (window_first + kWave) << SHIFT;
    }
    const int block = (key >> SHIFT) - window_first;
    const auto base = [&](int group) {
      return window.Base(c.data, block + ((16 * group) >> SHIFT)) +
             (16 * group & ((1 << SHIFT) - 1)) * DIM;
    };
    Scales s;
    s.loud = window.loud;
    s.there = static_cast<unsigned>(window.there >> block) & ((1u << kPages) - 1);
#pragma unroll
    for (int g = 0; g < kPages; ++g)
      s.factor[g] = Lane(window.factor, block + g);
    if constexpr (DIM == 128) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        k_codes[i] = reinterpret_cast<const u32x4*>(
            base(2 * i + (wave >> 1)))[(wave & 1) * 64 + lane];
      *values = reinterpret_cast<const u32x4*>(base(wave) + kHalf) + value_chunk;
      s.unit = Lane(window.unit, block + ((16 * wave) >> SHIFT));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        k_codes[i] = reinterpret_cast<const u32x4*>(base(4 * i + wave))[lane];
      const unsigned char* even = base(2 * wave);
      const unsigned char* odd = base(2 * wave + 1);
      *values = reinterpret_cast<const u32x4*>((half == 0 ? even : odd) + kHalf) + value_chunk;
      const float even_unit = Lane(window.unit, block + ((32 * wave) >> SHIFT));
      const float odd_unit = Lane(window.unit, block + ((32 * wave + 16) >> SHIFT));
      s.unit = half == 0 ? even_unit : odd_unit;
    }
    return s;
  };
  const auto fetch_values = [&](const u32x4* values) {
    v_codes[0] = values[0];
    v_codes[1] = values[32];
  };
  const auto convert_keys = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int index = tid + i * 256;
      const int group = index / kChunks, at = index % kChunks;
      x8* to = key_tiles[buffer] + ((group >> 1) * kK + (at >> 4)) * 64 + (group & 1) * 16 +
               (at & 15);
      to[0] = Operand<T>(k_codes[i][0], k_codes[i][1], 1.0F);
      to[32] = Operand<T>(k_codes[i][2], k_codes[i][3], 1.0F);
    }
  };
  const auto convert_values = [&](const Scales& s, int buffer) {
    const int d = value_at & 15, h = (value_at >> 4) & 1, quarter = value_at >> 5;
    x8* to = value_tiles[buffer] + (value_group * kDims + 2 * quarter) * 64 + 32 * h + d;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      to[(t >> 1) * 64 + (t & 1) * 16] = Operand<T>(v_codes[0][t], v_codes[1][t], s.unit);
  };
  floatx16 scores[kBlocks];
  const auto score = [&](int buffer, floatx16 (&to)[kBlocks]) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      floatx16 acc;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[r] = 0.0F;
#pragma unroll
      for (int i = 0; i < kK; ++i)
        acc = X::Mfma32(key_tiles[buffer][(b * kK + i) * 64 + lane], q[i], acc);
      to[b] = acc;
    }
  };

  if (begin < stop) {
    // Tiles now, one and two ahead; past the last one the scales and codes of
    // whatever block 0 holds, which nothing takes.
    const u32x4 *values, *values_next, *values_after;
    Scales now = fetch_keys(begin, &values);
    fetch_values(values);
    convert_keys(0);
    convert_values(now, 0);
    Scales next = fetch_keys(begin + kKeys, &values_next);
    fetch_values(values_next);
    convert_keys(1);
    Scales after = fetch_keys(begin + 2 * kKeys, &values_after);
    __syncthreads();
    score(0, scores);
    __syncthreads();
    int buffer = 0;  // of this tile's keys and values
    for (int key = begin; key < stop; key += kKeys) {
      if (now.loud > loud) {
        const float shrink = loud * InversePower(now.loud);
#pragma unroll
        for (int t = 0; t < kDims; ++t)
          o[t] *= shrink;
        loud = now.loud;
      }
      if (key < wave_end) {
        typename Scales::vec factor = now.factor;
        const auto page_of = [](int group) { return (16 * group) >> SHIFT; };
        if (now.there != (1u << kPages) - 1 || key + kKeys > all_see) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const int e = 8 * (g & 1) + r;
              const int at = key + 16 * g + 8 * (r / 4) + 4 * half + r % 4;
              scores[g / 2][e] = (now.there >> page_of(g) & 1) != 0 && at < seen
                                     ? scores[g / 2][e] * factor[page_of(g)]
                                     : -__builtin_inff();
            }
#pragma unroll
          for (int g = 0; g < kPages; ++g)
            factor[g] = 1.0F;
        }
        float peak = -__builtin_inff();
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float most = -__builtin_inff();
#pragma unroll
          for (int r = 0; r < 8; ++r)
            most = fmaxf(most, scores[g / 2][8 * (g & 1) + r]);
          peak = fmaxf(peak, most * factor[page_of(g)]);
        }
        peak = Max32(peak);
        if (__any(peak > m + kSlack)) {
          const float top = peak > m + kSlack ? peak : m;
          const float shrink = top == -__builtin_inff() ? 1.0F : __builtin_amdgcn_exp2f(m - top);
          m = top;
#pragma unroll
          for (int i = 0; i < kSums; ++i)
            l[i] *= shrink;
#pragma unroll
          for (int t = 0; t < kDims; ++t)
            o[t] *= shrink;
        }
        const float from = m == -__builtin_inff() ? 0.0F : m;
        floatx16 coming[kBlocks];
        score(buffer ^ 1, coming);
        x8 weights[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const int e = 8 * (g & 1) + r;
            const typename X::x2 pair = X::Round(
                __builtin_amdgcn_exp2f(__builtin_fmaf(scores[g / 2][e], factor[page_of(g)], -from)),
                __builtin_amdgcn_exp2f(__builtin_fmaf(scores[g / 2][e + 1], factor[page_of(g)], -from)));
            weights[g][r] = pair[0];
            weights[g][r + 1] = pair[1];
            l[r / 2] = X::AddPair(pair, l[r / 2]);
          }
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int t = 0; t < kDims; ++t)
            o[t] = X::Mfma32(value_tiles[buffer][(g * kDims + t) * 64 + lane], weights[g], o[t]);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
          scores[b] = coming[b];
        convert_keys(buffer);
        convert_values(next, buffer ^ 1);
      } else {
        convert_keys(buffer);
        convert_values(next, buffer ^ 1);
      }
      fetch_values(values_after);
      now = next;
      next = after;
      after = fetch_keys(key + 3 * kKeys, &values_after);
      buffer ^= 1;
      __syncthreads();
    }
  }

  const float total = Sum32((l[0] + l[1]) + (l[2] + l[3]));
  if (row >= rows)
    return;
  if (p.splits > 1) {
    const std::size_t slot =
        ((static_cast<std::size_t>(item) * c.kv_heads + head) * p.splits + blockIdx.z) *
            kManyRows + 32 * wave + column;
    if (half == 0) {
      p.partial_m[2 * slot] = m;
      p.partial_m[2 * slot + 1] = total;
    }
#pragma unroll
    for (int t = 0; t < kDims; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const floatx4 part = {o[t][r] * loud, o[t][r + 1] * loud, o[t][r + 2] * loud,
                              o[t][r + 3] * loud};
        *reinterpret_cast<floatx4*>(p.partial_o + slot * DIM + 32 * t + 2 * r + 4 * half) = part;
      }
    return;
  }
  // Nothing seen: zero.
  const float scale = total == 0.0F ? 0.0F : loud / total;
  T* to = static_cast<T*>(p.out) + static_cast<std::int64_t>(span.first + query) * p.out_stride +
          static_cast<std::int64_t>(head * p.group + of_group) * DIM + 4 * half;
#pragma unroll
  for (int t = 0; t < kDims; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      T rounded[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        rounded[e] = static_cast<T>(o[t][r + e] * scale);
      __builtin_memcpy(to + 32 * t + 2 * r, rounded, sizeof(rounded));
    }
}

// Joins the splits of one row: DIM / 4 lanes hold four of its dims each, and the
// work-group's 256 / (DIM / 4) such groups take its splits in turn.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void JoinKernel(CacheAttentionParams p) {
  constexpr int kLanes = DIM / 4, kGroups = 256 / kLanes;
  const CacheView& c = p.cache;
  int tile = blockIdx.y;
  const int sequence = SequenceOfItem(c, p.group, p.tile_shift, 1, &tile);
  const Span span = SpanOf(c, sequence);
  const int rows = span.count * p.group;
  const int in_tile = blockIdx.z;
  const int row = (tile << p.tile_shift) + in_tile;
  if (tile < 0 || row >= rows)
    return;
  const int head = blockIdx.x;
  const int tid = threadIdx.x, group = tid / kLanes, part = tid % kLanes;
  const std::size_t first =
      (((static_cast<std::size_t>(blockIdx.y) * c.kv_heads + head) * p.splits) << p.tile_shift) +
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
    weights[tid] = weight;
  const float part_total = WaveSum(l * weight);
  if ((tid & 63) == 0)
    totals[tid >> 6] = part_total;
  __syncthreads();
  const float total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
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
        sum += o[a] * weights[s0 + a * kGroups];
  }
  sums[group][part] = sum;
  __syncthreads();
  if (group != 0)
    return;
#pragma unroll
  for (int g = 1; g < kGroups; ++g)
    sum += sums[g][part];
  const float scale = total == 0.0F ? 0.0F : 1.0F / total;
  const int query = row / p.group, of_group = row % p.group;
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
  int tile = blockIdx.y;
  const int sequence = SequenceOfItem(c, p.group, p.tile_shift, 1, &tile);
  const Span span = SpanOf(c, sequence);
  const int rows = span.count * p.group;
  const int tid = threadIdx.x, part = tid % kLanes;
  const int in_tile = blockIdx.z * kGroups + tid / kLanes;
  const int row = (tile << p.tile_shift) + in_tile;
  if (tile < 0 || row >= rows)
    return;
  const int head = blockIdx.x;
  const std::size_t first =
      (((static_cast<std::size_t>(blockIdx.y) * c.kv_heads + head) * p.splits) << p.tile_shift) +
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
  floatx4 sum = {};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float w = __builtin_amdgcn_exp2f(m[s] - from);
    total += l[s] * w;
    if (s < p.splits)
      sum += o[s] * w;
  }
  const float scale = total == 0.0F ? 0.0F : 1.0F / total;
  const int query = row / p.group, of_group = row % p.group;
  T rounded[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    rounded[r] = static_cast<T>(sum[r] * scale);
  __builtin_memcpy(static_cast<T*>(p.out) +
                       static_cast<std::int64_t>(span.first + query) * p.out_stride +
                       static_cast<std::int64_t>(head * p.group + of_group) * DIM + 4 * part,
                   rounded, sizeof(rounded));
}

template <typename T, int DIM>
void Launch(const CacheAttentionParams& p, hipStream_t stream) {
  const int items = ItemBound(p.cache, p.group, p.tile_shift, 1);
  const dim3 grid(p.cache.kv_heads, items, p.splits), block(kFewWaves * kWave);
  const bool last = p.splits == 1;
  if (p.tile_shift == 4)
    Dispatch(FewRowsKernel<T, DIM, 1>, grid, block, 0, stream, true, last, p);
  else if (p.tile_shift == 5)
    Dispatch(FewRowsKernel<T, DIM, 2>, grid, block, 0, stream, true, last, p);
  else if (p.cache.block_shift == 4)
    Dispatch(ManyRowsKernel<T, DIM, 4>, grid, block, 0, stream, true, last, p);
  else if (p.cache.block_shift == 5)
    Dispatch(ManyRowsKernel<T, DIM, 5>, grid, block, 0, stream, true, last, p);
  else
    Dispatch(ManyRowsKernel<T, DIM, 6>, grid, block, 0, stream, true, last, p);
  if (last)
    return;
  constexpr int kJoined = 256 / (DIM / 4);  // rows of a work-group with few splits
  if (p.splits <= kFewSplits)
    Dispatch(JoinFewKernel<T, DIM>,
             dim3(p.cache.kv_heads, items, ((1 << p.tile_shift) + kJoined - 1) / kJoined),
             dim3(256), 0, stream, false, true, p);
  else
    Dispatch(JoinKernel<T, DIM>, dim3(p.cache.kv_heads, items, 1 << p.tile_shift), dim3(256), 0,
             stream, false, true, p);
}

}  // namespace

CacheAttentionPlan PlanCacheAttention(const CacheView& c, int group) {
  CacheAttentionPlan plan;
  if (c.rows == 0)
    return plan;
  // Rows of a sequence on average: 16 columns of the matrix operand where they
  // suffice, else 32, which halve what is read of the codes again.
  const std::int64_t all = static_cast<std::int64_t>(c.rows) * group;
  plan.tile_shift = all <= 16ll * c.count ? 4 : all <= 48ll * c.count ? 5 : 7;
  const int items = ItemBound(c, group, plan.tile_shift, 1);
  const std::int64_t groups = static_cast<std::int64_t>(items) * c.kv_heads;
  const std::int64_t capacity = static_cast<std::int64_t>(c.table_width) << c.block_shift;
  const std::int64_t aim = plan.tile_shift == 7                   ? kManyGroups
                           : plan.tile_shift == 4 && c.count > 1 ? kRaggedSplitGroups
                                                                 : kSplitGroups;
  const std::int64_t least = plan.tile_shift == 7 ? 2 * kLeastChunk : kLeastChunk;
  const std::int64_t wanted =
      plan.tile_shift == 7 ? aim / groups : (aim + groups - 1) / groups;
  plan.splits = static_cast<int>(std::max<std::int64_t>(
      1, std::min({wanted, capacity / least, std::int64_t{kMostSplits}})));
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
