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
#include <type_traits>

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
  static __device__ __forceinline__ floatx4 Mfma16(x8 a, x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
  static __device__ __forceinline__ floatx4 Mfma16(x8 a, x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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

constexpr int kFewWaves = 4;
constexpr int kFewRows = 16;

// A work-group takes 16 rows of one sequence and kv head; its waves take the
// steps of 32 keys in turn, each with a softmax of its own that runs along
// (maximum m, sum l, output o), and the four are joined in LDS at the end.
template <typename T, int DIM>
__global__ __launch_bounds__(kFewWaves* kWave) void FewRowsKernel(CacheAttentionParams p) {
  typedef typename Types<T>::x8 x8;
  constexpr int kSteps = DIM / 64;   // 16-byte loads of a key's codes in a lane
  constexpr int kTiles = DIM / 16;
  const CacheView& c = p.cache;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column = lane & 15, quad = lane >> 4;
  const int head = blockIdx.y;

  int tile = blockIdx.x;
  const int sequence = SequenceOfItem(c, p.group, 4, 1, &tile);
  const Span span = SpanOf(c, sequence);
  const int rows = span.count * p.group;
  if (tile * kFewRows >= rows)
    return;
  const int row = tile * kFewRows + column;
  const int query = min(row, rows - 1) / p.group;
  const int of_group = min(row, rows - 1) - query * p.group;
  const int capacity = c.table_width << c.block_shift;
  const int length = min(span.length, capacity);
  // Keys that this row sees, and that any row of the tile sees.
  const int seen =
      row >= rows ? 0 : p.causal ? min(span.start + query + 1, length) : length;
  const int last = min(tile * kFewRows + kFewRows, rows) - 1;
  const int end = p.causal ? min(span.start + last / p.group + 1, length) : length;

  x8 q[kSteps][2];
  {
    const T* from = static_cast<const T*>(p.q) +
                    static_cast<std::int64_t>(span.first + query) * p.q_stride +
                    static_cast<std::int64_t>(head * p.group + of_group) * DIM + 16 * quad;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      __builtin_memcpy(&q[i][0], from + 64 * i, sizeof(x8));
      __builtin_memcpy(&q[i][1], from + 64 * i + 8, sizeof(x8));
    }
  }

  float m = -__builtin_inff(), l = 0.0F;
  floatx4 o[kTiles] = {};
  for (int base = wave * 32; base < end; base += kFewWaves * 32) {
    float s[2][4];
    u32x4 v[2][kSteps];
    float level[2];
    float peak = -__builtin_inff();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = base + 16 * g;
      const int page = PageOf(c, sequence, key >> c.block_shift);
      const int at = max(page, 0);
      const std::size_t skip = static_cast<std::size_t>(key & ((1 << c.block_shift) - 1)) * DIM;
      const u32x4* kc = reinterpret_cast<const u32x4*>(HalfOf(c, at, head, 0) + skip);
      const u32x4* vc = reinterpret_cast<const u32x4*>(HalfOf(c, at, head, 1) + skip);
      const float k_scale = c.scales[ScaleIndex(c, at, head, 0)];
      const float v_scale = c.scales[ScaleIndex(c, at, head, 1)];
      floatx4 acc = {};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const u32x4 w = kc[i * 64 + lane];
        v[g][i] = vc[i * 64 + lane];
        acc = Types<T>::Mfma16(Operand<T>(w[0], w[1], 1.0F), q[i][0], acc);
        acc = Types<T>::Mfma16(Operand<T>(w[2], w[3], 1.0F), q[i][1], acc);
      }
      // A NaN scale, of keys or values, makes the block's scores NaN.
      const float factor = p.scale_log2 * k_scale + 0.0F * v_scale;
      level[g] = v_scale == v_scale ? v_scale : 0.0F;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool visible = page >= 0 && key + 4 * quad + r < seen;
        s[g][r] = visible ? acc[r] * factor : -__builtin_inff();
        peak = fmaxf(peak, s[g][r]);
      }
    }
    peak = fmaxf(peak, __shfl_xor(peak, 16));
    peak = fmaxf(peak, __shfl_xor(peak, 32));
    const float top = fmaxf(m, peak);
    const float from = top == -__builtin_inff() ? 0.0F : top;
    const float shrink = __builtin_amdgcn_exp2f(m - from);
    m = top;
    l *= shrink;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      o[t] *= shrink;
    x8 w;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const T rounded = static_cast<T>(__builtin_amdgcn_exp2f(s[g][r] - from));
        w[4 * g + r] = rounded;
        l += static_cast<float>(rounded);
      }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      // The values' scales differ by block: each group's product apart.
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        x8 half = {};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          half[4 * g + r] = w[4 * g + r];
        const floatx4 zero = {};
        const floatx4 d = Types<T>::Mfma16(
            Operand<T>(v[0][t / 4][t % 4], v[1][t / 4][t % 4], 1.0F), half, zero);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[t][r] = __builtin_fmaf(d[r], level[g], o[t][r]);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  __shared__ float shared_m[kFewWaves][kFewRows], shared_l[kFewWaves][kFewRows];
  __shared__ floatx4 shared_o[kFewWaves][kTiles][64];
  if (quad == 0) {
    shared_m[wave][column] = m;
    shared_l[wave][column] = l;
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
    shared_o[wave][t][lane] = o[t];
  __syncthreads();
  float top = -__builtin_inff(), total = 0.0F;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w)
    top = fmaxf(top, shared_m[w][column]);
  const float from = top == -__builtin_inff() ? 0.0F : top;
  float weight[kFewWaves];
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) {
    weight[w] = __builtin_amdgcn_exp2f(shared_m[w][column] - from);
    total += shared_l[w][column] * weight[w];
  }
  // Nothing seen: zero.
  const float scale = total == 0.0F ? 0.0F : 1.0F / total;
  if (row >= rows)
    return;
  T* to = static_cast<T*>(p.out) + static_cast<std::int64_t>(span.first + query) * p.out_stride +
          static_cast<std::int64_t>(head * p.group + of_group) * DIM + 4 * quad;
  for (int t = wave; t < kTiles; t += kFewWaves) {
    floatx4 sum = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
      sum += shared_o[w][t][lane] * weight[w];
    T rounded[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      rounded[r] = static_cast<T>(sum[r] * scale);
    __builtin_memcpy(to + 16 * t, rounded, sizeof(rounded));
  }
}

template <typename T, int DIM>
void Launch(const CacheAttentionParams& p, hipStream_t stream) {
  const dim3 grid(ItemBound(p.cache, p.group, 4, 1), p.cache.kv_heads);
  Dispatch(FewRowsKernel<T, DIM>, grid, dim3(kFewWaves * kWave), 0, stream, true, true, p);
}

}  // namespace

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
