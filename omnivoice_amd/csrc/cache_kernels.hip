// Writing tokens into the 8-bit key/value cache and reading them back.
//
// A block of 16, 32 or 64 tokens of one kv head holds its keys and its values
// as e4m3 codes with one power-of-two scale each: x ~ code * 2^e. With a
// power of two the block's scale can grow when louder tokens join it and the
// codes that stay move by a whole number of exponent steps: nothing is
// rounded again, but what falls under e4m3's smallest normal value.
//
// Order of the codes, in groups of 16 tokens: that of the attention's matrix
// operands, so that a lane's 16 bytes are one load and a wave's are 1 KB in a
// row (cache_attention.hip):
//   keys   [dim / 16][token][dim % 16]
//   values [dim / 64][token / 4][dim % 16][dim / 16 % 4][token % 4]
//
// Both kernels give one work-group of 256 threads one half (keys or values)
// of one head of one block: the unit that shares a scale. A thread takes 16
// dims of one token, so rows come and go as whole 32-byte (16-bit types) or
// 64-byte (float32) runs, eight threads a row; the values change between that
// order and the pool's in LDS.
//
// Bound: memory. 16 prompts of up to 2048 tokens (8 heads of 128, fp16, 163 MB both
// ways) are written in 35.5 to 36 us, 4.6 TB/s (29 when the same prompts are written again and
// come out of the Infinity Cache), 32 sequences of up to 4096 (612 MB) read in 133 us,
// 4.6 TB/s, where a copy of 1 GiB reaches 5.05. One token each of 64 sequences is the
// chain of the sequence, the table, the old scale and the old codes, 6 us.
#include "cache.hpp"

namespace ovg {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct Vec16 {  // 16 elements of T
  typedef T type __attribute__((ext_vector_type(16)));
};

__device__ __forceinline__ float ToFloat(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float ToFloat(__bf16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float ToFloat(float x) { return x; }

// The smallest power of two, 2^-100 or more, that takes amax (finite, given
// by its bits) into +-448, e4m3's range: 448 = 1.75 * 2^8.
__device__ __forceinline__ float ScaleFor(unsigned amax) {
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u);
  return __uint_as_float(static_cast<unsigned>(max(e, -100) + 127) << 23);
}
// 1 / scale of such a power of two.
__device__ __forceinline__ float Inverse(float scale) {
  return __uint_as_float((254u << 23) - __float_as_uint(scale));
}

__device__ __forceinline__ unsigned Encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
__device__ __forceinline__ float Decode(unsigned code) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code), 0);
}
// Four codes at another scale.
__device__ __forceinline__ unsigned Rescale4(unsigned w, float factor) {
  return Encode4(Decode(w) * factor, Decode(w >> 8) * factor, Decode(w >> 16) * factor,
                 Decode(w >> 24) * factor);
}

// Byte of (token, dim) in the values of a block.
__device__ __forceinline__ int ValueByte(int token, int dim, int width) {
  return (token >> 4) * 16 * width + (dim >> 6) * 1024 + ((token >> 2) & 3) * 256 +
         (dim & 15) * 16 + ((dim >> 4) & 3) * 4 + (token & 3);
}

// The block of the pool that work-group `item` handles, or false.
struct Touched {
  Span span;
  int end;          // position behind the rows' last
  int block, page;  // block of the sequence, of the pool
};
__device__ __forceinline__ bool Find(const CacheView& c, int item, Touched* t) {
  const Found f = FindItem(c, 1, c.block_shift, 2, item);
  t->span = f.span;
  if (f.span.count == 0 || f.item < 0)
    return false;
  t->end = f.span.start + f.span.count;
  t->block = (f.span.start >> c.block_shift) + f.item;
  if (t->block > (t->end - 1) >> c.block_shift)
    return false;
  t->page = PageOf(c, f.sequence, t->block);
  return true;
}

template <typename T, int DIM, int SHIFT>
__global__ __launch_bounds__(kThreads) void CacheWriteKernel(CacheWriteParams p) {
  constexpr int kBlock = 1 << SHIFT;
  constexpr int kChunks = kBlock * DIM / 16;              // 16-byte chunks
  constexpr int kPer = (kChunks + kThreads - 1) / kThreads;  // a thread's
  constexpr int kRow = DIM / 16;                          // chunks of a token
  typedef typename Vec16<T>::type vec;
  __shared__ unsigned wave_max[kThreads / kWave];
  __shared__ uint4 staged[kChunks];
  const CacheView& c = p.cache;
  Touched t;
  if (!Find(c, blockIdx.x, &t) || t.page < 0)
    return;
  const int head = blockIdx.y, half = blockIdx.z, tid = threadIdx.x;
  const int first = t.block << SHIFT;
  const int kept = max(t.span.start - first, 0);                // tokens that stay
  const int live = min(t.end - first, kBlock);                  // and the block's last
  unsigned char* const codes = HalfOf(c, t.page, head, half);
  const std::size_t scale_at = ScaleIndex(c, t.page, head, half);
  const T* const x = static_cast<const T*>(p.x[half]) + static_cast<std::int64_t>(head) * DIM;

  float value[kPer][16];
  unsigned amax = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int chunk = tid + k * kThreads;
    const int token = chunk / kRow;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      value[k][e] = 0.0F;
    if (chunk < kChunks && token >= kept && token < live) {
      const std::int64_t row = t.span.first + (first + token - t.span.start);
      const T* from = x + row * p.stride[half] + (chunk % kRow) * 16;
      vec v;
      __builtin_memcpy(&v, from, sizeof(v));
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        value[k][e] = ToFloat(v[e]);
        // The order of magnitudes' bits is the magnitudes' own, infinities
        // and NaN behind every number.
        amax = max(amax, __float_as_uint(value[k][e]) & 0x7FFFFFFFu);
      }
    }
  }
  for (int offset = kWave / 2; offset > 0; offset /= 2)
    amax = max(amax, static_cast<unsigned>(__shfl_xor(static_cast<int>(amax), offset)));
  if ((tid & (kWave - 1)) == 0)
    wave_max[tid / kWave] = amax;
  const float old = kept > 0 ? c.scales[scale_at] : 0.0F;
  __syncthreads();
  amax = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  const bool lost = amax >= 0x7F800000u || old != old;
  const float scale = fmaxf(ScaleFor(amax), old);
  // A block that holds an infinity or a NaN is NaN as a whole: its scale says
  // so and its codes stay numbers, which no masked product can spread.
  const float inverse = lost ? 0.0F : Inverse(scale);
  const float factor = old * inverse;
  if (tid == 0)
    c.scales[scale_at] = lost ? __builtin_nanf("") : scale;

#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int chunk = tid + k * kThreads;
    const int token = chunk / kRow, part = chunk % kRow;
    if (chunk >= kChunks)
      break;
    unsigned w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = lost ? 0u
                  : Encode4(value[k][4 * e] * inverse, value[k][4 * e + 1] * inverse,
                            value[k][4 * e + 2] * inverse, value[k][4 * e + 3] * inverse);
    if (half == 0) {
      uint4* to = reinterpret_cast<uint4*>(codes + (token >> 4) * 16 * DIM + part * 256 +
                                           (token & 15) * 16);
      if (token < kept) {
        const uint4 held = *to;
        const unsigned h[4] = {held.x, held.y, held.z, held.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = factor == 1.0F || lost ? h[e] : Rescale4(h[e], factor);
      }
      *to = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      unsigned char* to = reinterpret_cast<unsigned char*>(staged);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        to[ValueByte(token, part * 16 + e, DIM)] =
            static_cast<unsigned char>(w[e >> 2] >> (8 * (e & 3)));
    }
  }
  if (half == 0)
    return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int chunk = tid + k * kThreads;
    if (chunk >= kChunks)
      break;
    // This chunk's four tokens, for each of four dims.
    const int token = chunk / kRow / 16 * 16 + (chunk >> 4 & 3) * 4;
    uint4 v = staged[chunk];
    uint4* to = reinterpret_cast<uint4*>(codes) + chunk;
    if (token < kept) {
      const uint4 held = *to;
      const unsigned h[4] = {held.x, held.y, held.z, held.w};
      unsigned w[4] = {v.x, v.y, v.z, v.w};
      const int stay = min(kept - token, 4);
      const unsigned mask = stay == 4 ? ~0u : (1u << (8 * stay)) - 1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned r = factor == 1.0F || lost ? h[e] : Rescale4(h[e], factor);
        w[e] = (r & mask) | (w[e] & ~mask);
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *to = v;
  }
}

template <typename T, int DIM, int SHIFT>
__global__ __launch_bounds__(kThreads) void CacheReadKernel(CacheReadParams p) {
  constexpr int kBlock = 1 << SHIFT;
  constexpr int kChunks = kBlock * DIM / 16;
  constexpr int kPer = (kChunks + kThreads - 1) / kThreads;
  constexpr int kRow = DIM / 16;
  typedef typename Vec16<T>::type vec;
  __shared__ uint4 staged[kChunks];
  const CacheView& c = p.cache;
  Touched t;
  if (!Find(c, blockIdx.x, &t))
    return;
  const int head = blockIdx.y, half = blockIdx.z, tid = threadIdx.x;
  const int first = t.block << SHIFT;
  const uint4* const codes =
      t.page < 0 ? nullptr
                 : reinterpret_cast<const uint4*>(HalfOf(c, t.page, head, half));
  const float scale = t.page < 0 ? 0.0F : c.scales[ScaleIndex(c, t.page, head, half)];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int chunk = tid + k * kThreads;
    if (chunk < kChunks)
      staged[chunk] = codes == nullptr ? make_uint4(0, 0, 0, 0) : codes[chunk];
  }
  __syncthreads();
  T* const x = static_cast<T*>(p.x[half]) + static_cast<std::int64_t>(head) * DIM;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int chunk = tid + k * kThreads;
    const int token = chunk / kRow, part = chunk % kRow;
    const int at = first + token - t.span.start;  // of the sequence's rows
    if (chunk >= kChunks || at < 0 || at >= t.span.count)
      continue;
    vec v;
    const unsigned char* bytes = reinterpret_cast<const unsigned char*>(staged);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int byte = half == 0 ? (token >> 4) * 16 * DIM + part * 256 + (token & 15) * 16 + e
                                 : ValueByte(token, part * 16 + e, DIM);
      v[e] = static_cast<T>(Decode(bytes[byte]) * scale);
    }
    __builtin_memcpy(x + static_cast<std::int64_t>(t.span.first + at) * p.stride[half] +
                         part * 16,
                     &v, sizeof(v));
  }
}

template <typename P, typename F>
void EachShape(const P& p, F&& launch) {
  if (p.cache.dim == 64) {
    if (p.cache.block_shift == 4) return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    if (p.cache.block_shift == 5) return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 5>());
    return launch(std::integral_constant<int, 64>(), std::integral_constant<int, 6>());
  }
  if (p.cache.block_shift == 4) return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 4>());
  if (p.cache.block_shift == 5) return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 5>());
  return launch(std::integral_constant<int, 128>(), std::integral_constant<int, 6>());
}

// The kernel of the type, width and block size; one work-group per item, head and half.
template <typename T>
void Write(const CacheWriteParams& p, dim3 grid, hipStream_t s) {
  EachShape(p, [&](auto dim, auto shift) {
    Dispatch(CacheWriteKernel<T, dim(), shift()>, grid, dim3(kThreads), 0, s, true, true, p);
  });
}
template <typename T>
void Read(const CacheReadParams& p, dim3 grid, hipStream_t s) {
  EachShape(p, [&](auto dim, auto shift) {
    Dispatch(CacheReadKernel<T, dim(), shift()>, grid, dim3(kThreads), 0, s, true, true, p);
  });
}

dim3 Grid(const CacheView& c) {
  return dim3(ItemBound(c, 1, c.block_shift, 2), c.kv_heads, 2);
}

}  // namespace

void LaunchCacheWrite(const CacheWriteParams& p, DType type, hipStream_t stream) {
  if (p.cache.rows == 0)
    return;
  const dim3 grid = Grid(p.cache);
  if (type == DType::kF16)
    Write<_Float16>(p, grid, stream);
  else if (type == DType::kBf16)
    Write<__bf16>(p, grid, stream);
  else
    Write<float>(p, grid, stream);
  Check(hipGetLastError(), "cache write launch");
}

void LaunchCacheRead(const CacheReadParams& p, DType type, hipStream_t stream) {
  if (p.cache.rows == 0)
    return;
  const dim3 grid = Grid(p.cache);
  if (type == DType::kF16)
    Read<_Float16>(p, grid, stream);
  else if (type == DType::kBf16)
    Read<__bf16>(p, grid, stream);
  else
    Read<float>(p, grid, stream);
  Check(hipGetLastError(), "cache read launch");
}

}  // namespace ovg
