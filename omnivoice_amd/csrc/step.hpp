// A token's step around the cache: parameters and launchers of norm_kernels.hip
// (rows normed with their residual, rows in 8 bits), linear8.hip (their product),
// rotary.hip (positions) and sample.hip (the draw of a token).
#ifndef OMNIVOICE_AMD_STEP_HPP_
#define OMNIVOICE_AMD_STEP_HPP_

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "cache.hpp"
#include "kernels.hpp"

namespace ovg {

// ---------------------------------------------------------------- rows
// y = weight * s * rsqrt(mean s^2 + eps) of s = x (+ second), or y = x
// (* silu(second)); rows `..._stride` elements apart.
struct RowParams {
  const void* x;
  const void* second;  // the residual, or the gate; or null
  void* total;         // where x + residual goes, in the residual's type
  const float* weight;
  void* out;
  float* scales;       // of e4m3 rows
  std::int64_t x_stride, second_stride, total_stride, out_stride;
  int rows, width;
  float eps;
};
constexpr int kMostRows = (1 << 22) - 1;  // a launch of 1024 lanes a row counts under 2^32
constexpr int kMostWidth = 1 << 16;
// second: the residual's type, kE4m3 for none.
void LaunchAddNorm(const RowParams& p, DType x, DType second, DType out, hipStream_t stream);
void LaunchQuantize(const RowParams& p, DType x, hipStream_t stream);

// ---------------------------------------------------------------- 8-bit product
struct Linear8Params {
  const unsigned char* x;  // [rows][in] e4m3, rows x_stride bytes apart
  const float* x_scales;   // [rows]
  const unsigned char* w;  // [out][in] e4m3
  const float* w_scales;   // [out]
  void* y;                 // [rows][out], rows y_stride elements apart
  std::int64_t x_stride, y_stride;
  int rows, in, out;
};
void LaunchLinear8(const Linear8Params& p, DType type, hipStream_t stream);

// ---------------------------------------------------------------- rotary positions
struct RotaryParams {
  const void* x[2];        // queries, keys: [rows][heads][dim]
  void* out[2];
  std::int64_t x_stride[2], out_stride[2];
  const float* norm[2];    // [dim], or null
  int heads[2];
  int rows, dim, rotary;
  const float* frequencies;  // [rotary / 2]
  const int* positions;      // [rows], or null: the sequences' own
  CacheView sequences;       // begins, lengths, count and rows of it
  float magnitude, eps;
};
constexpr int kMostRotaryDim = 512;
constexpr int kMostRotaryRows = (1 << 24) - 1;  // of 256 lanes
void LaunchRotary(const RotaryParams& p, bool interleaved, DType type, hipStream_t stream);

// ---------------------------------------------------------------- sampling
struct SampleParams {
  const void* logits;  // [rows][vocab], rows `stride` elements apart
  const void* uncond;  // the same, or null
  std::int64_t stride, uncond_stride;
  float guidance;
  int rows, vocab, mask_id;
  const float* random;  // [rows]
  int* tokens;          // [rows]
  // Of every row, or each row's own where the pointer is not null.
  float temperature, top_p, min_p;
  int top_k;
  const float* temperatures;
  const int* top_ks;
  const float* top_ps;
  const float* min_ps;
  unsigned* work;  // SampleWorkBytes
};
// -1 for more rows and tokens than a launch covers.
std::int64_t SampleWorkBytes(std::int64_t rows, std::int64_t vocab);
void LaunchSample(const SampleParams& p, DType type, hipStream_t stream);

// ---------------------------------------------------------------- device helpers
// N elements of T that may lie at any address.
template <typename T, int N>
struct Pack {
  T v[N];
};
template <int N, typename T>
__device__ __forceinline__ void LoadFloats(const T* from, float (&to)[N]) {
  Pack<T, N> v;
  __builtin_memcpy(&v, from, sizeof(v));
#pragma unroll
  for (int i = 0; i < N; ++i)
    to[i] = static_cast<float>(v.v[i]);
}
template <int N, typename T>
__device__ __forceinline__ void StoreFloats(T* to, const float (&from)[N]) {
  Pack<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i)
    v.v[i] = static_cast<T>(from[i]);
  __builtin_memcpy(to, &v, sizeof(v));
}

// Calls f with a value of the type that `type` names.
template <typename F>
void WithType(DType type, F&& f) {
  if (type == DType::kF16)
    f(_Float16{});
  else if (type == DType::kBf16)
    f(__bf16{});
  else
    f(float{});
}

}  // namespace ovg

#endif  // OMNIVOICE_AMD_STEP_HPP_
