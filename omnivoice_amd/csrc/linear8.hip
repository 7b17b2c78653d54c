// The product of 8-bit rows with 8-bit weights.
//
//   y[r][o] = (sum over k of x[r][k] w[o][k]) * x_scales[r] * w_scales[o]
//
// e4m3 codes, float32 sums. A lane's operand of v_mfma_f32_16x16x128_f8f6f4 is 32
// codes in a row of K, at 32 (lane / 16) of row lane % 16, so that rows of codes as
// they lie in memory are operands: four lanes read 128 bytes of a row.
#include "step.hpp"

namespace ovg {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));

// D[4 (l / 16) + r][l % 16] of A (rows) and B (columns) in element r of lane l.
__device__ __forceinline__ floatx4 Mfma8(intx8 a, intx8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7F7F7F7F, 0,
                                                          0x7F7F7F7F);
}

// 32 codes at k of a row, zeros behind its end (a multiple of 16).
__device__ __forceinline__ intx8 LoadCodes(const unsigned char* row, int k, int in) {
  intx8 v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (k + 16 * h < in) {
      const intx4 part = *reinterpret_cast<const intx4*>(row + k + 16 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[4 * h + i] = part[i];
    }
  }
  return v;
}

constexpr int kWaves = 4;

// 16 MB rows by 16 columns; the four waves take every fourth step of K and join in LDS.
template <typename T, int MB>
__global__ __launch_bounds__(kWaves* kWave) void SkinnyKernel(Linear8Params p) {
  __shared__ floatx4 parts[kWaves][MB][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int row0 = blockIdx.y * 16 * MB, col0 = blockIdx.x * 16;
  const int part = (lane / 16) * 32;
  const unsigned char* const w =
      p.w + static_cast<std::size_t>(min(col0 + lane % 16, p.out - 1)) * p.in;
  const unsigned char* x[MB];
  floatx4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    x[m] = p.x + min(row0 + 16 * m + lane % 16, p.rows - 1) * p.x_stride;
    acc[m] = floatx4{0, 0, 0, 0};
  }
  for (int k = wave * 128; k < p.in; k += kWaves * 128) {
    const intx8 b = LoadCodes(w, k + part, p.in);
#pragma unroll
    for (int m = 0; m < MB; ++m)
      acc[m] = Mfma8(LoadCodes(x[m], k + part, p.in), b, acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
    parts[wave][m][lane] = acc[m];
  __syncthreads();
  const int col = col0 + lane % 16;
  for (int m = wave; m < MB; m += kWaves) {
    floatx4 sum = parts[0][m][lane];
#pragma unroll
    for (int i = 1; i < kWaves; ++i)
      sum += parts[i][m][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = row0 + 16 * m + 4 * (lane / 16) + r;
      if (row < p.rows && col < p.out)
        static_cast<T*>(p.y)[row * p.y_stride + col] =
            static_cast<T>(sum[r] * p.x_scales[row] * p.w_scales[col]);
    }
  }
}

template <typename T>
void Launch(const Linear8Params& p, hipStream_t s) {
  const auto skinny = [&](auto mb) {
    constexpr int kRows = 16 * mb();
    Dispatch(SkinnyKernel<T, mb()>, dim3((p.out + 15) / 16, (p.rows + kRows - 1) / kRows),
             dim3(kWaves * kWave), 0, s, true, true, p);
  };
  if (p.rows <= 16)
    skinny(std::integral_constant<int, 1>());
  else
    skinny(std::integral_constant<int, 4>());
}

}  // namespace

void LaunchLinear8(const Linear8Params& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.rows <= kMostRows && p.in >= 16 && p.in % 16 == 0 && p.out >= 1,
          "linear: shape outside the kernel's range");
  WithType(type, [&](auto t) { Launch<decltype(t)>(p, stream); });
  Check(hipGetLastError(), "linear launch");
}

}  // namespace ovg
