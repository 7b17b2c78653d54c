// The product of 8-bit rows with 8-bit weights.
//
//   y[r][o] = (sum over k of x[r][k] w[o][k]) * x_scales[r] * w_scales[o]
//
// e4m3 codes, float32 sums. A lane's operand of v_mfma_f32_16x16x128_f8f6f4 is 32
// codes of one row, four lanes a row; which of a step's 128 codes a lane has does not
// matter as long as both operands agree, so rows of codes as they lie in memory are
// operands and nothing is packed.
#include "step.hpp"

namespace ovg {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef half_t half2v __attribute__((ext_vector_type(2)));

constexpr int kStep = 128;  // codes of K in a step
constexpr std::int64_t kTileStride = 1 << 23;  // 256 rows of it are 32-bit offsets

// D[4 (l / 16) + r][l % 16] in element r of lane l, rows of `a` by rows of `b`.
//
// The instruction adds its products in groups, each aligned to the group's largest:
// what is under 2^-13 of that is cut off, 1.5e-5 of a sum of random terms. 16-bit
// results round by 2^-9 or 2^-12 and take it; float32 results go through fp16, which
// holds every e4m3 code, and whose products are added as float32 (6e-8), at half the
// rate and with the conversions.
template <bool HALF>
struct Operand {
  intx8 codes;
  __device__ __forceinline__ void Set(intx4 lo, intx4 hi) {
    codes = intx8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};
template <>
struct Operand<true> {
  half8 part[4];
  __device__ __forceinline__ void Set(intx4 lo, intx4 hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int word = i < 2 ? lo[2 * i + j] : hi[2 * (i - 2) + j];
        const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0F, false);
        const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0F, true);
        part[i][4 * j] = a[0];
        part[i][4 * j + 1] = a[1];
        part[i][4 * j + 2] = b[0];
        part[i][4 * j + 3] = b[1];
      }
  }
};
__device__ __forceinline__ floatx4 Multiply(const Operand<false>& a, const Operand<false>& b,
                                            floatx4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.codes, b.codes, c, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx4 Multiply(const Operand<true>& a, const Operand<true>& b,
                                            floatx4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.part[i], b.part[i], c, 0, 0, 0);
  return c;
}

// The lane's 32 codes of a row from k on, zeros behind the row's end (a multiple of 16).
template <bool HALF>
__device__ __forceinline__ void LoadOperand(const unsigned char* row, int k, int in,
                                            Operand<HALF>* to) {
  intx4 part[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    part[h] = intx4{0, 0, 0, 0};
    if (k + 16 * h < in)
      part[h] = *reinterpret_cast<const intx4*>(row + k + 16 * h);
  }
  to->Set(part[0], part[1]);
}

// ---------------------------------------------------------------- few rows
// 16 MB rows by 16 columns; the waves take every fourth step of K and join in LDS.
constexpr int kWaves = 4;

template <typename T, int MB>
__global__ __launch_bounds__(kWaves* kWave) void SkinnyKernel(Linear8Params p) {
  constexpr bool kHalf = std::is_same_v<T, float>;
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
  for (int k = wave * kStep; k < p.in; k += kWaves * kStep) {
    Operand<kHalf> b, a;
    LoadOperand(w, k + part, p.in, &b);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      LoadOperand(x[m], k + part, p.in, &a);
      acc[m] = Multiply(a, b, acc[m]);
    }
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

// ---------------------------------------------------------------- tiles
// BM rows by BN columns of a work-group, WM by WN waves, a ring of STAGES steps of both
// operands in LDS, filled by loads that go there directly. A row's 128 codes lie in LDS
// in 16-byte chunks, chunk c of row r at c ^ Swizzle(r), so that the 16 rows that a
// wave's operand reads at one c are in 16 different groups of banks.
//
// The weights are the left operand, so that a lane holds neighbouring columns of one
// row: their rows are dealt to the wave's FN operands such that a lane's 4 FN columns
// are next to each other.
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
struct Tile {
  static constexpr bool kHalf = std::is_same_v<T, float>;
  static constexpr int kWaveCount = WM * WN;
  static constexpr int kThreads = kWaveCount * kWave;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int kStageBytes = (BM + BN) * kStep;
  static constexpr int kXLoads = BM / 8 / kWaveCount, kWLoads = BN / 8 / kWaveCount;
  static constexpr int kLoads = kXLoads + kWLoads;
  static_assert(BM % (8 * kWaveCount) == 0 && BN % (8 * kWaveCount) == 0, "whole loads a wave");
  static __device__ __forceinline__ int SwizzleX(int r) { return (r >> 1) & 7; }
  static __device__ __forceinline__ int SwizzleW(int r) {
    return ((r >> 1) & 1) | ((r / (4 * FN)) & 3) << 1;
  }
};

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM* WN* kWave) void TileKernel(Linear8Params p, int row_tiles,
                                                            int col_tiles) {
  using S = Tile<T, BM, BN, WM, WN, STAGES>;
  constexpr int FM = S::FM, FN = S::FN;
  __shared__ __align__(16) unsigned char lds[STAGES * S::kStageBytes];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;

  // Work-groups go to the XCDs in turn: each XCD takes a run of tiles, ordered down
  // columns of eight row tiles.
  const int tiles = row_tiles * col_tiles;
  int tile = blockIdx.x;
  {
    const int each = tiles / kXcds, rest = tiles % kXcds;
    const int xcd = tile % kXcds, at = tile / kXcds;
    tile = xcd * each + min(xcd, rest) + at;
  }
  const int band = tile / (8 * col_tiles);
  const int high = min(8, row_tiles - 8 * band);
  const int in_band = tile - band * 8 * col_tiles;
  const int row0 = (band * 8 + in_band % high) * BM;
  const int col0 = in_band / high * BN;

  // This lane's chunk of the eight rows that one load brings.
  const int sub = lane / 8, chunk = lane % 8;
  std::uint32_t x_at[S::kXLoads], w_at[S::kWLoads];
#pragma unroll
  for (int i = 0; i < S::kXLoads; ++i) {
    const int r = (wave * S::kXLoads + i) * 8 + sub;
    x_at[i] = static_cast<std::uint32_t>(min(r, p.rows - 1 - row0)) *
                  static_cast<std::uint32_t>(p.x_stride) +
              (chunk ^ S::SwizzleX(r)) * 16;
  }
#pragma unroll
  for (int i = 0; i < S::kWLoads; ++i) {
    const int r = (wave * S::kWLoads + i) * 8 + sub;
    w_at[i] = static_cast<std::uint32_t>(min(r, p.out - 1 - col0)) *
                  static_cast<std::uint32_t>(p.in) +
              (chunk ^ S::SwizzleW(r)) * 16;
  }
  const unsigned char* const x = p.x + row0 * p.x_stride;
  const unsigned char* const w = p.w + static_cast<std::size_t>(col0) * p.in;
  const std::uint32_t lds0 = LdsAddress(lds);
  const auto fetch = [&](int step, int stage) {
    const std::uint32_t to = lds0 + stage * S::kStageBytes;
#pragma unroll
    for (int i = 0; i < S::kXLoads; ++i)
      DmaToLds(x + step * kStep, x_at[i], to + (wave * S::kXLoads + i) * 1024);
#pragma unroll
    for (int i = 0; i < S::kWLoads; ++i)
      DmaToLds(w + step * kStep, w_at[i],
               to + BM * kStep + (wave * S::kWLoads + i) * 1024);
  };

  // Operand m of x: rows 16 m + lane % 16 of the wave's; operand n of w: rows dealt.
  const int part = lane / 16, i16 = lane % 16;
  int x_read[2], w_read[2];
  {
    const int r = wm * FM * 16 + i16;
    const int c = wn * FN * 16 + (i16 / 4) * 4 * FN + i16 % 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x_read[h] = r * kStep + ((2 * part + h) ^ S::SwizzleX(r)) * 16;
      w_read[h] = BM * kStep + c * kStep + ((2 * part + h) ^ S::SwizzleW(c)) * 16;
    }
  }
  floatx4 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n)
      acc[m][n] = floatx4{0, 0, 0, 0};

  const int steps = p.in / kStep;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps)
      fetch(s, s);
  int stage = 0;
  for (int step = 0; step < steps; ++step) {
    if (step + STAGES - 1 <= steps)
      WaitLoads<S::kLoads*(STAGES - 2)>();
    else
      WaitLoads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (step + STAGES - 1 < steps)
      fetch(step + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
    const unsigned char* const from = lds + stage * S::kStageBytes;
    Operand<S::kHalf> b[FN];
#pragma unroll
    for (int n = 0; n < FN; ++n)
      b[n].Set(*reinterpret_cast<const intx4*>(from + w_read[0] + n * 4 * kStep),
               *reinterpret_cast<const intx4*>(from + w_read[1] + n * 4 * kStep));
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      Operand<S::kHalf> a;
      a.Set(*reinterpret_cast<const intx4*>(from + x_read[0] + m * 16 * kStep),
            *reinterpret_cast<const intx4*>(from + x_read[1] + m * 16 * kStep));
#pragma unroll
      for (int n = 0; n < FN; ++n)
        acc[m][n] = Multiply(b[n], a, acc[m][n]);
    }
    asm volatile("" ::: "memory");
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }

  const int first_row = row0 + wm * FM * 16 + i16;
  const int first_col = col0 + wn * FN * 16 + part * 4 * FN;
  if (p.in % kStep != 0) {  // the last, partial step comes straight from memory
    Operand<S::kHalf> a, b[FN];
    const int k = steps * kStep + part * 32;
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      const int c = min(col0 + wn * FN * 16 + (i16 / 4) * 4 * FN + n * 4 + i16 % 4, p.out - 1);
      LoadOperand(p.w + static_cast<std::size_t>(c) * p.in, k, p.in, &b[n]);
    }
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      LoadOperand(p.x + min(first_row + 16 * m, p.rows - 1) * p.x_stride, k, p.in, &a);
#pragma unroll
      for (int n = 0; n < FN; ++n)
        acc[m][n] = Multiply(b[n], a, acc[m][n]);
    }
  }

  constexpr int kCols = 4 * FN;  // of a lane
  constexpr int kVec = 16 / sizeof(T);
  const bool whole = first_col + kCols <= p.out;
  float ws[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    ws[c] = p.w_scales[min(first_col + c, p.out - 1)];
  T* const y = static_cast<T*>(p.y);
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const int row = first_row + 16 * m;
    if (row >= p.rows)
      break;
    const float xs = p.x_scales[row];
    T* const to = y + row * p.y_stride + first_col;
    T v[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      v[c] = static_cast<T>(acc[m][c / 4][c % 4] * xs * ws[c]);
    if (whole) {
#pragma unroll
      for (int c = 0; c < kCols; c += kVec)
        __builtin_memcpy(to + c, v + c, 16);
    } else {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (first_col + c < p.out)
          to[c] = v[c];
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
  const auto tiled = [&](auto bm, auto bn, auto wm, auto wn, auto stages) {
    const int row_tiles = (p.rows + bm() - 1) / bm(), col_tiles = (p.out + bn() - 1) / bn();
    Require(static_cast<std::int64_t>(row_tiles) * col_tiles < (1 << 23),
            "linear: too many tiles");
    Dispatch(TileKernel<T, bm(), bn(), wm(), wn(), stages()>, dim3(row_tiles * col_tiles),
             dim3(wm() * wn() * kWave), 0, s, true, true, p, row_tiles, col_tiles);
  };
  using std::integral_constant;
  const auto groups = [&](int bm, int bn) {
    return static_cast<std::int64_t>((p.rows + bm - 1) / bm) * ((p.out + bn - 1) / bn);
  };
  if (p.rows <= 16)
    skinny(integral_constant<int, 1>());
  else if (p.rows <= 64 || p.x_stride > kTileStride)
    skinny(integral_constant<int, 4>());
  else if (groups(256, 256) >= 2 * kCus)
    tiled(integral_constant<int, 256>(), integral_constant<int, 256>(),
          integral_constant<int, 2>(), integral_constant<int, 4>(), integral_constant<int, 2>());
  else if (groups(128, 128) >= kCus)
    tiled(integral_constant<int, 128>(), integral_constant<int, 128>(),
          integral_constant<int, 2>(), integral_constant<int, 2>(), integral_constant<int, 2>());
  else
    tiled(integral_constant<int, 64>(), integral_constant<int, 64>(),
          integral_constant<int, 2>(), integral_constant<int, 2>(), integral_constant<int, 4>());
}

}  // namespace

void LaunchLinear8(const Linear8Params& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.rows <= kMostRows && p.in >= 16 && p.in % 16 == 0 && p.out >= 1,
          "linear: shape outside the kernel's range");
  WithType(type, [&](auto t) { Launch<decltype(t)>(p, stream); });
  Check(hipGetLastError(), "linear launch");
}

}  // namespace ovg
