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
// The 8-bit instruction adds the products of eight codes in a row at a time, aligned to the
// largest: bits below 2^-13 of that one's power of two are cut off, at most 7/8192 of the
// products' magnitudes and 1.5e-5 of a sum of random ones (the 8-bit one of 32 codes does the same).
// fp16 holds every e4m3 code, and its products are added as float32 (6e-8), at half the rate
// and with the conversions. Few rows and float32 results go through fp16, which costs few rows
// 1 to 5 % (16 x 1024 x 4096 in bf16 3.5 us both ways, 32 x 8192 x 8192 18.9 and 18.1 by the
// codes' own products); 16-bit results of tiles, which round by 2^-8 or 2^-11, take the codes'
// own (on one card 4096 x 4096 x 8192 in bf16 101 us, 187 through fp16; 64 x 4096 x 3000 10.8
// and 16.1).
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
// 16 MB rows by 16 NB columns; the waves take every fourth step of K and join in LDS, in a
// fixed order. Operands come straight from memory: a weight is used once, and 16 lines of
// 64 bytes in flight a wave, two steps of them, are what the latency asks for. Bound by
// reading the weights: 16 x 1024 x 4096 (4 MiB) 3.5 us, of which an empty launch is 2; 16 x
// 4096 x 8192 (32 MiB) 9.4 us, 3.6 TB/s; 32 x 8192 x 8192 18.9 us, 3.6 TB/s.
constexpr int kWaves = 4;

template <typename T, int MB, int NB>
__global__ __launch_bounds__(kWaves* kWave) void SkinnyKernel(Linear8Params p) {
  using Codes = Operand<true>;
  __shared__ floatx4 parts[kWaves][MB * NB][kWave];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row0 = blockIdx.y * 16 * MB, col0 = blockIdx.x * 16 * NB;
  const int part = lane / 16;
  const unsigned char *x[MB], *w[NB];
  floatx4 acc[MB][NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
    w[n] = p.w + static_cast<std::size_t>(min(col0 + 16 * n + lane % 16, p.out - 1)) * p.in;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    x[m] = p.x + min(row0 + 16 * m + lane % 16, p.rows - 1) * p.x_stride;
#pragma unroll
    for (int n = 0; n < NB; ++n)
      acc[m][n] = floatx4{0, 0, 0, 0};
  }
  // Whole steps without a question, two in flight, each load of 64 bytes in a row; the
  // last, partial one with it.
  const int whole = p.in / kStep * kStep;
  int k = wave * kStep;
  const auto load = [&](const unsigned char* row, Codes* to) {
    to->Set(*reinterpret_cast<const intx4*>(row + k + part * 16),
            *reinterpret_cast<const intx4*>(row + k + part * 16 + 64));
  };
#pragma unroll 2
  for (; k < whole; k += kWaves * kStep) {
    Codes a[MB], b[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
      load(w[n], &b[n]);
#pragma unroll
    for (int m = 0; m < MB; ++m)
      load(x[m], &a[m]);
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
        acc[m][n] = Multiply(a[m], b[n], acc[m][n]);
  }
  if (k < p.in) {
    Codes a, b[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
      LoadOperand(w[n], k + part * 32, p.in, &b[n]);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      LoadOperand(x[m], k + part * 32, p.in, &a);
#pragma unroll
      for (int n = 0; n < NB; ++n)
        acc[m][n] = Multiply(a, b[n], acc[m][n]);
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
      parts[wave][m * NB + n][lane] = acc[m][n];
  __syncthreads();
  for (int i = wave; i < MB * NB; i += kWaves) {
    floatx4 sum = parts[0][i][lane];
#pragma unroll
    for (int v = 1; v < kWaves; ++v)
      sum += parts[v][i][lane];
    const int col = col0 + i % NB * 16 + lane % 16;
    const int first = row0 + i / NB * 16 + 4 * part;
    const float ws = p.w_scales[min(col, p.out - 1)];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = first + r;
      const float xs = p.x_scales[min(row, p.rows - 1)];
      if (row < p.rows && col < p.out)
        static_cast<T*>(p.y)[row * p.y_stride + col] = static_cast<T>(sum[r] * xs * ws);
    }
  }
}

// ---------------------------------------------------------------- tiles
// BM rows by BN columns of a work-group, WM by WN waves, a ring of STAGES steps of both
// operands in LDS, filled by loads that go there directly. A row's 128 codes lie in LDS
// in 16-byte chunks, chunk c of row r at c ^ Swizzle(r), so that the 16 rows that a
// wave's operand reads at one c are in 16 different groups of banks (no conflicts by the
// counters; a third of the reads' time without).
//
// The weights are the left operand, so that a lane holds neighbouring columns of one
// row: their rows are dealt to the wave's FN operands such that a lane's 4 FN columns
// are next to each other.
//
// Bound by the matrix cores and the reads from LDS that feed them: 4096 x 4096 x 8192 takes
// 99 to 107 us in bf16 by card and run, 2780 to 2570 TFLOP/s, beside 97 to 104 of the card's
// library at 8 bits; float32, at half the products' rate, 198 to 203. Small products are bound
// by their steps' latency: 580 x 2048 x 1024 in float32 9.7 to 10.4 us, of which 16 steps, a
// launch and the results' stores.
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
struct Tile {
  static constexpr bool kHalf = std::is_same_v<T, float>;
  static constexpr int kWaveCount = WM * WN;
  static constexpr int kThreads = kWaveCount * kWave;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  // x has STAGES stages, w one more: its loads have a step more to arrive.
  static constexpr int kXBytes = BM * kStep, kWBytes = BN * kStep;
  static constexpr int kBytes = STAGES * kXBytes + (STAGES + 1) * kWBytes;
  static constexpr int kXLoads = BM / 8 / kWaveCount, kWLoads = BN / 8 / kWaveCount;
  static constexpr int kLoads = kXLoads + kWLoads;
  static_assert(BM % (8 * kWaveCount) == 0 && BN % (8 * kWaveCount) == 0, "whole loads a wave");
  static __device__ __forceinline__ int SwizzleX(int r) { return (r >> 1) & 7; }
  static __device__ __forceinline__ int SwizzleW(int r) {
    return ((r >> 1) & 1) | ((r / (4 * FN)) & 3) << 1;
  }
};

// A block of ROWS rows by COLS columns of a wave's results goes through the wave's part of
// LDS, so that every store writes whole runs of a row: 16 bytes a lane, next to each other.
// (Stores of a lane's own columns, 16 bytes of every 64, took 23 us of a tile of 256 by 256,
// these 4.) `staged` is what the lanes wrote; rows are kRowBytes apart.
template <typename T, int ROWS, int COLS>
struct Staged {
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kLanes = COLS / kVec;  // of a row
  static constexpr int kRowBytes = COLS * sizeof(T) + 16;
  static constexpr int kBytes = ROWS * kRowBytes;
  static __device__ __forceinline__ void Store(const unsigned char* staged, T* y,
                                               std::int64_t stride, int row0, int rows, int col0,
                                               int cols) {
    const int lane = threadIdx.x % kWave;
    const int col = col0 + lane % kLanes * kVec;
#pragma unroll
    for (int i = 0; i < ROWS; i += kWave / kLanes) {
      const int r = i + lane / kLanes;
      const unsigned char* const from = staged + r * kRowBytes + lane % kLanes * 16;
      T* const to = y + (row0 + r) * stride + col;
      if (row0 + r < rows && col + kVec <= cols)
        __builtin_memcpy(to, from, 16);
      else if (row0 + r < rows)
#pragma unroll 1
        for (int e = 0; col + e < cols; ++e)
          to[e] = reinterpret_cast<const T*>(from)[e];
    }
  }
};
// Between a wave's own writes and reads of LDS.
__device__ __forceinline__ void WaitLds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A work-group's tile. Work-groups go to the XCDs in turn: each XCD takes a run of tiles,
// ordered down columns of eight row tiles.
__device__ __forceinline__ void TileOf(int row_tiles, int col_tiles, int bm, int bn, int* row0,
                                       int* col0) {
  const int tiles = row_tiles * col_tiles;
  const int each = tiles / kXcds, rest = tiles % kXcds;
  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds;
  const int tile = xcd * each + min(xcd, rest) + at;
  const int band = tile / (8 * col_tiles);
  const int high = min(8, row_tiles - 8 * band);
  const int in_band = tile - band * 8 * col_tiles;
  *row0 = (band * 8 + in_band % high) * bm;
  *col0 = in_band / high * bn;
}

// Where a wave's part of the tile lies, and how it is fetched and read.
template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool WHOLE>
struct TileWork {
  using S = Tile<T, BM, BN, WM, WN, STAGES>;
  static constexpr int FM = S::FM, FN = S::FN;
  int wave, row0, col0, part, i16, first_row, first_col;
  std::uint32_t x_at[S::kXLoads], w_at[S::kWLoads], lds0;
  const unsigned char* x;
  const unsigned char* w;
  int x_read[2], w_read[2];

  __device__ __forceinline__ TileWork(const Linear8Params& p, int row_tiles, int col_tiles,
                                      const unsigned char* lds) {
    const int lane = threadIdx.x % kWave;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / WN, wn = wave % WN;
    TileOf(row_tiles, col_tiles, BM, BN, &row0, &col0);
    // This lane's chunk of the eight rows that one load brings.
    const int sub = lane / 8, chunk = lane % 8;
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
    x = p.x + row0 * p.x_stride;
    w = p.w + static_cast<std::size_t>(col0) * p.in;
    lds0 = LdsAddress(lds);
    // Operand m of x: rows 16 m + lane % 16 of the wave's; operand n of w: rows dealt.
    part = lane / 16;
    i16 = lane % 16;
    const int r = wm * FM * 16 + i16;
    const int c = wn * FN * 16 + (i16 / 4) * 4 * FN + i16 % 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x_read[h] = r * kStep + ((part + 4 * h) ^ S::SwizzleX(r)) * 16;
      w_read[h] = c * kStep + ((part + 4 * h) ^ S::SwizzleW(c)) * 16;
    }
    first_row = row0 + r;
    first_col = col0 + wn * FN * 16 + part * 4 * FN;
  }

  // Load i of this wave's of a step into a stage.
  __device__ __forceinline__ void LoadX(int step, int stage, int i) const {
    DmaToLds(x + step * kStep, x_at[i],
             lds0 + stage * S::kXBytes + (wave * S::kXLoads + i) * 1024);
  }
  __device__ __forceinline__ void LoadW(int step, int stage, int i) const {
    DmaToLds(w + step * kStep, w_at[i],
             lds0 + STAGES * S::kXBytes + stage * S::kWBytes + (wave * S::kWLoads + i) * 1024);
  }
  __device__ __forceinline__ void ReadX(const unsigned char* from, int m,
                                        Operand<S::kHalf>* to) const {
    to->Set(*reinterpret_cast<const intx4*>(from + x_read[0] + m * 16 * kStep),
            *reinterpret_cast<const intx4*>(from + x_read[1] + m * 16 * kStep));
  }
  __device__ __forceinline__ void ReadW(const unsigned char* from, int n,
                                        Operand<S::kHalf>* to) const {
    to->Set(*reinterpret_cast<const intx4*>(from + w_read[0] + n * 4 * kStep),
            *reinterpret_cast<const intx4*>(from + w_read[1] + n * 4 * kStep));
  }

  // The last, partial step, which comes straight from memory, and the results.
  __device__ __forceinline__ void Finish(const Linear8Params& p, floatx4 (&acc)[FM][FN],
                                         unsigned char* lds) const {
    const int steps = p.in / kStep;
    if (!WHOLE && p.in % kStep != 0) {
      Operand<S::kHalf> a, b[FN];
      const int k = steps * kStep + part * 32;
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const int c = first_col - part * 4 * FN + (i16 / 4) * 4 * FN + n * 4 + i16 % 4;
        LoadOperand(p.w + static_cast<std::size_t>(min(c, p.out - 1)) * p.in, k, p.in, &b[n]);
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
    using Out = Staged<T, 16, 16 * FN>;
    // All scales at once, before the first store.
    float ws[kCols], xs[FM];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      ws[c] = p.w_scales[min(first_col + c, p.out - 1)];
#pragma unroll
    for (int m = 0; m < FM; ++m)
      xs[m] = p.x_scales[min(first_row + 16 * m, p.rows - 1)];
    __syncthreads();  // the stages are read
    unsigned char* const staged = lds + wave * Out::kBytes;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      T v[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        v[c] = static_cast<T>(acc[m][c / 4][c % 4] * xs[m] * ws[c]);
      WaitLds();
      __builtin_memcpy(staged + i16 * Out::kRowBytes + part * kCols * sizeof(T), v, sizeof(v));
      WaitLds();
      Out::Store(staged, static_cast<T*>(p.y), p.y_stride, first_row - i16 + 16 * m, p.rows,
                 first_col - part * kCols, p.out);
    }
  }
};

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool WHOLE>
__global__ __launch_bounds__(WM* WN* kWave) void TileKernel(Linear8Params p, int row_tiles,
                                                            int col_tiles) {
  using S = Tile<T, BM, BN, WM, WN, STAGES>;
  constexpr int FM = S::FM, FN = S::FN;
  __shared__ __align__(16) unsigned char lds[S::kBytes];
  const TileWork<T, BM, BN, WM, WN, STAGES, WHOLE> t(p, row_tiles, col_tiles, lds);
  floatx4 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n)
      acc[m][n] = floatx4{0, 0, 0, 0};
  const int steps = p.in / kStep;
  // Loads in the order in which the loop goes on with them.
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    if (s > 0 && s - 1 < steps)
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i)
        t.LoadX(s - 1, s - 1, i);
    if (s < steps)
#pragma unroll
      for (int i = 0; i < S::kWLoads; ++i)
        t.LoadW(s, s, i);
  }
  int x_stage = 0, w_stage = 0;
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    if (step + STAGES - 1 < steps)
      WaitLoads<S::kWLoads + (STAGES - 2) * S::kLoads>();
    else
      WaitLoads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const unsigned char* const x_from = lds + x_stage * S::kXBytes;
    const unsigned char* const w_from = lds + STAGES * S::kXBytes + w_stage * S::kWBytes;
    const int x_to = x_stage == 0 ? STAGES - 1 : x_stage - 1;
    const int w_to = w_stage == 0 ? STAGES : w_stage - 1;
    Operand<S::kHalf> b[FN], a[2];
#pragma unroll
    for (int n = 0; n < FN; ++n)
      t.ReadW(w_from, n, &b[n]);
    t.ReadX(x_from, 0, &a[0]);
    // The loads go out a few at a time between the products: all at once they hold every
    // wave up until the address unit has taken them.
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      if (m + 1 < FM)
        t.ReadX(x_from, m + 1, &a[(m + 1) & 1]);
#pragma unroll
      for (int n = 0; n < FN; ++n)
        acc[m][n] = Multiply(b[n], a[m & 1], acc[m][n]);
      constexpr int kEach = (S::kLoads + FM - 1) / FM;
#pragma unroll
      for (int i = m * kEach; i < (m + 1) * kEach && i < S::kLoads; ++i) {
        if (i < S::kXLoads) {
          if (step + STAGES - 1 < steps)
            t.LoadX(step + STAGES - 1, x_to, i);
        } else if (step + STAGES < steps) {
          t.LoadW(step + STAGES, w_to, i - S::kXLoads);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" ::: "memory");
    x_stage = x_stage == STAGES - 1 ? 0 : x_stage + 1;
    w_stage = w_stage == STAGES ? 0 : w_stage + 1;
  }
  t.Finish(p, acc, lds);
}

template <typename T>
void Launch(const Linear8Params& p, hipStream_t s) {
  const auto groups = [&](int bm, int bn) {
    return static_cast<std::int64_t>((p.rows + bm - 1) / bm) * ((p.out + bn - 1) / bn);
  };
  // Twice the columns, which halves what is read of x, where a work-group is left to every
  // CU (32 x 8192 x 8192: 18.9 us, 24.5 without; 32 x 4096 x 4096, 128 work-groups: 10.2, 8.4
  // without).
  const auto skinny_of = [&](auto mb, auto nb) {
    constexpr int kRows = 16 * mb(), kCols = 16 * nb();
    Dispatch(SkinnyKernel<T, mb(), nb()>,
             dim3((p.out + kCols - 1) / kCols, (p.rows + kRows - 1) / kRows),
             dim3(kWaves * kWave), 0, s, true, true, p);
  };
  const auto skinny = [&](auto mb) {
    if (groups(16 * mb(), 32) >= kCus)
      skinny_of(mb, std::integral_constant<int, 2>());
    else
      skinny_of(mb, std::integral_constant<int, 1>());
  };
  const auto tiled = [&](auto bm, auto bn, auto wm, auto wn, auto stages, auto whole) {
    const int row_tiles = (p.rows + bm() - 1) / bm(), col_tiles = (p.out + bn() - 1) / bn();
    Require(static_cast<std::int64_t>(row_tiles) * col_tiles < (1 << 23),
            "linear: too many tiles");
    Dispatch(TileKernel<T, bm(), bn(), wm(), wn(), stages(), whole()>, dim3(row_tiles * col_tiles),
             dim3(wm() * wn() * kWave), 0, s, true, true, p, row_tiles, col_tiles);
  };
  using std::integral_constant;
  if (p.rows <= 32 || groups(64, 64) < kCus / 6 || p.x_stride > kTileStride) {
    // Few rows, or few tiles: 64 x 4096 x 2048 (32 tiles) takes 8.4 us, 10.8 with tiles, 64 x
    // 4096 x 3000 (47) 13.6 and 10.9, 64 x 8192 x 8192 32 and 22; 32 x 4096 x 4096, half of
    // whose tiles' rows are none, 8.4 and 10.8 (bf16; in float32 tiles take half as long again).
    // 32 rows to a work-group where that leaves one to every CU: 32 x 8192 x 8192 24.5 us, 31
    // with 16; 64 x 4096 x 1024, 128 work-groups of 32, 8.0 and 6.3.
    if (p.rows > 16 && groups(32, 16) >= kCus)
      skinny(integral_constant<int, 2>());
    else
      skinny(integral_constant<int, 1>());
  } else if (p.in % kStep == 0 && groups(256, 256) >= kCus) {
    // A tile for every CU: 4096 x 4096 x 4096 takes 54 us, 62 in tiles of 128, 4096 x 4096 x
    // 2048, half as many, 46 and 34; float32 98 and 112, 90 and 61. Without the partial step
    // the kernel's code is as long as its registers reach.
    tiled(integral_constant<int, 256>(), integral_constant<int, 256>(),
          integral_constant<int, 2>(), integral_constant<int, 4>(), integral_constant<int, 2>(),
          std::true_type());
  } else if (groups(128, 128) > kCus) {
    // 4096 x 4096 x 2048 (512 tiles) takes 34 us, 49 in tiles of 64, 3000 x 2048 x 2048 (384)
    // 18.8 and 21.7, 2048 x 2048 x 2048 (256) 14.2 and 14.0, 1500 x 2048 x 2048 (192) 13.9 and
    // 11.8; float32 61 and 74, 31 and 32, 23 and 22, 22 and 18.
    tiled(integral_constant<int, 128>(), integral_constant<int, 128>(),
          integral_constant<int, 2>(), integral_constant<int, 2>(), integral_constant<int, 2>(),
          std::false_type());
  } else if (groups(64, 64) > 2 * kCus) {
    // Four stages leave two work-groups to a CU, two four: 1400 x 2048 x 2048 (704 tiles)
    // takes 11.6 us with two stages, 13.9 with four, 1000 x 1024 x 2048 (512) 7.0 and 6.6, 580
    // x 2048 x 1024 (160) 10.2 and 7.2; float32 18.1 and 20.8, 9.4 and 9.7, 12.2 and 10.3.
    tiled(integral_constant<int, 64>(), integral_constant<int, 64>(),
          integral_constant<int, 2>(), integral_constant<int, 2>(), integral_constant<int, 2>(),
          std::false_type());
  } else {
    tiled(integral_constant<int, 64>(), integral_constant<int, 64>(),
          integral_constant<int, 2>(), integral_constant<int, 2>(), integral_constant<int, 4>(),
          std::false_type());
  }
}

}  // namespace

void LaunchLinear8(const Linear8Params& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.rows <= kMostRows && p.in >= 16 && p.in % 16 == 0 && p.out >= 1,
          "linear: shape outside the kernel's range");
  WithType(type, [&](auto t) { Launch<decltype(t)>(p, stream); });
  Check(hipGetLastError(), "linear launch");
}

}  // namespace ovg
