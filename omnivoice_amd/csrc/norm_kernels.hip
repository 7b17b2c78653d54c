// Rows of a layer's stream: RMS norm with the residual's addition, and rows in 8
// bits with their scale, plain or gated.
//
//   norm:     s = x + residual (float32, rounded to the residual's type, stored)
//             y = weight * (s * rsqrt(mean s^2 + eps))
//   quantize: y = x, or x * g / (1 + exp(-g))
//   8 bits:   scale = the smallest power of two, 2^-100 or more, with
//             max |y| / scale <= 448; e4m3 codes of y / scale, to nearest even
//
// A row lies in the registers of a wave (to 2048 elements), of four waves (to 8192)
// or of sixteen, eight elements in a row to a lane, so that it is read once; the
// sums are joined over the lanes by DPP and over the waves through LDS, in a fixed
// order. Bound by memory: 16384 rows of 1024 bf16 with a bf16 residual to 8 bits, 118
// MB, take 22.5 us from inputs in the caches and 27 from memory (4.4 TB/s; a copy
// reaches 5.0 to 5.3), 580 rows of 4096 gated in fp16 6 us, of which 2.4 are their
// bytes' and the rest a launch and the latency of load, sum and store. Sums are float32. Where
// the largest magnitude is so near to a power's border that float32 may have taken it over
// (kBeside), or the squares leave float32's range, the row is summed and its maximum found
// again in 64 bits, so that the scale is the one that the formulas give.
#include "step.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

constexpr int kVec = 8;  // a lane's elements in a row
constexpr int kRowThreads = 256;

enum class Mode { kNorm, kPlain, kGate };

struct None {};

template <int THREADS>
struct Group {
  // Joins over the row's lanes; `scratch` holds a slot a wave. Every lane gets the
  // result.
  template <typename T, typename F>
  static __device__ __forceinline__ T Join(T v, T* scratch, F&& join) {
    for (int offset = kWave / 2; offset > 0; offset /= 2)
      v = join(v, __shfl_xor(v, offset));
    if constexpr (THREADS > kWave) {
      const int wave = threadIdx.x / kWave;
      __syncthreads();  // the slots' last readers are done
      if (threadIdx.x % kWave == 0)
        scratch[wave] = v;
      __syncthreads();
      v = scratch[0];
      for (int i = 1; i < THREADS / kWave; ++i)
        v = join(v, scratch[i]);
    }
    return v;
  }
  static __device__ __forceinline__ float Sum(float v, double* scratch) {
    v = WaveSumFast(v);
    if constexpr (THREADS > kWave) {
      float* slots = reinterpret_cast<float*>(scratch);
      __syncthreads();
      if (threadIdx.x % kWave == 0)
        slots[threadIdx.x / kWave] = v;
      __syncthreads();
      v = slots[0];
      for (int i = 1; i < THREADS / kWave; ++i)
        v += slots[i];
    }
    return v;
  }
  static __device__ __forceinline__ unsigned Max(unsigned v, double* scratch) {
    return Join(v, reinterpret_cast<unsigned*>(scratch),
                [](unsigned a, unsigned b) { return max(a, b); });
  }
  static __device__ __forceinline__ double Sum(double v, double* scratch) {
    return Join(v, scratch, [](double a, double b) { return a + b; });
  }
  static __device__ __forceinline__ double Max(double v, double* scratch) {
    return Join(v, scratch, [](double a, double b) { return fmax(a, b); });
  }
};

// The exponent of the smallest power of two, -100 or more, that takes amax into
// +-448 = 1.75 * 2^8.
__device__ __forceinline__ int ScaleExponent(unsigned amax) {
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u);
  return max(e, -100);
}
__device__ __forceinline__ int ScaleExponent(double amax) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, amax);
  const int e = static_cast<int>(bits >> 52) - 1023 - 8 +
                ((bits & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull);
  return max(e, -100);
}
__device__ __forceinline__ float PowerOf(int e) {  // -126 .. 127
  return __uint_as_float(static_cast<unsigned>(e + 127) << 23);
}

__device__ __forceinline__ float Gated(float x, float g) { return x * (g / (1.0F + __expf(-g))); }
// From -88 down to where nothing is left of float32's largest number: x g e^g, of which e^g
// alone is below float32's range. e^g = 2^n 2^f.
constexpr float kDeep = -88.0F;
__device__ __forceinline__ bool Deep(float g) { return g < kDeep && g > -300.0F; }
__device__ __forceinline__ float GatedDeep(float x, float g) {
  constexpr double kLog2E = 1.4426950408889634074;
  constexpr float kHigh = static_cast<float>(kLog2E), kLow = static_cast<float>(kLog2E - kHigh);
  const float n = rintf(g * kHigh);
  const float f = fmaf(g, kHigh, -n) + g * kLow;
  return ldexpf(ldexpf(x, -32) * (g * __builtin_amdgcn_exp2f(f)), static_cast<int>(n) + 32);
}

// How many steps of 2^-23 from a power's border, 1.75, float32 may take a row's largest
// value over it. A norm is off by 26 * 2^-24: 23 steps. e^-g is off by 1.5 |g| 2^-24, the
// product's and the constant's roundings, and 2^-23 of its own, the rest by 6 * 2^-24: 123
// steps for a gate of -88, and fewer where the power is formed in two parts.
template <Mode MODE>
constexpr int kBeside = MODE == Mode::kGate ? 128 : 32;

// Eight elements of a row, those before `d` and behind the row not among them: a
// row's last, partial run is loaded from its end backwards, so that no load is
// conditional.
template <typename T>
__device__ __forceinline__ void LoadRun(const T* row, int d, int width, float (&v)[kVec]) {
  if (width >= kVec) {
    LoadFloats<kVec>(row + min(d, width - kVec), v);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      v[i] = i < width ? static_cast<float>(row[i]) : 0.0F;
  }
}
// First element of the run that LoadRun gives for `d`.
__device__ __forceinline__ int RunStart(int d, int width) {
  return width >= kVec ? min(d, width - kVec) : 0;
}
__device__ __forceinline__ bool Owned(int e, int d, int width) { return e >= d && e < width; }

template <typename T>
__device__ __forceinline__ void StoreRun(T* row, int d, int width, const float (&v)[kVec]) {
  if (d + kVec <= width) {
    StoreFloats<kVec>(row + d, v);
    return;
  }
  const int start = RunStart(d, width);
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (Owned(start + i, d, width))
      row[start + i] = static_cast<T>(v[i]);
}

__device__ __forceinline__ unsigned Encode4(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
__device__ __forceinline__ void StoreCodes(unsigned char* row, int d, int width,
                                           const float (&v)[kVec]) {
  const unsigned w[2] = {Encode4(v[0], v[1], v[2], v[3]), Encode4(v[4], v[5], v[6], v[7])};
  if (d + kVec <= width) {
    __builtin_memcpy(row + d, w, sizeof(w));
    return;
  }
  const int start = RunStart(d, width);
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (Owned(start + i, d, width))
      row[start + i] = static_cast<unsigned char>(w[i / 4] >> (8 * (i % 4)));
}

// `In` and `Second` are the elements' types (None: there is none), `Out` too
// (unsigned char: e4m3). THREADS a row, CHUNKS runs a lane.
template <typename In, typename Second, typename Out, Mode MODE, int THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS < kRowThreads ? kRowThreads : THREADS) void RowKernel(
    RowParams p) {
  using Lanes = Group<THREADS>;
  constexpr int kRows = THREADS < kRowThreads ? kRowThreads / THREADS : 1;
  constexpr bool kCodes = std::is_same_v<Out, unsigned char>;
  constexpr bool kSecond = !std::is_same_v<Second, None>;
  __shared__ double scratch[16];
  const int tid = threadIdx.x % THREADS;
  const int row = blockIdx.x * kRows + threadIdx.x / THREADS;
  if (row >= p.rows)  // whole waves; with more than one a row there is one row
    return;
  const int width = p.width;
  const In* const x = static_cast<const In*>(p.x) + row * p.x_stride;

  // The weights, or gates, and the results stay in registers where there is room. The
  // lanes of 1024 have 128 registers: from 32 elements a lane on weights and gates are read
  // again from the caches, a run after the other.
  constexpr bool kHeld = THREADS < 1024 || CHUNKS <= 2;
  const auto one_by_one = [] {
    if constexpr (!kHeld)
      __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int kHolds = kHeld && MODE != Mode::kPlain ? CHUNKS : 1;
  float v[CHUNKS][kVec];
  float g[kHolds][kVec];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    LoadRun(x, (c * THREADS + tid) * kVec, width, v[c]);
  const auto load_g = [&](int c, float (&to)[kVec]) {
    if constexpr (MODE == Mode::kNorm)
      LoadRun(p.weight, (c * THREADS + tid) * kVec, width, to);
    else if constexpr (MODE == Mode::kGate)
      LoadRun(static_cast<const Second*>(p.second) + row * p.second_stride,
              (c * THREADS + tid) * kVec, width, to);
  };
  if constexpr (kHeld && MODE != Mode::kPlain) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      load_g(c, g[c]);
  }
  if constexpr (kSecond) {
    const Second* const second = static_cast<const Second*>(p.second) + row * p.second_stride;
    if constexpr (MODE != Mode::kGate) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float s[kVec];
        LoadRun(second, (c * THREADS + tid) * kVec, width, s);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          v[c][i] = static_cast<float>(static_cast<Second>(v[c][i] + s[i]));
        one_by_one();
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int d = (c * THREADS + tid) * kVec, start = RunStart(d, width);
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (!Owned(start + i, d, width))
        v[c][i] = 0.0F;
  }

  // The factor of a norm's row.
  float factor = 1.0F;
  bool careful = false;
  const auto total64 = [&] {
    double t = 0.0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        t += static_cast<double>(v[c][i]) * static_cast<double>(v[c][i]);
      one_by_one();
    }
    return 1.0 / sqrt(Lanes::Sum(t, scratch) / width + static_cast<double>(p.eps));
  };
  if constexpr (MODE == Mode::kNorm) {
    float squares = 0.0F;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float part = 0.0F;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        part += v[c][i] * v[c][i];
      squares += part;
    }
    squares = Lanes::Sum(squares, scratch);
    const float mean = squares / static_cast<float>(width) + p.eps;
    factor = rsqrtf(mean);
    careful = !(mean > 1e-30F && mean < __builtin_inff());
    if (careful)
      factor = static_cast<float>(total64());
    if constexpr (kSecond) {
      Second* const total = static_cast<Second*>(p.total) + row * p.total_stride;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        StoreRun(total, (c * THREADS + tid) * kVec, width, v[c]);
    }
  }
  // The weights or gates of a run, and its results.
  const auto g_of = [&](int c, float (&to)[kVec]) {
    if constexpr (kHeld && MODE != Mode::kPlain) {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        to[i] = g[c][i];
    } else {
      load_g(c, to);
    }
  };
  float deepest = 0.0F;
  bool deep = false;  // the wave's gates go below kDeep
  const auto values = [&](int c, float (&to)[kVec]) {
    float by[kVec];
    g_of(c, by);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if constexpr (MODE == Mode::kNorm)
        to[i] = by[i] * (v[c][i] * factor);
      else if constexpr (MODE == Mode::kGate)
        to[i] = Gated(v[c][i], by[i]);
      else
        to[i] = v[c][i];
    }
    if constexpr (MODE == Mode::kGate) {
      // Asked once for all runs where they are held, for each where they are not: 512 rows of
      // 65536 in fp16 take 80 us so, 104 with one question (91 without any).
      if (!deep) {
        float least = by[0];
#pragma unroll
        for (int i = 1; i < kVec; ++i)
          least = fminf(least, by[i]);
        deepest = kHeld ? fminf(deepest, least) : least;
      }
      if (kHeld ? deep : __any(deepest < kDeep))
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          to[i] = Deep(by[i]) ? GatedDeep(v[c][i], by[i]) : to[i];
    }
  };

  if constexpr (!kCodes) {
    Out* const out = static_cast<Out*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float y[kVec];
      values(c, y);
      StoreRun(out, (c * THREADS + tid) * kVec, width, y);
      one_by_one();
    }
  } else {
    // The order of magnitudes' bits is the magnitudes' own, infinities and NaN
    // behind every number. A run's elements of other lanes are zeros times the row's own
    // weights or gates: a NaN there is the row's, too.
    float held[kHeld ? CHUNKS : 1][kVec];
    unsigned amax = 0;
    const auto all_values = [&] {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        auto& y = held[kHeld ? c : 0];
        values(c, y);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          amax = max(amax, __float_as_uint(y[i]) & 0x7FFFFFFFu);
        one_by_one();
      }
    };
    all_values();
    if constexpr (MODE == Mode::kGate && kHeld) {
      deep = __any(deepest < kDeep);
      if (deep)  // hardly ever
        all_values();
    }
    amax = Lanes::Max(amax, scratch);
    const bool lost = amax >= 0x7F800000u;
    int e = ScaleExponent(amax);
    if constexpr (MODE != Mode::kPlain) {
      const int off = static_cast<int>(amax & 0x7FFFFFu) - 0x600000;
      if (!lost && (careful || (off <= kBeside<MODE> && off >= -kBeside<MODE>))) {
        double most = 0.0;
        const double r = MODE == Mode::kNorm ? total64() : 1.0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          auto& y = held[kHeld ? c : 0];
          if (!kHeld)
            values(c, y);
          float by[kVec];
          g_of(c, by);
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            // Far from the largest they cannot be it.
            if (!(fabsf(y[i]) >= __uint_as_float(amax) * 0.999F))
              continue;
            const double a = v[c][i], b = by[i];
            most = fmax(most, fabs(MODE == Mode::kNorm ? b * a * r : a * (b / (1.0 + exp(-b)))));
          }
          one_by_one();
        }
        e = ScaleExponent(Lanes::Max(most, scratch));
      }
    }
    const float inverse = lost ? 0.0F : PowerOf(-e);
    unsigned char* const out = static_cast<unsigned char*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      auto& y = held[kHeld ? c : 0];
      if (!kHeld)
        values(c, y);
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        y[i] = lost ? 0.0F : y[i] * inverse;
      StoreCodes(out, (c * THREADS + tid) * kVec, width, y);
      one_by_one();
    }
    if (tid == 0)
      p.scales[row] = lost ? __builtin_nanf("") : PowerOf(e);
  }
}

template <typename In, typename Second, typename Out, Mode MODE>
void LaunchRows(const RowParams& p, hipStream_t s) {
  const auto launch = [&](auto threads, auto chunks) {
    constexpr int kThreads = threads() < kRowThreads ? kRowThreads : threads();
    constexpr int kRows = kThreads / threads();
    Dispatch(RowKernel<In, Second, Out, MODE, threads(), chunks()>,
             dim3((p.rows + kRows - 1) / kRows), dim3(kThreads), 0, s, true, true, p);
  };
  // As few lanes as hold the row: more waves a row join through LDS and leave lanes idle,
  // more runs a lane cost registers that other rows' waves would have. bf16 norms to 8 bits:
  // 16384 x 1024 takes 22.5 us in 64 lanes of 2 runs, 38.6 of 4; 8192 x 2048 25.8 in 64 of 4,
  // 32.2 in 256 of 2 (16 rows 5.4 and 4.4); 580 x 4096 6.6 in 256 of 2, 9.4 of 4; 4096 x 8192
  // 60 in 256 of 4, 103 in 1024 of 2; 2048 x 16384 64 in 1024 of 2, 92 of 4; 1024 x 32768 61 in
  // 1024 of 4, 209 of 8.
  using std::integral_constant;
  if (p.width <= 2 * kVec * kWave)
    launch(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (p.width <= 4 * kVec * kWave)
    launch(integral_constant<int, 64>(), integral_constant<int, 4>());
  else if (p.width <= 2 * kVec * 256)
    launch(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (p.width <= 4 * kVec * 256)
    launch(integral_constant<int, 256>(), integral_constant<int, 4>());
  else if (p.width <= 2 * kVec * 1024)
    launch(integral_constant<int, 1024>(), integral_constant<int, 2>());
  else if (p.width <= 4 * kVec * 1024)
    launch(integral_constant<int, 1024>(), integral_constant<int, 4>());
  else
    launch(integral_constant<int, 1024>(), integral_constant<int, 8>());
}

template <typename In, typename Second>
void NormTo(const RowParams& p, DType out, hipStream_t s) {
  if (out == DType::kE4m3)
    LaunchRows<In, Second, unsigned char, Mode::kNorm>(p, s);
  else
    WithType(out, [&](auto o) { LaunchRows<In, Second, decltype(o), Mode::kNorm>(p, s); });
}

void CheckRows(const RowParams& p) {
  Require(p.rows >= 1 && p.rows <= kMostRows && p.width >= 1 && p.width <= kMostWidth,
          "rows: shape outside the kernel's range");
}

}  // namespace

void LaunchAddNorm(const RowParams& p, DType x, DType second, DType out, hipStream_t stream) {
  CheckRows(p);
  Require(second == DType::kE4m3 || second == x || second == DType::kF32,
          "norm: the residual is float32 or of x's type");
  WithType(x, [&](auto in) {
    using In = decltype(in);
    if (second == DType::kE4m3)
      NormTo<In, None>(p, out, stream);
    else if (second == x)
      NormTo<In, In>(p, out, stream);
    else
      NormTo<In, float>(p, out, stream);
  });
  Check(hipGetLastError(), "norm launch");
}

void LaunchQuantize(const RowParams& p, DType x, hipStream_t stream) {
  CheckRows(p);
  WithType(x, [&](auto in) {
    using In = decltype(in);
    if (p.second != nullptr)
      LaunchRows<In, In, unsigned char, Mode::kGate>(p, stream);
    else
      LaunchRows<In, None, unsigned char, Mode::kPlain>(p, stream);
  });
  Check(hipGetLastError(), "quantize launch");
}

}  // namespace ovg
