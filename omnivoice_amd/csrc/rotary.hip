// Rotary positions: pairs of a head's dims turned by their position's angle.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) * magnitude, t = position * f[i]
//
// for pair i < rotary / 2: dims i and i + rotary / 2 (half layout) or 2 i and 2 i + 1
// (interleaved); dims from `rotary` on stay. With norm weights the head is first
// y = weight * (x * rsqrt(mean x^2 + eps)), all dims of it.
//
// The angle is formed in 64 bits and brought into an eighth of a turn around zero
// there, so that far positions lose nothing; its sine and cosine are Taylor sums in
// float32 (their rest is under 2^-29). A work-group has a row, whose sines and cosines
// go to LDS once for all heads. A lane has eight pairs in a row of a head, 16-byte loads
// where the layout's sizes are multiples of eight pairs, a power of two of lanes a head.
// Bound by memory: 12000 rows of 24 heads of 128 in bf16, 147 MB, take 33.7 us (4.4
// TB/s; a copy reaches 5.0 to 5.3); 48 rows of 24 heads, normed, 4.5 us, of which 2 are a
// launch and the rest one latency of loads, the turns beside it, and the stores.
#include "step.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

constexpr int kThreads = 256;
constexpr int kPairs = 8;  // of a lane

// cos and sin of position * f.
__device__ __forceinline__ float2 Turn(int position, float f) {
  const double turns =
      static_cast<double>(position) * static_cast<double>(f) * 0.15915494309189533577;
  const double quarters = turns * 4.0;
  const double whole = rint(quarters);
  const float a = static_cast<float>((quarters - whole) * 1.57079632679489661923);
  const int turn = static_cast<int>(static_cast<long long>(whole)) & 3;
  const float q = a * a;
  const float s = a + a * q * (-1.0F / 6 + q * (1.0F / 120 + q * (-1.0F / 5040 + q * (1.0F / 362880))));
  const float c = 1.0F + q * (-0.5F + q * (1.0F / 24 + q * (-1.0F / 720 + q * (1.0F / 40320 + q * (-1.0F / 3628800)))));
  const float x = turn & 1 ? s : c, y = turn & 1 ? c : s;
  return float2{turn == 1 || turn == 2 ? -x : x, turn >= 2 ? -y : y};
}

// Elements of pair-slot s: the pairs, then what stays two by two.
template <bool INTERLEAVED>
__device__ __forceinline__ void ElementsOf(int s, int half, int dim, int* lo, int* hi) {
  if (INTERLEAVED) {
    *lo = 2 * s;
    *hi = 2 * s + 1;
  } else if (s < half) {
    *lo = s;
    *hi = s + half;
  } else {
    *lo = half + s;
    *hi = s + dim / 2;
  }
}

template <typename T, bool INTERLEAVED, bool VECTOR>
__global__ __launch_bounds__(kThreads) void RotaryKernel(RotaryParams p, int lanes) {
  __shared__ float2 turns[kMostRotaryDim / 2];
  __shared__ int held;
  const int tid = threadIdx.x, row = blockIdx.x;
  const int half = p.rotary / 2, slots = p.dim / 2;
  // A group of lanes a head.
  const int groups = kThreads / lanes, lane = tid % lanes;
  const int heads = p.heads[0] + p.heads[1];
  const int s0 = lane * kPairs;
  const bool there = s0 < slots;
  int lo, hi;
  ElementsOf<INTERLEAVED>(s0, half, p.dim, &lo, &hi);
  float a[kPairs], b[kPairs];
  const auto load = [&](int head) {
    const int which = head >= p.heads[0];
    const T* x = static_cast<const T*>(p.x[which]) + row * p.x_stride[which] +
                 static_cast<std::int64_t>(head - (which ? p.heads[0] : 0)) * p.dim;
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      a[i] = b[i] = 0.0F;
    if (!there)
      return;
    if (VECTOR && INTERLEAVED) {
      float v[2 * kPairs];
      LoadFloats<2 * kPairs>(x + lo, v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        a[i] = v[2 * i];
        b[i] = v[2 * i + 1];
      }
    } else if (VECTOR) {
      LoadFloats<kPairs>(x + lo, a);
      LoadFloats<kPairs>(x + hi, b);
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        if (s0 + i < slots) {
          int l, h;
          ElementsOf<INTERLEAVED>(s0 + i, half, p.dim, &l, &h);
          a[i] = static_cast<float>(x[l]);
          b[i] = static_cast<float>(x[h]);
        }
    }
  };

  // The first head's loads are on their way while the first wave forms the turns.
  int head = tid / lanes;
  if (head < heads)
    load(head);
  if (tid < kWave) {
    int position = 0;
    bool valid = true;
    if (p.positions != nullptr) {
      position = p.positions[row];
    } else {
      const Found f = FindItem(p.sequences, 1, 0, 0, row);
      valid = f.item >= 0 && f.item < f.span.count;
      position = f.span.start + f.item;
    }
    for (int i = tid; i < half; i += kWave) {
      const float2 t = Turn(position, p.frequencies[i]);
      turns[i] = float2{t.x * p.magnitude, t.y * p.magnitude};
    }
    if (tid == 0)
      held = valid;
  }
  __syncthreads();
  if (!held)
    return;

  while (head < heads) {
    const int which = head >= p.heads[0];
    const float* const norm = p.norm[which];
    if (norm != nullptr) {
      float squares = 0.0F;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        squares += a[i] * a[i] + b[i] * b[i];
      for (int offset = lanes / 2; offset > 0; offset /= 2)
        squares += __shfl_xor(squares, offset);
      const float mean = squares / static_cast<float>(p.dim) + p.eps;
      float factor = rsqrtf(mean);
      if (!(mean > 1e-30F && mean < __builtin_inff())) {  // the same in the head's lanes
        double wide = 0.0;
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          wide += static_cast<double>(a[i]) * a[i] + static_cast<double>(b[i]) * b[i];
        for (int offset = lanes / 2; offset > 0; offset /= 2)
          wide += __shfl_xor(wide, offset);
        factor = static_cast<float>(1.0 / sqrt(wide / p.dim + static_cast<double>(p.eps)));
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        if (s0 + i < slots) {
          int l, h;
          ElementsOf<INTERLEAVED>(s0 + i, half, p.dim, &l, &h);
          a[i] = norm[l] * (a[i] * factor);
          b[i] = norm[h] * (b[i] * factor);
        }
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      if (s0 + i < half) {
        const float2 t = turns[s0 + i];
        const float x0 = a[i], x1 = b[i];
        a[i] = x0 * t.x - x1 * t.y;
        b[i] = x1 * t.x + x0 * t.y;
      }
    T* out = static_cast<T*>(p.out[which]) + row * p.out_stride[which] +
             static_cast<std::int64_t>(head - (which ? p.heads[0] : 0)) * p.dim;
    if (!there) {
    } else if (VECTOR && INTERLEAVED) {
      float v[2 * kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        v[2 * i] = a[i];
        v[2 * i + 1] = b[i];
      }
      StoreFloats<2 * kPairs>(out + lo, v);
    } else if (VECTOR) {
      StoreFloats<kPairs>(out + lo, a);
      StoreFloats<kPairs>(out + hi, b);
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        if (s0 + i < slots) {
          int l, h;
          ElementsOf<INTERLEAVED>(s0 + i, half, p.dim, &l, &h);
          out[l] = static_cast<T>(a[i]);
          out[h] = static_cast<T>(b[i]);
        }
    }
    head += groups;
    if (head < heads)
      load(head);
  }
}

}  // namespace

void LaunchRotary(const RotaryParams& p, bool interleaved, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.dim >= 2 && p.dim <= kMostRotaryDim && p.dim % 2 == 0 &&
              p.rotary >= 2 && p.rotary <= p.dim && p.rotary % 2 == 0,
          "rotary: shape outside the kernel's range");
  int lanes = 1;
  while (lanes * kPairs < p.dim / 2)
    lanes *= 2;
  // Else a head's eight pairs may hold turned and other dims, or begin at any element.
  const bool vector = p.dim % (2 * kPairs) == 0 && (interleaved || p.rotary % (2 * kPairs) == 0);
  WithType(type, [&](auto t) {
    using T = decltype(t);
    const auto launch = [&](auto i, auto v) {
      Dispatch(RotaryKernel<T, i(), v()>, dim3(p.rows), dim3(kThreads), 0, stream, true, true, p,
               lanes);
    };
    if (interleaved && vector)
      launch(std::true_type(), std::true_type());
    else if (interleaved)
      launch(std::true_type(), std::false_type());
    else if (vector)
      launch(std::false_type(), std::true_type());
    else
      launch(std::false_type(), std::false_type());
  });
  Check(hipGetLastError(), "rotary launch");
}

}  // namespace ovg
