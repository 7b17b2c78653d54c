// Log probabilities of given tokens with the entropy and the best
// alternatives of their distributions, in one pass over the logits.
//
//   z = c, or c + g (c - u) with unconditional logits, each step rounded to
//   float32 (c = -inf stays -inf, the token being impossible)
//   Z = log sum exp z, log p(token) = z[token] - Z, H = Z - sum p z
//
// A wave keeps, per lane, the maximum m so far, s = sum exp(z - m) and
// t = sum exp(z - m) (z - m), so that H = log s - t / s needs no second pass.
// The best `top` values are a list in the wave's lanes, lane j holding the
// j-th. What may enter it is found by comparing against its last value, which
// few elements pass; for the first segment of a wave, whose list is empty, the
// top-th largest of the lanes' own maxima stands in (that many elements reach
// it, so no lower one can be listed).
#include "cache.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

constexpr int kWaves = 4;
constexpr int kElements = 16;  // a lane's elements of a segment
constexpr float kLog2e = 1.44269504088896341F;

__device__ __forceinline__ float ExpOf(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// (value, index) pairs in descending order, equal values by index.
__device__ __forceinline__ bool Before(float a, int i, float b, int j) {
  return a > b || (a == b && i < j);
}

struct Alternatives {
  float value;  // lane j: the j-th best so far
  int index;
  int top;
  // Every lane's (v, i) is the same.
  __device__ __forceinline__ void Insert(float v, int i, int lane) {
    const unsigned long long ahead = __ballot(lane < top && Before(value, index, v, i));
    const int at = __popcll(ahead);
    const float up = __shfl_up(value, 1);
    const int up_index = __shfl_up(index, 1);
    if (lane == at) {
      value = v;
      index = i;
    } else if (lane > at) {
      value = up;
      index = up_index;
    }
  }
};

struct Sums {
  float m, s, t;
  __device__ __forceinline__ void Move(float to) {
    const float d = m == -__builtin_inff() ? 0.0F : m - to;
    const float f = ExpOf(d);
    t = (t + s * d) * f;
    s = s * f;
    m = to;
  }
};

template <typename T>
__device__ __forceinline__ float Guided(const T* c, const T* u, std::int64_t at, float g) {
  const float x = static_cast<float>(c[at]);
  if (u == nullptr)
    return x;
  const float d = x - static_cast<float>(u[at]);
  const float z = x + g * d;
  return x == -__builtin_inff() ? x : z;
}

// One work-group of four waves per row.
template <typename T>
__global__ __launch_bounds__(kWaves* kWave) void LogprobKernel(LogprobParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const std::int64_t row = blockIdx.x;
  const T* const c = static_cast<const T*>(p.logits) + row * p.stride;
  const T* const u =
      p.uncond == nullptr ? nullptr : static_cast<const T*>(p.uncond) + row * p.uncond_stride;
  const float inf = __builtin_inff();
  Sums sums{-inf, 0.0F, 0.0F};
  Alternatives best{-inf, -1, p.top};
  constexpr int kSegment = kElements * kWave;
  for (int base = wave * kSegment; base < p.vocab; base += kWaves * kSegment) {
    float z[kElements];
    float peak = -inf, listed = -inf;
#pragma unroll
    for (int e = 0; e < kElements; ++e) {
      const int at = base + e * kWave + lane;
      z[e] = at < p.vocab ? Guided(c, u, at, p.guidance) : -inf;
      peak = fmaxf(peak, z[e]);
      listed = at == p.mask_id ? listed : fmaxf(listed, z[e]);
    }
    if (peak > sums.m)
      sums.Move(peak);
    const float from = sums.m == -inf ? 0.0F : sums.m;
#pragma unroll
    for (int e = 0; e < kElements; ++e) {
      const float d = z[e] - from;
      const float x = ExpOf(d);
      sums.s += x;
      sums.t += d < -1000.0F ? 0.0F : x * d;
    }
    if (p.top == 0)
      continue;
    float floor = __shfl(best.value, p.top - 1);
    int floor_index = __shfl(best.index, p.top - 1);
    if (floor == -inf) {
      // The list is not full: take the top-th largest lane maximum.
      float mine = listed;
      for (int k = 0; k < p.top; ++k) {
        floor = WaveMax(mine);
        const unsigned long long who = __ballot(mine == floor);
        if (lane == __ffsll(who) - 1)
          mine = -inf;
      }
      floor_index = 0x7FFFFFFF;
    }
#pragma unroll
    for (int e = 0; e < kElements; ++e) {
      const int at = base + e * kWave + lane;
      unsigned long long left = __ballot(z[e] > -inf && at != p.mask_id &&
                                         Before(z[e], at, floor, floor_index));
      while (left != 0) {
        const int who = __ffsll(left) - 1;
        left &= left - 1;
        const float v = __shfl(z[e], who);
        const int i = base + e * kWave + who;
        if (Before(v, i, __shfl(best.value, p.top - 1), __shfl(best.index, p.top - 1)))
          best.Insert(v, i, lane);
      }
    }
  }
  // The wave's sums, then the work-group's.
  const float m = WaveMax(sums.m);
  sums.Move(m == -inf ? sums.m : m);
  sums.s = WaveSum(sums.s);
  sums.t = WaveSum(sums.t);
  __shared__ Sums shared[kWaves];
  __shared__ float shared_value[kWaves][kMostAlternatives];
  __shared__ int shared_index[kWaves][kMostAlternatives];
  if (lane == 0)
    shared[wave] = {m, sums.s, sums.t};
  if (lane < p.top) {
    shared_value[wave][lane] = best.value;
    shared_index[wave][lane] = best.index;
  }
  __syncthreads();
  if (wave != 0)
    return;
  float top = -inf;
  for (int w = 0; w < kWaves; ++w)
    top = fmaxf(top, shared[w].m);
  float s = 0.0F, t = 0.0F;
  for (int w = 0; w < kWaves; ++w) {
    Sums part = shared[w];
    part.Move(top == -inf ? part.m : top);
    s += part.s;
    t += part.t;
    if (w == 0)
      continue;
    for (int k = 0; k < p.top; ++k) {
      const float v = shared_value[w][k];
      const int i = shared_index[w][k];
      if (v == -inf || !Before(v, i, __shfl(best.value, p.top - 1),
                               __shfl(best.index, p.top - 1)))
        break;
      best.Insert(v, i, lane);
    }
  }
  // No distribution: a NaN or +infinity among the logits, or nothing above -infinity.
  const bool none = !(s > 0.0F && s < inf);
  const float log_s = logf(s);
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (p.logprob != nullptr) {
      const int token = p.tokens[row];
      const float z = token >= 0 && token < p.vocab ? Guided(c, u, token, p.guidance) : -inf;
      p.logprob[row] = none ? nan : z - top - log_s;
    }
    if (p.entropy != nullptr)
      p.entropy[row] = none ? nan : log_s - t / s;
  }
  if (lane < p.top) {
    p.top_ids[row * p.top + lane] = none ? -1 : best.index;
    p.top_logprobs[row * p.top + lane] = none ? nan : best.value - top - log_s;
  }
}

}  // namespace

void LaunchLogprobs(const LogprobParams& p, DType type, hipStream_t stream) {
  if (p.rows == 0)
    return;
  const dim3 grid(p.rows), block(kWaves * kWave);
  if (type == DType::kF16)
    Dispatch(LogprobKernel<_Float16>, grid, block, 0, stream, true, true, p);
  else if (type == DType::kBf16)
    Dispatch(LogprobKernel<__bf16>, grid, block, 0, stream, true, true, p);
  else
    Dispatch(LogprobKernel<float>, grid, block, 0, stream, true, true, p);
  Check(hipGetLastError(), "logprobs launch");
}

}  // namespace ovg
