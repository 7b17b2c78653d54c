// The draw of a token from a row of logits at a temperature, among its best.
//
//   z = c, or c + g (c - u) with unconditional logits, each step rounded to
//   float32 (c = -inf stays -inf); the order of tokens is z descending, equal ones
//   by index; w = exp((z - max z) / T)
//   top_k keeps the first k; top_p of these the shortest prefix that holds p of
//   their weight; min_p what has w >= min_p; the best stays always
//   token = the first index whose kept weights up to it pass u * (all kept)
//
// What is kept is a prefix of the order: the keys above a threshold and the first
// `need` of those equal to it. Weights are whole numbers of 2^-shift, rounded from a
// sum in 64 bits (2^x by its Taylor series, whose rest is 2^-47), so that every sum
// is exact and none depends on its order. `shift` is 62 less the vocabulary's bits,
// 51 at most: a draw can differ from the exact one where u falls within
// vocab * 2^-shift of a token's border.
#include "step.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 256;

// Keys order logits as unsigned numbers; 0 is what cannot be drawn.
__device__ __forceinline__ unsigned KeyOf(float z) {
  const unsigned bits = __float_as_uint(z + 0.0F);  // one zero
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
constexpr unsigned kKeyOfInf = 0xFF800000u;      // and NaN from here on
constexpr unsigned kKeyOfMinusInf = 0x007FFFFFu;
__device__ __forceinline__ float LogitOf(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

template <typename T>
__device__ __forceinline__ unsigned KeyAt(const SampleParams& p, int row, int i) {
  if (i == p.mask_id)
    return 0;
  float z = static_cast<float>(static_cast<const T*>(p.logits)[row * p.stride + i]);
  if (p.uncond != nullptr && z != -__builtin_inff()) {
    const float u = static_cast<float>(static_cast<const T*>(p.uncond)[row * p.uncond_stride + i]);
    z = z + p.guidance * (z - u);
  }
  if (z != z)
    return ~0u;
  const unsigned key = KeyOf(z);
  return key <= kKeyOfMinusInf ? 0 : key;
}

// The weight of a key in units of 2^-shift; per = log2(e) / T.
struct Weigher {
  double top, per;
  int shift;
  __device__ __forceinline__ double Exact(unsigned key) const {
    const double x = (static_cast<double>(LogitOf(key)) - top) * per;
    if (!(x > -64.0))
      return 0.0;
    const double n = rint(x), f = (x - n) * 0.69314718055994530942;
    double e = 1.0 / 39916800.0;
    constexpr double kTerms[] = {1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040,
                                 1.0 / 720,     1.0 / 120,    1.0 / 24,    1.0 / 6,
                                 0.5,           1.0,          1.0};
    for (double t : kTerms)
      e = __fma_rn(e, f, t);
    return ldexp(e, static_cast<int>(n));
  }
  // The sum's last bit is one unit.
  __device__ __forceinline__ u64 operator()(unsigned key) const {
    if (key == 0)
      return 0;
    const double d = Exact(key) + ldexp(1.0, 52 - shift);
    return __builtin_bit_cast(u64, d) & ((u64{1} << 52) - 1);
  }
};

template <typename V, typename F>
__device__ __forceinline__ V Join(V v, V* scratch, F&& join) {
  for (int offset = kWave / 2; offset > 0; offset /= 2)
    v = join(v, __shfl_xor(v, offset));
  __syncthreads();
  if (threadIdx.x % kWave == 0)
    scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < kThreads / kWave; ++i)
    v = join(v, scratch[i]);
  return v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void SampleKernel(SampleParams p, int shift) {
  __shared__ u64 scratch[kThreads / kWave];
  __shared__ u64 prefix[kThreads];
  const int row = blockIdx.x, tid = threadIdx.x;
  const auto sum = [&](u64 v) {
    return Join(v, scratch, [](u64 a, u64 b) { return a + b; });
  };
  const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float u = p.random[row];

  unsigned best = 0;
  for (int i = tid; i < p.vocab; i += kThreads)
    best = max(best, KeyAt<T>(p, row, i));
  best = static_cast<unsigned>(Join(static_cast<u64>(best), scratch,
                                    [](u64 a, u64 b) { return a > b ? a : b; }));
  if (best == 0 || best >= kKeyOfInf || temperature != temperature || u != u || top_p != top_p ||
      min_p != min_p) {
    if (tid == 0)
      p.tokens[row] = -1;
    return;
  }
  const bool greedy = !(temperature > 0.0F);
  const Weigher weigh{LogitOf(best), 1.4426950408889634074 / (greedy ? 1.0 : temperature), shift};
  const auto count = [&](unsigned t) {  // keys >= t
    u64 n = 0;
    for (int i = tid; i < p.vocab; i += kThreads)
      n += KeyAt<T>(p, row, i) >= t;
    return sum(n);
  };
  const auto mass = [&](unsigned t) {
    u64 n = 0;
    for (int i = tid; i < p.vocab; i += kThreads) {
      const unsigned key = KeyAt<T>(p, row, i);
      n += key >= t ? weigh(key) : 0;
    }
    return sum(n);
  };
  // The largest key t for which `reached`, which holds for all lower ones.
  const auto search = [&](auto reached) {
    unsigned low = 1, high = best;  // reached(low) is known
    while (low < high) {
      const unsigned mid = low + (high - low + 1) / 2;
      if (reached(mid))
        low = mid;
      else
        high = mid - 1;
    }
    return low;
  };
  unsigned t = 1;
  u64 need = ~u64{0}, kept;  // of the keys equal to t; the weight kept
  if (greedy) {
    t = best;
    need = 1;
  } else if (top_k > 0 && count(1) > static_cast<u64>(top_k)) {
    t = search([&](unsigned m) { return count(m) >= static_cast<u64>(top_k); });
    need = top_k - (t == best ? 0 : count(t + 1));
  }
  const auto weight = [&] {
    const u64 above = t == best ? 0 : mass(t + 1);
    return above + (need == ~u64{0} ? mass(t) - above : need * weigh(t));
  };
  kept = weight();
  if (!greedy && top_p < 1.0F) {
    const double want = ceil(static_cast<double>(fmaxf(top_p, 0.0F)) * static_cast<double>(kept));
    const u64 target = min(max(static_cast<u64>(want), u64{1}), kept);
    const u64 above_t = t == best ? 0 : mass(t + 1);
    if (above_t >= target) {
      t = search([&](unsigned m) { return m <= t || mass(m) >= target; });
      need = ~u64{0};
    }
    const u64 above = t == best ? 0 : mass(t + 1);
    const u64 each = weigh(t);
    if (each > 0)
      need = min(need, (target - above + each - 1) / each);
    kept = weight();
  }
  if (!greedy && min_p > 0.0F) {
    const double least = fmin(static_cast<double>(min_p), 1.0);
    const unsigned m = search([&](unsigned key) { return !(weigh.Exact(key - 1) >= least); });
    if (m > t) {
      t = m;
      need = ~u64{0};
      kept = weight();
    }
  }

  // Segments of the row in order, a thread each.
  u64 target = static_cast<u64>(static_cast<double>(fminf(fmaxf(u, 0.0F), 1.0F)) *
                                static_cast<double>(kept));
  target = min(target, kept - 1);
  const int each = (p.vocab + kThreads - 1) / kThreads;
  const int first = tid * each, last = min(first + each, p.vocab);
  u64 equal = 0;
  for (int i = first; i < last; ++i)
    equal += KeyAt<T>(p, row, i) == t;
  prefix[tid] = equal;
  __syncthreads();
  u64 before = 0;
  for (int i = 0; i < tid; ++i)
    before += prefix[i];
  u64 own = 0, seen = before;
  for (int i = first; i < last; ++i) {
    const unsigned key = KeyAt<T>(p, row, i);
    if (key > t || (key == t && seen++ < need))
      own += weigh(key);
  }
  __syncthreads();
  prefix[tid] = own;
  __syncthreads();
  u64 sum_before = 0;
  for (int i = 0; i < tid; ++i)
    sum_before += prefix[i];
  if (sum_before <= target && target < sum_before + own) {
    seen = before;
    for (int i = first; i < last; ++i) {
      const unsigned key = KeyAt<T>(p, row, i);
      if (key > t || (key == t && seen++ < need)) {
        sum_before += weigh(key);
        if (sum_before > target) {
          p.tokens[row] = i;
          break;
        }
      }
    }
  }
}

}  // namespace

void LaunchSample(const SampleParams& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.vocab >= 1, "sample: empty shape");
  int bits = 0;
  while ((std::int64_t{1} << bits) < p.vocab)
    ++bits;
  const int shift = 62 - bits < 51 ? 62 - bits : 51;
  WithType(type, [&](auto t) {
    Dispatch(SampleKernel<decltype(t)>, dim3(p.rows), dim3(kThreads), 0, stream, true, true, p,
             shift);
  });
  Check(hipGetLastError(), "sample launch");
}

}  // namespace ovg
