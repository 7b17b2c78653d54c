// The draw of a token from a row of logits at a temperature, among its best.
//
//   z = c, or c + g (c - u) with unconditional logits, each step rounded to
//   float32 (c = -inf stays -inf); the order of tokens is z descending, equal ones
//   by index; w = exp((z - max z) / T), none below 2^-50
//   top_k keeps the first k; top_p of these the shortest prefix that holds p of
//   their weight; min_p what has w >= min_p; the best stays always
//   token = the first index whose kept weights up to it pass u * (all kept)
//
// What is kept is a prefix of the order: the keys (logits as ordered numbers) above a
// threshold and the first `need` of those equal to it.
//
// Up to 2048 tokens a wave has its row in registers and searches thresholds by halves
// (2000 guided rows of 1025 float32, the best 50: 11 us, 16 MB). Larger vocabularies take
// two launches, or four with filters:
//   1  A wave for every chunk of 2048 tokens leaves the largest key of each quarter and,
//      where the row needs it, the chunk's weight beside its own largest.
//   2  Rows without filters: a work-group a row finds the chunk by the chunks' weights and
//      reads only that one. Rows with filters: the k best lie in the k quarters with the
//      largest keys, so a work-group a row reads those (64 for top_p alone) and lists the
//      few elements that reach the last one's, from which a wave draws. Where that will not
//      do, or may not (a large k, a share that may need more), other work-groups meanwhile
//      form the row's sums of 2048 steps of the logit.
//   3  For rows that were not drawn: the steps that hold the threshold by those sums, the
//      list of the elements in them, and the chunks' weights above them.
//   4  The threshold from the list, or from passes over the row where the list does not hold
//      it (thousands of equals, or of near ones at a high temperature), and the draw.
// Bound by the arithmetic of the weights, 16 operations in 64 bits and a table's value for
// each: 300 rows of 151936 bf16 without filters 43 us (40 + 8 with the launches overlapped;
// their 91 MB are 18 us), 64 rows with settings of all kinds 69 us (10 + 24 + 19 + 18), of
// which the bytes are 4: there the chain of short, dependent searches of launches 2 to 4 is
// what bounds.
//
// A draw lands where sums of up to 2^17 weights say, so weights have 2^-42 and better:
// 2^x in 64 bits from a table of 256 powers and three terms (ten terms without a table: 47
// us for launch 1 of the 300 rows, so 40). Sums that several lanes form in any order are
// whole numbers of 2^-shift; the others are 64-bit numbers in a fixed order. No result
// depends on the order of the work, nor on the rows beside.
#include <algorithm>

#include "step.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

typedef unsigned long long u64;
constexpr int kRun = 8;                     // elements in a row of a lane
constexpr int kQuarter = kRun * kWave;      // of a wave
constexpr int kQuarters = 4;
constexpr int kChunk = kQuarter * kQuarters;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kRowThreads = 1024;           // of a row's work-group in the second launch
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kMostQuarters = 2048;         // that are ranked
constexpr int kMostOpened = 256;            // quarters that are read for a list
constexpr int kShortList = 512;             // elements of a list that one wave holds
constexpr int kList = 2048;                 // elements of a list
// Opened for a share alone, of which the loudest quarters hold most: 512 rows of 32000 bf16
// with top_p 0.9 take 140 us, 159 with 32 and 140 with 128; a row of 151936, whose share they
// do not hold, 49, 46 and 52.
constexpr int kShareOpened = 64;
constexpr int kOctaves = 50;                // weights below 2^-50 do not count
constexpr int kTable = 256;

// ---------------------------------------------------------------- lanes
// The wave's number, which the compiler then knows to be the same in all lanes.
__device__ __forceinline__ int WaveIndex() {
  return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave));
}
template <int CTRL>
__device__ __forceinline__ u64 Dpp64(u64 v) {
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, 0xF, 0xF, false);
  return static_cast<u64>(static_cast<unsigned>(hi)) << 32 | static_cast<unsigned>(lo);
}
__device__ __forceinline__ u64 Lane64(u64 v, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<u64>(hi) << 32 | lo;
}
// Sums and maxima over a wave, the same in every lane, in a fixed order.
__device__ __forceinline__ u64 WaveSum64(u64 v) {
  v += Dpp64<0xB1>(v);
  v += Dpp64<0x4E>(v);
  v += Dpp64<0x141>(v);
  v += Dpp64<0x140>(v);
  return (Lane64(v, 0) + Lane64(v, 16)) + (Lane64(v, 32) + Lane64(v, 48));
}
__device__ __forceinline__ double WaveSum64(double v) {
  const auto bits = [](double d) { return __builtin_bit_cast(u64, d); };
  const auto number = [](u64 d) { return __builtin_bit_cast(double, d); };
  v += number(Dpp64<0xB1>(bits(v)));
  v += number(Dpp64<0x4E>(bits(v)));
  v += number(Dpp64<0x141>(bits(v)));
  v += number(Dpp64<0x140>(bits(v)));
  return (number(Lane64(bits(v), 0)) + number(Lane64(bits(v), 16))) +
         (number(Lane64(bits(v), 32)) + number(Lane64(bits(v), 48)));
}
template <typename F>
__device__ __forceinline__ unsigned WaveJoin(unsigned v, F&& join) {
  const auto step = [&](auto ctrl) {
    v = join(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(
                    static_cast<int>(v), static_cast<int>(v), ctrl(), 0xF, 0xF, false)));
  };
  step(std::integral_constant<int, 0xB1>());
  step(std::integral_constant<int, 0x4E>());
  step(std::integral_constant<int, 0x141>());
  step(std::integral_constant<int, 0x140>());
  const unsigned a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const unsigned c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return join(join(a, b), join(c, d));
}
__device__ __forceinline__ unsigned WaveMaxKey(unsigned v) {
  return WaveJoin(v, [](unsigned a, unsigned b) { return max(a, b); });
}
__device__ __forceinline__ unsigned WaveMinKey(unsigned v) {
  return WaveJoin(v, [](unsigned a, unsigned b) { return min(a, b); });
}
// The lanes' sums up to and with themselves: within rows of 16 lanes, then the rows'
// last lanes to the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned Shifted(unsigned v) {
  return static_cast<unsigned>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 Shifted(u64 v) {
  return static_cast<u64>(Shifted<CTRL, ROWS>(static_cast<unsigned>(v >> 32))) << 32 |
         Shifted<CTRL, ROWS>(static_cast<unsigned>(v));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double Shifted(double v) {
  return __builtin_bit_cast(double, Shifted<CTRL, ROWS>(__builtin_bit_cast(u64, v)));
}
template <typename V>
__device__ __forceinline__ V WaveScan(V v) {
  v += Shifted<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += Shifted<0x112, 0xF>(v);
  v += Shifted<0x114, 0xF>(v);
  v += Shifted<0x118, 0xF>(v);
  v += Shifted<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
  v += Shifted<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
  return v;
}

// ---------------------------------------------------------------- keys
// Keys order logits as unsigned numbers; 0 is what cannot be drawn.
constexpr unsigned kKeyOfInf = 0xFF800000u;  // and NaN from here on
constexpr unsigned kKeyOfMinusInf = 0x007FFFFFu;
__device__ __forceinline__ unsigned KeyOf(float z) {
  const unsigned bits = __float_as_uint(z + 0.0F);  // one zero
  unsigned key = bits ^ (static_cast<unsigned>(static_cast<int>(bits) >> 31) | 0x80000000u);
  key = key > kKeyOfMinusInf ? key : 0;
  return z == z ? key : ~0u;
}
__device__ __forceinline__ float LogitOf(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// A lane's run of eight logits of quarter q. The row's last run is moved to its end, so
// that no load is conditional: RunStart is its first element. What the run before has,
// what is behind the row and the masked token are -infinity.
__device__ __forceinline__ int RunStart(int q, int vocab) {
  const int d = (q * kWave + static_cast<int>(threadIdx.x % kWave)) * kRun;
  return vocab >= kRun ? min(d, vocab - kRun) : 0;
}
template <typename T>
__device__ __forceinline__ void LoadRun(const T* row, int start, int vocab, float (&v)[kRun]) {
  if (vocab >= kRun) {
    LoadFloats<kRun>(row + start, v);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      v[i] = i < vocab ? static_cast<float>(row[i]) : 0.0F;
  }
}
template <typename T>
__device__ __forceinline__ void LoadLogits(const SampleParams& p, std::int64_t row, int q,
                                           float (&z)[kRun]) {
  const int start = RunStart(q, p.vocab);
  LoadRun(static_cast<const T*>(p.logits) + row * p.stride, start, p.vocab, z);
  if (p.uncond != nullptr) {
    float u[kRun];
    LoadRun(static_cast<const T*>(p.uncond) + row * p.uncond_stride, start, p.vocab, u);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const float guided = z[i] + p.guidance * (z[i] - u[i]);
      z[i] = z[i] == -__builtin_inff() ? z[i] : guided;
    }
  }
  const int first = q * kQuarter;
  if (first + kQuarter > p.vocab || (p.mask_id >= first && p.mask_id < first + kQuarter)) {
    const int d = first + static_cast<int>(threadIdx.x % kWave) * kRun;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int e = start + i;
      const bool in = (e >= d) & (e < p.vocab) & (e != p.mask_id);
      z[i] = in ? z[i] : -__builtin_inff();
    }
  }
}
// One that is not masked.
template <typename T>
__device__ __forceinline__ float LogitAt(const SampleParams& p, std::int64_t row, int token) {
  const float z = static_cast<float>(static_cast<const T*>(p.logits)[row * p.stride + token]);
  if (p.uncond == nullptr)
    return z;
  const float u =
      static_cast<float>(static_cast<const T*>(p.uncond)[row * p.uncond_stride + token]);
  return z == -__builtin_inff() ? z : z + p.guidance * (z - u);
}
// ---------------------------------------------------------------- weights
// 2^(j / 256), by the series of e^x.
struct Powers {
  double v[kTable];
};
constexpr Powers PowersOfTwo() {
  Powers t{};
  for (int j = 0; j < kTable; ++j) {
    const double x = j * (0.69314718055994530942 / kTable);
    double e = 1.0;
    for (int n = 18; n > 0; --n)
      e = 1.0 + e * x / n;
    t.v[j] = e;
  }
  return t;
}
__device__ const Powers kPowers = PowersOfTwo();
__device__ __forceinline__ void FillTable(double* powers) {
  for (int j = threadIdx.x; j < kTable; j += blockDim.x)
    powers[j] = kPowers.v[j];
}

struct Weigher {
  const double* powers;  // in LDS
  double top, per;       // the largest logit; 256 log2(e) / T
  // 2^((z - top) per / 256): the table's power times three terms of the rest,
  // which is under ln 2 / 512, so that 1.4e-13 is left out.
  __device__ __forceinline__ double Raw(float z) const {
    constexpr double kA = 0.69314718055994530942 / kTable;
    const double t = fmax((static_cast<double>(z) - top) * per, -1e9);  // also of -infinity
    const double whole = __builtin_rint(t);
    const double r = t - whole;
    const int k = static_cast<int>(whole);
    double e = __fma_rn(r, kA * kA * kA / 6, kA * kA / 2);
    e = __fma_rn(r, e, kA);
    e = __fma_rn(r, e, 1.0);
    return ldexp(e * powers[k & (kTable - 1)], k >> 8);
  }
  // None where it is below 2^-50.
  __device__ __forceinline__ double Of(float z) const {
    const double w = Raw(z);
    return w >= 0x1p-50 ? w : 0.0;
  }
  __device__ __forceinline__ double operator()(unsigned key) const {
    return key != 0 ? Of(LogitOf(key)) : 0.0;
  }
};
// In whole units of 2^-shift, shift <= 51: the last bits of a sum with 2^(52 - shift).
__device__ __forceinline__ u64 UnitsOf(double w, int shift) {
  const double d = w + __builtin_bit_cast(double, static_cast<u64>(1023 + 52 - shift) << 52);
  return __builtin_bit_cast(u64, d) & ((u64{1} << 52) - 1);
}

struct Settings {
  float temperature, top_p, min_p, u;
  int top_k;  // 0: all
  bool lost, greedy;
  __device__ __forceinline__ bool Whole() const { return !greedy && top_k == 0; }
};
__device__ __forceinline__ Settings SettingsOf(const SampleParams& p, int row) {
  Settings s;
  s.temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  s.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  s.min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  s.top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  s.u = p.random[row];
  s.lost = s.temperature != s.temperature || s.u != s.u || s.top_p != s.top_p ||
           s.min_p != s.min_p;
  s.greedy = !(s.temperature > 0.0F);
  s.top_k = s.top_k <= 0 || s.top_k >= p.vocab ? 0 : s.top_k;
  return s;
}
__device__ __forceinline__ Weigher WeigherOf(const double* powers, unsigned best, float t) {
  return {powers, static_cast<double>(LogitOf(best)), kTable * 1.4426950408889634074 / t};
}

// The smallest key, up to best, that weighs `least` of the best: 64 keys at once.
__device__ __forceinline__ unsigned KeyOfShare(const Weigher& w, unsigned best, float least) {
  const double share = fmin(static_cast<double>(least), 1.0);
  unsigned low = 0, high = best;  // low is below, high is not
  const int lane = threadIdx.x % kWave;
  while (high - low > 1) {
    const unsigned step = (high - low + kWave - 1) / kWave;
    const unsigned key = min(low + step * (lane + 1), high);
    const u64 reached = __ballot(w(key) >= share || key == high);
    const int first = __builtin_ctzll(reached);
    high = min(low + step * (first + 1), high);
    low = low + step * first;
  }
  return high;
}

// u's place among `all`, which is at least 1.
__device__ __forceinline__ u64 TargetOf(float u, u64 all) {
  const double at = static_cast<double>(fminf(fmaxf(u, 0.0F), 1.0F)) * static_cast<double>(all);
  return min(static_cast<u64>(at), all - 1);
}
// The weight that holds the share p of `all`.
__device__ __forceinline__ u64 ShareOf(float p, u64 all) {
  const double want = ceil(static_cast<double>(fmaxf(p, 0.0F)) * static_cast<double>(all));
  return min(max(static_cast<u64>(want), u64{1}), all);
}

// What is kept of a row: keys above t and the first `need` of those equal to t.
struct Kept {
  unsigned t;
  u64 need;
  u64 weight;  // in units
};
constexpr u64 kAll = ~u64{0};

// N elements a lane.
template <int N>
struct Held {
  unsigned key[N];
  u64 weight[N];
  __device__ __forceinline__ int Count(unsigned t) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n += __popcll(__ballot(key[i] >= t));
    }
    return n;
  }
  __device__ __forceinline__ u64 Weight(unsigned t) const {
    u64 n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n += key[i] >= t ? weight[i] : 0;
    }
    return WaveSum64(n);
  }
  __device__ __forceinline__ unsigned Least() const {  // 1 or more
    unsigned n = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n = key[i] != 0 ? min(n, key[i]) : n;
    }
    return WaveMinKey(n);
  }
  // The largest key in [low, high] for which `reached`, which low is.
  template <typename F>
  static __device__ __forceinline__ unsigned Search(unsigned low, unsigned high, F&& reached) {
    while (low < high) {
      const unsigned mid = low + (high - low + 1) / 2;
      if (reached(mid))
        low = mid;
      else
        high = mid - 1;
    }
    return low;
  }
  // top_p's share is of `whole`, or of what top_k keeps.
  __device__ __forceinline__ Kept Select(const Settings& s, const Weigher& w, unsigned best,
                                         int shift, u64 whole = 0) const {
    const unsigned least = Least();
    Kept kept{least, kAll, Weight(1)};
    if (s.top_k > 0 && Count(1) > s.top_k) {
      kept.t = Search(least, best, [&](unsigned t) { return Count(t) >= s.top_k; });
      const unsigned above = kept.t + 1;
      kept.need = s.top_k - Count(above);
      kept.weight = Weight(above) + kept.need * UnitsOf(w(kept.t), shift);
    }
    if (s.top_p < 1.0F) {
      const u64 want = ShareOf(s.top_p, whole != 0 ? whole : kept.weight);
      const unsigned low = kept.t;
      u64 above = Weight(low + 1);
      if (above >= want) {
        kept.t = Search(low + 1, best, [&](unsigned t) { return Weight(t) >= want; });
        kept.need = kAll;
        above = Weight(kept.t + 1);
      }
      const u64 each = UnitsOf(w(kept.t), shift);
      if (each > 0) {
        kept.need = min(kept.need, (want - above + each - 1) / each);
        kept.need = min(kept.need, static_cast<u64>(Count(kept.t) - Count(kept.t + 1)));
        kept.weight = above + kept.need * each;
      }
    }
    if (s.min_p > 0.0F) {
      const unsigned t = KeyOfShare(w, best, s.min_p);
      if (t > kept.t) {
        kept.t = t;
        kept.need = kAll;
        kept.weight = Weight(t);
      }
    }
    return kept;
  }
};

// Of R elements a lane in the row's order, lane by lane: whether the kept weights pass
// `left` here, and then which element of which lane. `need` and `left` go on to what
// follows.
template <int R>
__device__ __forceinline__ bool DrawOf(const unsigned (&key)[R], const u64 (&weight)[R],
                                       unsigned t, u64* need, u64* left, int* lane, int* place) {
  unsigned equal = 0;
#pragma unroll
  for (int i = 0; i < R; ++i)
    equal += key[i] == t;
  // Most runs have no equal: their scan is left out.
  const bool equals = __ballot(equal != 0) != 0;
  const unsigned equal_to = equals ? WaveScan(equal) : 0;
  u64 seen = equal_to - equal, mine = 0;
  u64 to_place[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    mine += key[i] > t || (key[i] == t && seen++ < *need) ? weight[i] : 0;
    to_place[i] = mine;
  }
  const u64 to = WaveScan(mine);
  const u64 hit = __ballot(to > *left);
  if (hit == 0) {
    *left -= Lane64(to, kWave - 1);
    *need -= min(*need, static_cast<u64>(__builtin_amdgcn_readlane(equal_to, kWave - 1)));
    return false;
  }
  *lane = __builtin_ctzll(hit);
  int at = R - 1;
#pragma unroll
  for (int i = R - 2; i >= 0; --i)
    at = to - mine + to_place[i] > *left ? i : at;
  *place = __builtin_amdgcn_readlane(at, *lane);
  return true;
}

// ---------------------------------------------------------------- small rows
// A wave a row of up to 512 Q tokens. With a top_k of 128 or less, the largest keys of the
// lanes' halves give a floor that the k best reach, and the few elements that do go
// through LDS, in the row's order, to two or four a lane.
constexpr int kFew = 4 * kWave;

// The draw from `listed` elements in the row's order, R a lane; top_p's share is of `whole`,
// or of what top_k keeps. False where the list does not hold the share.
template <int R>
__device__ __forceinline__ bool DrawFew(const SampleParams& p, int row, const u64* few,
                                        int listed, const Settings& s, const Weigher& w,
                                        unsigned best, int shift, u64 whole = 0) {
  const int lane = threadIdx.x % kWave;
  Held<R> held;
  int index[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const u64 e = R * lane + i < listed ? few[R * lane + i] : 0;
    held.key[i] = static_cast<unsigned>(e >> 32);
    index[i] = static_cast<int>(e);
    held.weight[i] = UnitsOf(w(held.key[i]), shift);
  }
  if (whole != 0 && held.Weight(1) < ShareOf(s.top_p, whole))
    return false;
  const Kept kept = held.Select(s, w, best, shift, whole);
  u64 left = TargetOf(s.u, kept.weight), need = kept.need;
  int of, place;
  if (DrawOf(held.key, held.weight, kept.t, &need, &left, &of, &place)) {
    int token = index[0];
#pragma unroll
    for (int i = 1; i < R; ++i)
      token = place == i ? index[i] : token;
    if (lane == of)
      p.tokens[row] = token;
  }
  return true;
}

template <typename T, int Q>
__global__ __launch_bounds__(kThreads) void SmallKernel(SampleParams p, int shift) {
  constexpr int N = Q * kRun;
  __shared__ double powers[kTable];
  __shared__ u64 few[kWaves][kFew];  // key, index
  FillTable(powers);
  const int lane = threadIdx.x % kWave, wave = WaveIndex();
  const int row = blockIdx.x * kWaves + wave;
  Held<N> held;
  Settings s{};
  if (row < p.rows) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float z[kRun];
      LoadLogits<T>(p, row, q, z);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        held.key[q * kRun + i] = KeyOf(z[i]);
    }
  }
  __syncthreads();
  if (row >= p.rows)
    return;
  unsigned most[2] = {0, 0};  // of the lane's halves
#pragma unroll
  for (int i = 0; i < N; ++i)
    most[i < N / 2] = max(most[i < N / 2], held.key[i]);
  const unsigned best = WaveMaxKey(max(most[0], most[1]));
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (lane == 0)
      p.tokens[row] = -1;
    return;
  }
  const Weigher w = WeigherOf(powers, best, s.greedy ? 1.0F : s.temperature);
  Kept kept{best, 1, 1};
  u64 left, need;
  int of, place;
  if (!s.greedy && s.top_k > 0 && s.top_k <= 2 * kWave) {
    unsigned floor = 1, high = best;
    while (floor < high) {
      const unsigned mid = floor + (high - floor + 1) / 2;
      if (__popcll(__ballot(most[0] >= mid)) + __popcll(__ballot(most[1] >= mid)) >= s.top_k)
        floor = mid;
      else
        high = mid - 1;
    }
    unsigned from[Q];  // where the lane's elements go
    int listed = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      unsigned n = 0;
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        n += held.key[q * kRun + i] >= floor;
      const unsigned to = WaveScan(n);
      from[q] = listed + to - n;
      listed += __builtin_amdgcn_readlane(to, kWave - 1);
    }
    if (listed <= kFew) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int start = RunStart(q, p.vocab);
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          if (held.key[q * kRun + i] >= floor)
            few[wave][from[q]++] = static_cast<u64>(held.key[q * kRun + i]) << 32 |
                                   static_cast<unsigned>(start + i);
      }
      // The wave's own part of LDS: its writes are done before its reads.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (listed <= kFew / 2)
        DrawFew<2>(p, row, few[wave], listed, s, w, best, shift);
      else
        DrawFew<4>(p, row, few[wave], listed, s, w, best, shift);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    held.weight[i] = s.greedy ? held.key[i] == best : UnitsOf(w(held.key[i]), shift);
  if (!s.greedy)
    kept = held.Select(s, w, best, shift);
  left = TargetOf(s.greedy ? 0.0F : s.u, kept.weight);
  need = kept.need;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    unsigned run_key[kRun];
    u64 run_weight[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      run_key[i] = held.key[q * kRun + i];
      run_weight[i] = held.weight[q * kRun + i];
    }
    if (DrawOf(run_key, run_weight, kept.t, &need, &left, &of, &place)) {
      if (lane == of)
        p.tokens[row] = RunStart(q, p.vocab) + place;
      return;
    }
  }
}

// ---------------------------------------------------------------- large rows
// A row's part of the workspace: the chunks' weights, the quarters' largest keys.
struct Work {
  double* weight;
  unsigned* most;
};
// What a row that needs its threshold goes on with, and its sums.
struct RowState {
  enum : unsigned { kDone, kCollect, kKnown, kSlow };
  unsigned status, best;
  unsigned t;       // kKnown: all from it on is kept
  unsigned raised;  // where min_p's key is above the steps below: all from it on is kept
  unsigned listed;  // elements of the list
  u64 whole;        // the row's weight in units, without a top_k
  // The steps whose elements are listed: the one in which top_k ends, and low .. high, in
  // which the share does; what is above them.
  int k_step, low_step, high_step;
  u64 k_count, k_weight, low_count, low_weight;
  unsigned counts[kList];
  u64 weights[kList];
  u64 list[kList];  // key, index
};
// Rows that have a state at once: 41 KB each, so that the workspace of 4096 rows is 28 MB and
// not 175; 1024 rows take launches 2 to 4 twice.
constexpr int kBatch = 512;

struct RowCall {
  SampleParams p;
  int first, rows;  // of the launch
  int chunks, quarters, shift;
};
__host__ __device__ constexpr std::int64_t WorkWords(std::int64_t chunks) {
  return (chunks * (2 + kQuarters) + 3) / 4 * 4;
}
__device__ __forceinline__ Work WorkOf(const SampleParams& p, int row, int chunks) {
  double* const base = reinterpret_cast<double*>(p.work + WorkWords(chunks) * row);
  return {base, reinterpret_cast<unsigned*>(base + chunks)};
}
__device__ __forceinline__ RowState* StateOf(const RowCall& c, int i) {
  return reinterpret_cast<RowState*>(c.p.work + WorkWords(c.chunks) * c.p.rows) + i;
}

// A wave's four quarters of a chunk, all loads on their way at once; then f(first element
// of the lane's run, logits) for one after the other, in a loop that stays one.
template <typename T, typename F>
__device__ __forceinline__ void EachQuarter(const SampleParams& p, int row, int chunk, F&& f) {
  float z[kQuarters][kRun];
#pragma unroll
  for (int q = 0; q < kQuarters; ++q)
    LoadLogits<T>(p, row, chunk * kQuarters + q, z[q]);
#pragma unroll 1
  for (int q = 0; q < kQuarters; ++q) {
    float v[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const float front = q == 0 ? z[0][i] : z[1][i], back = q == 2 ? z[2][i] : z[3][i];
      v[i] = q < 2 ? front : back;
    }
    f(RunStart(chunk * kQuarters + q, p.vocab), v);
  }
}

// Clears what the launches behind add to; `part` of `parts` work-groups.
__device__ __forceinline__ void ClearState(RowState* state, int part, int parts) {
  for (int i = part * kThreads + threadIdx.x; i < kList; i += parts * kThreads) {
    state->counts[i] = 0;
    state->weights[i] = 0;
  }
  if (part == 0 && threadIdx.x == 0) {
    state->status = RowState::kDone;
    state->listed = 0;
    state->raised = 0;
  }
}
__global__ __launch_bounds__(kThreads) void ClearKernel(RowCall c) {
  ClearState(StateOf(c, blockIdx.x), 0, 1);
}

// The largest key of every quarter of a chunk, and the chunk's weight beside the
// chunk's own largest.
template <typename T>
__global__ __launch_bounds__(kThreads) void ChunkKernel(RowCall c, int groups, bool clear) {
  __shared__ double powers[kTable];
  const SampleParams& p = c.p;
  const int chunks = c.chunks;
  __builtin_assume(p.vocab > kChunk);
  FillTable(powers);
  const int lane = threadIdx.x % kWave;
  const int row = blockIdx.x / groups;
  const int chunk = (blockIdx.x - row * groups) * kWaves + WaveIndex();
  float z[kQuarters][kRun];
  Settings s{};
  if (chunk < chunks) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
      LoadLogits<T>(p, row, chunk * kQuarters + q, z[q]);
  }
  if (clear)
    ClearState(StateOf(c, row), blockIdx.x - row * groups, groups);
  __syncthreads();
  if (chunk >= chunks)
    return;
  const Work work = WorkOf(p, row, chunks);
  float best = -__builtin_inff();
  bool lost = false;
#pragma unroll
  for (int q = 0; q < kQuarters; ++q) {
    float most = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      most = fmaxf(most, z[q][i]);
      lost |= __builtin_amdgcn_classf(z[q][i], 0x203);  // a NaN or +infinity
    }
    most = WaveMaxFast(most);
    best = fmaxf(best, most);
    if (lane == 0)
      work.most[chunk * kQuarters + q] = KeyOf(most);
  }
  if (__ballot(lost) != 0) {
    if (lane == 0)
      work.most[chunk * kQuarters] = ~0u;
    return;
  }
  if (!s.Whole())
    return;
  double sum[2] = {0.0, 0.0};
  if (best != -__builtin_inff()) {
    const Weigher w{powers, best, kTable * 1.4426950408889634074 / s.temperature};
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        sum[i & 1] += w.Raw(z[q][i]);
  }
  const double all = WaveSum64(sum[0] + sum[1]);
  if (lane == 0)
    work.weight[chunk] = all;
}

// v is the same in every lane of a wave.
template <int WAVES, typename V, typename F>
__device__ __forceinline__ V RowJoin(V v, u64* scratch, F&& join) {
  V* const slots = reinterpret_cast<V*>(scratch);
  __syncthreads();
  if (threadIdx.x % kWave == 0)
    slots[threadIdx.x / kWave] = v;
  __syncthreads();
  v = slots[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i)
    v = join(v, slots[i]);
  return v;
}
template <int WAVES, typename V>
__device__ __forceinline__ V RowSum(V v, u64* scratch) {
  return RowJoin<WAVES>(WaveSum64(v), scratch, [](V a, V b) { return a + b; });
}

// The largest key of the row; also in sh_most, where the quarters fit.
template <int WAVES>
__device__ __forceinline__ unsigned BestOf(const Work& work, int quarters, unsigned* sh_most,
                                           u64* slots) {
  unsigned best = 0;
  for (int i = threadIdx.x; i < quarters; i += WAVES * kWave) {
    const unsigned m = work.most[i];
    if (i < kMostQuarters)
      sh_most[i] = m;
    best = max(best, m);
  }
  return RowJoin<WAVES>(WaveMaxKey(best), slots, [](unsigned a, unsigned b) { return max(a, b); });
}

// The first token of the largest key.
template <typename T, int WAVES>
__device__ __forceinline__ void DrawBest(const RowCall& c, int row, const Work& work, unsigned best,
                                         u64* slots) {
  unsigned first = ~0u;
  for (int i = threadIdx.x; i < c.quarters && first == ~0u; i += WAVES * kWave)
    if (work.most[i] == best)
      first = i;
  first = RowJoin<WAVES>(WaveMinKey(first), slots,
                         [](unsigned a, unsigned b) { return min(a, b); });
  if (threadIdx.x >= kWave)
    return;
  float z[kRun];
  LoadLogits<T>(c.p, row, static_cast<int>(first), z);
  unsigned token = ~0u;
#pragma unroll
  for (int i = kRun - 1; i >= 0; --i)
    token = KeyOf(z[i]) == best ? RunStart(static_cast<int>(first), c.p.vocab) + i : token;
  token = WaveMinKey(token);
  if (threadIdx.x == 0)
    c.p.tokens[row] = static_cast<int>(token);
}

// The chunks' weights beside the row's best, and their sum.
template <int WAVES>
__device__ __forceinline__ double WholeOf(const RowCall& c, const Work& work, const Weigher& w,
                                          u64* slots) {
  double all = 0.0;
  for (int i = threadIdx.x; i < c.chunks; i += WAVES * kWave) {
    unsigned top = 0;
    for (int q = i * kQuarters; q < min((i + 1) * kQuarters, c.quarters); ++q)
      top = max(top, work.most[q]);
    const double sum = work.weight[i] * w(top);
    work.weight[i] = sum;
    all += sum;
  }
  return RowSum<WAVES>(all, slots);
}

struct PickShared {
  unsigned equal[kQuarters];
  int hit[kQuarters], token[kQuarters];
  double total[kQuarters];
};
// The draw by the chunks' kept weights: the chunk, 64 at a time, then the place in it. The
// whole work-group calls this, behind a barrier; four waves of it work. Kept is what is
// above t (0: all) and of what equals it the first `need`, which `equals` counts by chunk
// (null: none).
template <typename T>
__device__ __forceinline__ void Pick(const RowCall& c, int row, const double* weights,
                                     const unsigned* equals, const Settings& s, const Weigher& w,
                                     unsigned t, u64 need0, PickShared& sh) {
  const SampleParams& p = c.p;
  const int lane = threadIdx.x % kWave, wave = WaveIndex();
  const bool mine = wave < kQuarters;
  const bool bounded = t != 0;
  const double each = bounded ? w(t) : 0.0;
  const auto last_lane = [](double v) {
    return __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, v), kWave - 1));
  };
  // Twice over the chunks: their sum, then the place.
  double total = 0.0, left = __builtin_inf(), last_before = 0.0;
  int last = 0;  // the chunk; the last one that keeps any where rounding leaves none
  u64 last_need = 0;
#pragma unroll 1
  for (int turn = mine ? 0 : 2; turn < 2; ++turn) {
    u64 need = need0;
    double before = 0.0;
    bool done = false;
#pragma unroll 1
    for (int c0 = 0; c0 < c.chunks && !done; c0 += kWave) {
      const bool there = c0 + lane < c.chunks;
      const unsigned equal = there && equals != nullptr ? equals[c0 + lane] : 0;
      const u64 equal_to = equals != nullptr ? WaveScan(static_cast<u64>(equal)) : 0;
      const u64 equal_before = equal_to - equal;
      const u64 in = need > equal_before ? min(need - equal_before, static_cast<u64>(equal)) : 0;
      const double kept = (there ? weights[c0 + lane] : 0.0) + static_cast<double>(in) * each;
      const double to = before + WaveScan(kept);
      const u64 hit = __ballot(kept > 0.0 && to > left), any = __ballot(kept > 0.0);
      if (any != 0) {
        const int l = hit != 0 ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
        last = c0 + l;
        last_before = __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, to - kept), l));
        last_need = need - min(need, Lane64(equal_before, l));
      }
      done = hit != 0;
      before = last_lane(to);
      need -= min(need, Lane64(equal_to, kWave - 1));
    }
    if (turn == 0) {
      total = before;
      left = static_cast<double>(fminf(fmaxf(s.u, 0.0F), 1.0F)) * total;
      if (!(left < total))
        left = total * (1.0 - 0x1p-53);
    }
  }
  left -= last_before;
  // A wave a quarter: the equals, then the kept weights before it, then the place.
  const int q = last * kQuarters + wave;
  float z[kRun];
  unsigned equal = 0, equal_to = 0;
  if (mine) {
    LoadLogits<T>(p, row, q, z);
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      equal += bounded && KeyOf(z[i]) == t;
    equal_to = WaveScan(equal);
    if (lane == kWave - 1)
      sh.equal[wave] = equal_to;
  }
  __syncthreads();
  u64 need = last_need;
  double to_place[kRun], weight_of = 0.0, to = 0.0;
  int end = -1;  // the lane's last kept one
  if (mine) {
    for (int i = 0; i < wave; ++i)
      need -= min(need, static_cast<u64>(sh.equal[i]));
    u64 seen = equal_to - equal;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const unsigned key = KeyOf(z[i]);
      const bool in = !bounded || key > t || (key == t && seen++ < need);
      const double weight = in ? w(key) : 0.0;
      end = weight > 0.0 ? i : end;
      weight_of += weight;
      to_place[i] = weight_of;
    }
    to = WaveScan(weight_of);
    if (lane == kWave - 1)
      sh.total[wave] = to;
  }
  __syncthreads();
  if (mine) {
    for (int i = 0; i < wave; ++i)
      left -= sh.total[i];
    const u64 hit = __ballot(weight_of > 0.0 && to > left), any = __ballot(weight_of > 0.0);
    int place = end;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const double before = i > 0 ? to_place[i - 1] : 0.0;
      place = to_place[i] > before && (to - weight_of) + to_place[i] > left ? i : place;
    }
    const int token = RunStart(q, p.vocab) + place;
    if (lane == 0)
      sh.hit[wave] = hit != 0;
    const int of = hit != 0 ? __builtin_ctzll(hit) : any != 0 ? 63 - __builtin_clzll(any) : 0;
    if (lane == of)
      sh.token[wave] = any != 0 ? token : -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int token = -1;  // the last kept one, where rounding leaves none
    for (int i = 0; i < kQuarters; ++i) {
      token = sh.token[i] >= 0 ? sh.token[i] : token;
      if (sh.hit[i])
        break;
    }
    p.tokens[row] = token;
  }
}

// Rows of which none has a filter, or that are decided by the chunks' numbers.
template <typename T>
__global__ __launch_bounds__(kThreads) void PlainKernel(RowCall c) {
  __shared__ double powers[kTable];
  __shared__ unsigned most[kMostQuarters];
  __shared__ u64 slots[kWaves];
  __shared__ PickShared pick;
  const int row = c.first + blockIdx.x;
  const Settings s = SettingsOf(c.p, row);
  const Work work = WorkOf(c.p, row, c.chunks);
  FillTable(powers);
  const unsigned best = BestOf<kWaves>(work, c.quarters, most, slots);
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (threadIdx.x == 0)
      c.p.tokens[row] = -1;
    return;
  }
  if (s.greedy) {
    DrawBest<T, kWaves>(c, row, work, best, slots);
    return;
  }
  const Weigher w = WeigherOf(powers, best, s.temperature);
  WholeOf<kWaves>(c, work, w, slots);
  __syncthreads();
  Pick<T>(c, row, work.weight, nullptr, s, w, 0, 0, pick);
}

// ---------------------------------------------------------------- rows with filters
struct RowShared {
  double powers[kTable];
  u64 weights[kList];   // of bins; as 64-bit numbers, the chunks'
  unsigned counts[kList];
  u64 list[kList];      // key, index
  unsigned most[kMostQuarters];
  unsigned short open[kMostQuarters];
  u64 slots[kRowWaves], count_slots[kRowWaves];
  PickShared pick;
  int bin;
  unsigned floor;
  u64 above_weight, above_count;
};

// 2048 equal steps of the logit from the best down to the smallest weight that counts.
struct Steps {
  float top, scale;
  // kList where the element is none of them.
  __device__ __forceinline__ int operator()(float z) const {
    const float at = fminf(top - z, 3e38F) * scale;
    return at < static_cast<float>(kList) && z > -__builtin_inff() ? static_cast<int>(at) : kList;
  }
};
__device__ __forceinline__ Steps StepsOf(const Weigher& w) {
  return {static_cast<float>(w.top),
          fminf(static_cast<float>(w.per * (static_cast<double>(kList) / (kOctaves * kTable))),
                1e30F)};
}

// The bin (0 is the top one) in which the sums of sh.counts, or of sh.weights, reach
// `want` from what is above them; sh.bin, and what is above it in sh.above_count and
// sh.above_weight. Two bins a thread; the whole work-group calls this.
__device__ __forceinline__ void FindBin(RowShared& sh, bool by_weight, u64 want, u64 above_count,
                                        u64 above_weight) {
  static_assert(kList == 2 * kRowThreads, "two bins a thread");
  const int tid = threadIdx.x, wave = WaveIndex();
  __syncthreads();
  const u64 w0 = sh.weights[2 * tid], w1 = sh.weights[2 * tid + 1];
  const unsigned c0 = sh.counts[2 * tid], c1 = sh.counts[2 * tid + 1];
  u64 weight_to = WaveScan(w0 + w1), count_to = WaveScan(c0 + c1);
  if (tid % kWave == kWave - 1) {
    sh.slots[wave] = weight_to;
    sh.count_slots[wave] = count_to;
  }
  __syncthreads();
  weight_to += above_weight;
  count_to += above_count;
  for (int i = 0; i < wave; ++i) {
    weight_to += sh.slots[i];
    count_to += sh.count_slots[i];
  }
  const u64 weight = weight_to - w0 - w1, count = count_to - c0 - c1;
  const u64 to = by_weight ? weight_to : count_to, from = by_weight ? weight : count;
  // The last bin stands for sums that do not reach it.
  if ((to >= want && (from < want || tid == 0)) || (tid == kRowThreads - 1 && to < want)) {
    const bool second = (by_weight ? weight + w0 : count + c0) < want;
    sh.bin = 2 * tid + second;
    sh.above_weight = weight + (second ? w0 : 0);
    sh.above_count = count + (second ? c0 : 0);
  }
  __syncthreads();
}

// The largest key, up to best, that `opened` of the quarters' largest reach (1: fewer do),
// by halves. The first wave searches, which has 512 of them in registers; the whole
// work-group calls this.
__device__ __forceinline__ unsigned ReachedBy(RowShared& sh, int quarters, int opened,
                                              unsigned best) {
  const int lane = threadIdx.x % kWave;
  if (threadIdx.x < kWave) {
    constexpr int kHeld = 8;
    unsigned held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      held[i] = i * kWave + lane < quarters ? sh.most[i * kWave + lane] : 0;
    unsigned low = 1, high = best;
#pragma unroll 1
    while (low < high) {
      const unsigned mid = low + (high - low + 1) / 2;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        n += __popcll(__ballot(held[i] >= mid));
      for (int i = kHeld * kWave; i < quarters; i += kWave)
        n += __popcll(__ballot(i + lane < quarters && sh.most[i + lane] >= mid));
      if (n >= opened)
        low = mid;
      else
        high = mid - 1;
    }
    if (lane == 0)
      sh.floor = low;
  }
  __syncthreads();
  return sh.floor;
}

// The list of the row's keys from `floor` on in the row's order; the number of them, or
// kShortList + 1 where it does not hold them. The whole work-group calls this.
template <typename T>
__device__ __forceinline__ int Gather(const RowCall& c, int row, RowShared& sh, unsigned floor) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = WaveIndex();
  const float from = LogitOf(max(floor, kKeyOfMinusInf + 1));
  // A sum over the waves before this one, and over all.
  const auto before_wave = [&](int n, int* all) {
    if (lane == 0)
      sh.count_slots[wave] = n;
    __syncthreads();
    int before = 0;
    *all = 0;
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) {
      const int m = static_cast<int>(sh.count_slots[i]);
      before += i < wave ? m : 0;
      *all += m;
    }
    __syncthreads();
    return before;
  };
  int opened = 0;  // quarters that have any
  for (int q0 = 0; q0 < c.quarters; q0 += kRowThreads) {
    const bool open = q0 + tid < c.quarters && sh.most[q0 + tid] >= floor;
    const u64 lanes = __ballot(open);
    int all;
    const int at = opened + before_wave(__popcll(lanes), &all);
    if (open)
      sh.open[at + __popcll(lanes & ((u64{1} << lane) - 1))] =
          static_cast<unsigned short>(q0 + tid);
    opened += all;
  }
  if (opened > kShortList)
    return kShortList + 1;
  __syncthreads();
  constexpr int kAtOnce = 4;  // quarters' loads of a wave
  int listed = 0;
#pragma unroll 1
  for (int o = 0; o < opened; o += kAtOnce * kRowWaves) {
    const int each = min((opened - o + kRowWaves - 1) / kRowWaves, kAtOnce);
    const int first = o + wave * each, count = min(each, opened - first);
    float z[kAtOnce][kRun];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (i < count)
        LoadLogits<T>(c.p, row, sh.open[first + i], z[i]);
    unsigned in = 0;  // a bit an element
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (i < count)
#pragma unroll
        for (int e = 0; e < kRun; ++e)
          in |= z[i][e] >= from ? 1u << (i * kRun + e) : 0;
    int all;
    int at = listed + before_wave(static_cast<int>(WaveSum64(static_cast<u64>(__popc(in)))), &all);
    listed += all;
    if (listed > kShortList)
      return kShortList + 1;
    // The few elements' logits come from memory again: a loop instead of a store for each.
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      unsigned mine = in >> (i * kRun) & ((1u << kRun) - 1);
      const unsigned n = __popc(mine), scan = WaveScan(n);
      const int start = RunStart(sh.open[first + i], c.p.vocab);
      for (int to = at + static_cast<int>(scan - n); mine != 0; ++to, mine &= mine - 1) {
        const int token = start + __builtin_ctz(mine);
        sh.list[to] = static_cast<u64>(KeyOf(LogitAt<T>(c.p, row, token))) << 32 |
                      static_cast<unsigned>(token);
      }
      at += __builtin_amdgcn_readlane(scan, kWave - 1);
    }
  }
  __syncthreads();
  return listed;
}

// What is to be done of a batch by work-groups that take items of it in turn: of the rows
// in sh.open, parts of 16 waves with `per` quarters each, as few as leave each work-group
// one item, else whole chunks.
struct Items {
  int count, parts, per;
};
template <typename F>
__device__ __forceinline__ Items ItemsOf(const RowCall& c, RowShared& sh, int groups, F&& in) {
  static_assert(kBatch <= kRowThreads, "a thread a row");
  const int tid = threadIdx.x, wave = WaveIndex();
  const bool mine = tid < c.rows && in(tid);
  const u64 lanes = __ballot(mine);
  if (tid % kWave == 0)
    sh.slots[wave] = lanes;
  __syncthreads();
  int before = 0, rows = 0;
  for (int i = 0; i < kRowWaves; ++i) {
    const int n = __popcll(sh.slots[i]);
    before += i < wave ? n : 0;
    rows += n;
  }
  if (mine)
    sh.open[before + __popcll(lanes & ((u64{1} << tid % kWave) - 1))] =
        static_cast<unsigned short>(tid);
  Items items{0, 0, 0};
  for (int per = 1; per <= kQuarters; per *= 2)
    if (items.count == 0 || items.count > groups) {
      items.per = per;
      items.parts = (c.quarters + per * kRowWaves - 1) / (per * kRowWaves);
      items.count = rows * items.parts;
    }
  return items;  // the caller's next barrier is sh.open's too
}

// The sums of the logit's steps of a part of a row, added to its state.
template <typename T>
__device__ __forceinline__ void AddSteps(const RowCall& c, int row, RowState* state, int part,
                                         int per, const Settings& s, const Weigher& w,
                                         RowShared& sh) {
  for (int i = threadIdx.x; i < kList; i += kRowThreads) {
    sh.counts[i] = 0;
    sh.weights[i] = 0;
  }
  __syncthreads();
  const Steps steps = StepsOf(w);
  const bool share = s.top_p < 1.0F;
  const int first = (part * kRowWaves + WaveIndex()) * per;
#pragma unroll 1
  for (int q = first; q < min(first + per, c.quarters); ++q) {
    float z[kRun];
    LoadLogits<T>(c.p, row, q, z);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int step = steps(z[i]);
      if (step < kList) {
        atomicAdd(&sh.counts[step], 1u);
        if (share)
          atomicAdd(&sh.weights[step], UnitsOf(w.Of(z[i]), c.shift));
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kList; i += kRowThreads)
    if (sh.counts[i] != 0) {
      atomicAdd(&state->counts[i], sh.counts[i]);
      if (share)
        atomicAdd(&state->weights[i], sh.weights[i]);
    }
}

// Whether a list of the quarters' loudest may do, and whether the row's sums of steps are
// formed meanwhile.
__device__ __forceinline__ int OpenedOf(const Settings& s) {
  return s.top_k > 0 ? s.top_k : kShareOpened;
}
__device__ __forceinline__ bool ShortList(const RowCall& c, const Settings& s) {
  return c.quarters <= kMostQuarters && OpenedOf(s) <= min(kMostOpened, c.quarters);
}
__device__ __forceinline__ bool Searches(const RowCall& c, const Settings& s) {
  return !s.lost && !s.greedy && (s.top_k > 0 ? !ShortList(c, s) : s.top_p < 1.0F);
}

// A work-group a row draws what needs no threshold, or from a short list; those behind
// sum the steps of rows that will need them.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void FirstKernel(RowCall c) {
  __shared__ RowShared sh;
  __builtin_assume(c.p.vocab > kChunk);
  const int tid = threadIdx.x, wave = WaveIndex();
  FillTable(sh.powers);
  if (static_cast<int>(blockIdx.x) >= c.rows) {
    const int helpers = gridDim.x - c.rows;
    const Items items = ItemsOf(c, sh, helpers, [&](int at) {
      return Searches(c, SettingsOf(c.p, c.first + at));
    });
#pragma unroll 1
    for (int item = blockIdx.x - c.rows; item < items.count; item += helpers) {
      __syncthreads();  // the last item's sums are read
      const int at = sh.open[item / items.parts], row = c.first + at;
      const Settings s = SettingsOf(c.p, row);
      const unsigned best =
          BestOf<kRowWaves>(WorkOf(c.p, row, c.chunks), c.quarters, sh.most, sh.slots);
      if (best == 0 || best >= kKeyOfInf)
        continue;
      const Weigher w = WeigherOf(sh.powers, best, s.temperature);
      AddSteps<T>(c, row, StateOf(c, at), item % items.parts, items.per, s, w, sh);
    }
    return;
  }
  const int at = blockIdx.x, row = c.first + at;
  const Settings s = SettingsOf(c.p, row);
  const bool share = s.top_p < 1.0F, ranked = c.quarters <= kMostQuarters;
  RowState* const state = StateOf(c, at);
  const Work work = WorkOf(c.p, row, c.chunks);
  const unsigned best = BestOf<kRowWaves>(work, c.quarters, sh.most, sh.slots);
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (tid == 0)
      c.p.tokens[row] = -1;
    return;
  }
  const Weigher w = WeigherOf(sh.powers, best, s.greedy ? 1.0F : s.temperature);
  if (s.greedy) {
    DrawBest<T, kRowWaves>(c, row, work, best, sh.slots);
    return;
  }
  double whole = 0.0;
  if (s.top_k == 0) {
    whole = WholeOf<kRowWaves>(c, work, w, sh.slots);
    if (!share && !(s.min_p > 0.0F)) {
      __syncthreads();
      Pick<T>(c, row, work.weight, nullptr, s, w, 0, 0, sh.pick);
      return;
    }
  }
  const bool known = s.top_k == 0 && !share;  // min_p says the threshold itself
  unsigned floor = known ? KeyOfShare(w, best, s.min_p) : 1;
  if (known ? ranked : ShortList(c, s)) {
    if (!known)
      floor = ReachedBy(sh, c.quarters, OpenedOf(s), best);
    const int listed = Gather<T>(c, row, sh, floor);
    if (listed <= kShortList) {
      if (wave != 0)
        return;
      const u64 of = s.top_k == 0 && share ? static_cast<u64>(ldexp(whole, c.shift)) : 0;
      const auto draw = [&](auto each) {
        return DrawFew<each()>(c.p, row, sh.list, listed, s, w, best, c.shift, of);
      };
      using std::integral_constant;
      if (listed <= 2 * kWave    ? draw(integral_constant<int, 2>())
          : listed <= 4 * kWave  ? draw(integral_constant<int, 4>())
                                 : draw(integral_constant<int, kShortList / kWave>()))
        return;
    }
  }
  if (tid == 0) {
    state->status = known              ? RowState::kKnown
                    : Searches(c, s) ? RowState::kCollect
                                     : RowState::kSlow;
    state->best = best;
    state->t = floor;
    state->whole = static_cast<u64>(ldexp(whole, c.shift));
  }
}

// Every chunk's weight above the steps in which the threshold is, and the list of the
// elements in them, of a part of a row. Each work-group finds the steps from the row's sums
// by itself.
template <typename T>
__device__ __forceinline__ void Collect(const RowCall& c, int at, int part, int per,
                                        RowShared& sh) {
  const int tid = threadIdx.x, row = c.first + at;
  RowState* const state = StateOf(c, at);
  const unsigned status = state->status;
  const Settings s = SettingsOf(c.p, row);
  const bool share = s.top_p < 1.0F;
  const Weigher w = WeigherOf(sh.powers, state->best, s.temperature);
  const Steps steps = StepsOf(w);
  int k_step = kList, low_step = kList, high_step = -1;
  bool raised = false;  // to what is kept from `from` on
  float from = 0.0F;
  if (status == RowState::kKnown) {
    raised = true;
    from = LogitOf(state->t);
  } else {
    for (int i = tid; i < kList; i += kRowThreads) {
      sh.counts[i] = state->counts[i];
      sh.weights[i] = state->weights[i];
    }
    u64 least = state->whole, most = state->whole;  // of what the share is of
    u64 k_count = 0, k_weight = 0;
    if (s.top_k > 0) {
      FindBin(sh, false, s.top_k, 0, 0);
      k_step = low_step = high_step = sh.bin;
      k_count = sh.above_count;
      k_weight = least = sh.above_weight;
      most = k_weight + sh.weights[k_step];
    }
    if (share) {
      FindBin(sh, true, ShareOf(s.top_p, most), 0, 0);
      high_step = min(sh.bin, k_step);
      FindBin(sh, true, ShareOf(s.top_p, max(least, u64{1})), 0, 0);
      low_step = min(sh.bin, high_step);
    }
    unsigned elements = k_step < kList && (k_step < low_step || k_step > high_step)
                            ? sh.counts[k_step] : 0;
    u64 low_count = 0, low_weight = 0;
    for (int i = tid; i < low_step; i += kRowThreads) {
      low_count += sh.counts[i];
      low_weight += sh.weights[i];
    }
    low_count = RowSum<kRowWaves>(low_count, sh.slots);
    low_weight = RowSum<kRowWaves>(low_weight, sh.slots);
    for (int i = low_step; i <= high_step; ++i)
      elements += sh.counts[i];
    if (part == 0 && tid == 0) {
      state->k_step = k_step;
      state->low_step = low_step;
      state->high_step = high_step;
      state->k_count = k_count;
      state->k_weight = k_weight;
      state->low_count = low_count;
      state->low_weight = low_weight;
    }
    // The row's work-groups all see the same; the first one tells the next launch.
    if (s.min_p > 0.0F) {
      const unsigned t = KeyOfShare(w, state->best, s.min_p);
      raised = steps(LogitOf(t)) < low_step;
      from = LogitOf(t);
      if (raised && part == 0 && tid == 0)
        state->raised = t;
    }
    if (!raised && elements > kList) {
      if (part == 0 && tid == 0)
        state->listed = kList + 1;
      return;
    }
  }
  double* const weights = WorkOf(c.p, row, c.chunks).weight;
  const int first = (part * kRowWaves + WaveIndex()) * per;
  double* const sums = reinterpret_cast<double*>(sh.weights);  // of the quarters
  __syncthreads();  // the bins are read
#pragma unroll 1
  for (int i = 0; i < per; ++i) {
    double sum = 0.0;
    if (first + i < c.quarters) {
      float z[kRun];
      LoadLogits<T>(c.p, row, first + i, z);
      const int start = RunStart(first + i, c.p.vocab);
#pragma unroll
      for (int e = 0; e < kRun; ++e) {
        const int step = steps(z[e]);
        if (raised ? z[e] >= from : step < low_step)
          sum += w.Of(z[e]);
        if (!raised && step < kList &&
            ((step >= low_step && step <= high_step) || step == k_step)) {
          const unsigned to = atomicAdd(&state->listed, 1u);
          state->list[min(to, kList - 1u)] =
              static_cast<u64>(KeyOf(z[e])) << 32 | static_cast<unsigned>(start + e);
        }
      }
    }
    sum = WaveSum64(sum);
    if (tid % kWave == 0)
      sums[WaveIndex() * per + i] = sum;
  }
  __syncthreads();
  const int of_part = kRowWaves * per / kQuarters, chunk = part * of_part + tid;
  if (tid < of_part && chunk < c.chunks) {
    const double* const of = sums + tid * kQuarters;
    weights[chunk] = (of[0] + of[1]) + (of[2] + of[3]);
  }
}
template <typename T>
__global__ __launch_bounds__(kRowThreads) void CollectKernel(RowCall c) {
  __shared__ RowShared sh;
  __builtin_assume(c.p.vocab > kChunk);
  FillTable(sh.powers);
  const Items items = ItemsOf(c, sh, gridDim.x, [&](int at) {
    const unsigned status = StateOf(c, at)->status;
    return status == RowState::kCollect || status == RowState::kKnown;
  });
#pragma unroll 1
  for (int item = blockIdx.x; item < items.count; item += gridDim.x) {
    __syncthreads();  // the last item's sums are read
    Collect<T>(c, sh.open[item / items.parts], item % items.parts, items.per, sh);
  }
}

// The threshold from the list of the steps that hold it, or from passes over the row, and
// the draw.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void FinishKernel(RowCall c) {
  __shared__ RowShared sh;
  __builtin_assume(c.p.vocab > kChunk);
  const int tid = threadIdx.x, lane = tid % kWave, wave = WaveIndex();
  const int row = c.first + blockIdx.x;
  RowState* const state = StateOf(c, blockIdx.x);
  const unsigned status = state->status;
  if (status == RowState::kDone)
    return;
  const Settings s = SettingsOf(c.p, row);
  const unsigned best = state->best;
  const Work work = WorkOf(c.p, row, c.chunks);
  FillTable(sh.powers);
  __syncthreads();
  const Weigher w = WeigherOf(sh.powers, best, s.temperature);
  const unsigned from = status == RowState::kKnown ? state->t : state->raised;
  if (from != 0) {
    Pick<T>(c, row, work.weight, nullptr, s, w, from - 1, 0, sh.pick);
    return;
  }
  const Steps steps = StepsOf(w);
  const unsigned listed = state->listed;
  const bool slow = status == RowState::kSlow || listed > kList;
  const bool share = s.top_p < 1.0F;
  if (!slow)
    for (unsigned i = tid; i < listed; i += kRowThreads)
      sh.list[i] = state->list[i];
  __syncthreads();
  // Calls f(key, index) for the listed elements, or the row's.
  const auto each_key = [&](auto&& f) {
    if (!slow) {
      for (unsigned i = tid; i < listed; i += kRowThreads)
        f(static_cast<unsigned>(sh.list[i] >> 32), static_cast<int>(sh.list[i]));
      return;
    }
#pragma unroll 1
    for (int q = wave; q < c.quarters; q += kRowWaves) {
      float z[kRun];
      LoadLogits<T>(c.p, row, q, z);
      const int start = RunStart(q, c.p.vocab);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        f(KeyOf(z[i]), start + i);
    }
  };
  // Of all that can be drawn -infinity is a border that a comparison of logits knows too.
  Kept kept{kKeyOfMinusInf, kAll, 0};
  u64 whole = state->whole;
  // First where top_k ends, then where the share does: sums of 2048 ranges of the keys
  // that may hold the threshold, then of the range that does, until that is one key.
#pragma unroll 1
  for (int turn = s.top_k > 0 ? 0 : 1; turn < (share ? 2 : 1); ++turn) {
    const bool by_weight = turn == 1;
    const u64 want = by_weight ? ShareOf(s.top_p, whole) : s.top_k;
    const int first_step = slow ? 0 : by_weight ? state->low_step : state->k_step;
    const int last_step = slow ? kList : by_weight ? state->high_step : state->k_step;
    u64 above_count = slow ? 0 : by_weight ? state->low_count : state->k_count;
    u64 above_weight = slow ? 0 : by_weight ? state->low_weight : state->k_weight;
    const unsigned floor = kept.t;
    unsigned low = ~0u, high = 0;
    each_key([&](unsigned key, int) {
      const int step = steps(LogitOf(key));
      if (key >= floor && step >= first_step && step <= last_step) {
        low = min(low, key);
        high = max(high, key);
      }
    });
    low = RowJoin<kRowWaves>(WaveMinKey(low), sh.slots,
                             [](unsigned a, unsigned b) { return min(a, b); });
    high = RowJoin<kRowWaves>(WaveMaxKey(high), sh.slots,
                              [](unsigned a, unsigned b) { return max(a, b); });
    low = min(low, high);
    // A top_k that all tokens fit into, or a share that the sums' rounding leaves above all of
    // them, cuts nothing off; the first sums, which are of every key, say so.
    bool one = false, fewer = false;
#pragma unroll 1
    while (!one) {
      const int bits = high == low ? 0 : 32 - __builtin_clz(high - low);
      const int down = bits > 11 ? bits - 11 : 0;
      __syncthreads();
      for (int i = tid; i < kList; i += kRowThreads) {
        sh.weights[i] = 0;
        sh.counts[i] = 0;
      }
      __syncthreads();
      each_key([&](unsigned key, int) {
        if (key >= low && key <= high && key != 0) {
          const unsigned bin = (high - key) >> down;
          atomicAdd(&sh.counts[bin], 1u);
          atomicAdd(&sh.weights[bin], UnitsOf(w(key), c.shift));
        }
      });
      FindBin(sh, by_weight, want, above_count, above_weight);
      const unsigned bin = sh.bin;
      fewer = (by_weight ? sh.above_weight + sh.weights[bin]
                         : sh.above_count + sh.counts[bin]) < want;
      if (fewer) {
        whole = sh.above_weight + sh.weights[bin];
        break;
      }
      above_count = sh.above_count;
      above_weight = sh.above_weight;
      high -= min(bin << down, high - low);
      low = max(low, high - min(high, (1u << down) - 1));
      one = down == 0;
    }
    if (fewer)
      continue;
    const u64 equal = sh.counts[sh.bin], each = UnitsOf(w(high), c.shift);
    u64 need = equal;
    if (!by_weight)
      need = min(need, want - min(want, above_count));
    else if (each > 0)
      need = min(need, (want - min(want, above_weight) + each - 1) / each);
    if (by_weight && high == kept.t)
      need = min(need, kept.need);
    kept = Kept{high, need, 0};
    whole = above_weight + need * each;  // what top_k keeps
    __syncthreads();
  }
  if (s.min_p > 0.0F) {
    const unsigned t = KeyOfShare(w, best, s.min_p);
    if (t > kept.t)
      kept = Kept{t, kAll, 0};
  }
  // The chunks' kept weights: above the listed steps by the launch before, and the list's.
  const bool held = c.chunks <= kList;  // in LDS
  double* const weights = reinterpret_cast<double*>(sh.weights);
  if (!slow && held) {
    __syncthreads();
    for (int i = tid; i < c.chunks; i += kRowThreads) {
      sh.weights[i] = 0;
      sh.counts[i] = 0;
    }
    __syncthreads();
    const int first_step = state->low_step;
    each_key([&](unsigned key, int index) {
      if (steps(LogitOf(key)) < first_step)
        return;
      if (key > kept.t)
        atomicAdd(&sh.weights[index / kChunk], UnitsOf(w(key), c.shift));
      else if (key == kept.t)
        atomicAdd(&sh.counts[index / kChunk], 1u);
    });
    __syncthreads();
    for (int i = tid; i < c.chunks; i += kRowThreads)
      weights[i] = work.weight[i] + ldexp(static_cast<double>(sh.weights[i]), -c.shift);
    __syncthreads();
    Pick<T>(c, row, weights, sh.counts, s, w, kept.t, kept.need, sh.pick);
    return;
  }
  // The whole row once more, for its chunks above the threshold and the equals. The equals
  // take the place of the quarters' largest keys, which are no longer needed.
  unsigned* const equals = work.most;
  const float border = LogitOf(kept.t);
#pragma unroll 1
  for (int chunk = wave; chunk < c.chunks; chunk += kRowWaves) {
    double sum = 0.0;
    unsigned equal = 0;
    EachQuarter<T>(c.p, row, chunk, [&](int, const float (&z)[kRun]) {
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if (z[i] > border)
          sum += w.Of(z[i]);
        equal += z[i] == border;
      }
    });
    sum = WaveSum64(sum);
    equal = static_cast<unsigned>(WaveSum64(static_cast<u64>(equal)));
    if (lane == 0) {
      work.weight[chunk] = sum;
      equals[chunk] = equal;
    }
  }
  __syncthreads();
  Pick<T>(c, row, work.weight, equals, s, w, kept.t, kept.need, sh.pick);
}

constexpr std::int64_t kMostGroups = 1 << 23;  // of the first launch: lanes count under 2^32
int ChunksOf(int vocab) { return vocab <= kChunk ? 0 : (vocab - 1) / kChunk + 1; }

}  // namespace

std::int64_t SampleWorkBytes(std::int64_t rows, std::int64_t vocab) {
  const std::int64_t chunks = ChunksOf(static_cast<int>(vocab));
  if (rows * ((chunks + kWaves - 1) / kWaves) >= kMostGroups)
    return -1;
  if (chunks == 0)
    return 0;
  return rows * WorkWords(chunks) * static_cast<std::int64_t>(sizeof(unsigned)) +
         std::min<std::int64_t>(rows, kBatch) * static_cast<std::int64_t>(sizeof(RowState));
}

void LaunchSample(const SampleParams& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.vocab >= 1, "sample: empty shape");
  int bits = 0;
  while ((std::int64_t{1} << bits) < p.vocab)
    ++bits;
  RowCall c{p, 0, p.rows, ChunksOf(p.vocab), (p.vocab - 1) / kQuarter + 1, std::min(62 - bits, 51)};
  const int groups = (c.chunks + kWaves - 1) / kWaves;
  WithType(type, [&](auto t) {
    using T = decltype(t);
    const auto small = [&](auto q) {
      Dispatch(SmallKernel<T, q()>, dim3((p.rows + kWaves - 1) / kWaves), dim3(kThreads), 0,
               stream, true, true, p, c.shift);
    };
    if (c.chunks == 0) {
      if (c.quarters == 1)
        small(std::integral_constant<int, 1>());
      else if (c.quarters == 2)
        small(std::integral_constant<int, 2>());
      else if (c.quarters == 3)
        small(std::integral_constant<int, 3>());
      else
        small(std::integral_constant<int, kQuarters>());
      return;
    }
    const bool filters = p.top_ks != nullptr || p.top_ps != nullptr || p.min_ps != nullptr ||
                         p.top_k > 0 || p.top_p < 1.0F || p.min_p > 0.0F;
    const bool clear = filters && p.rows <= kBatch;  // else batch by batch
    Dispatch(ChunkKernel<T>, dim3(p.rows * groups), dim3(kThreads), 0, stream, true, false, c,
             groups, clear);
    if (!filters) {
      Dispatch(PlainKernel<T>, dim3(p.rows), dim3(kThreads), 0, stream, false, true, c);
      return;
    }
    for (c.first = 0; c.first < p.rows; c.first += kBatch) {
      c.rows = std::min(p.rows - c.first, kBatch);
      const bool last = c.first + kBatch >= p.rows;
      if (!clear)
        Dispatch(ClearKernel, dim3(c.rows), dim3(kThreads), 0, stream, false, false, c);
      // A work-group fills a CU.
      const int parts = static_cast<int>(std::min<std::int64_t>(
          std::int64_t{c.rows} * ((c.quarters + kRowWaves - 1) / kRowWaves), kCus));
      // What the rows leave of the CUs, or half of them where they leave less: with an eighth
      // 300 rows of 151936 with top_p 0.9 take 685 us, with half 328, 512 of 32000 265 and
      // 140 (with all 280 and 121); 64 rows of 151936 97 with what is left, 106 with half.
      const int helpers = std::min(parts, std::max(kCus - c.rows, kCus / 2));
      Dispatch(FirstKernel<T>, dim3(c.rows + helpers), dim3(kRowThreads), 0, stream, false, false,
               c);
      Dispatch(CollectKernel<T>, dim3(parts), dim3(kRowThreads), 0, stream, false, false, c);
      Dispatch(FinishKernel<T>, dim3(c.rows), dim3(kRowThreads), 0, stream, false, last, c);
    }
  });
  Check(hipGetLastError(), "sample launch");
}

}  // namespace ovg
