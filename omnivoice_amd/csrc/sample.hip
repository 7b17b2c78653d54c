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
// Up to 2048 tokens a wave has its row in registers and searches thresholds by halves.
// Larger vocabularies take two launches. The first has a wave for every chunk of 2048
// tokens, which leaves the largest key of each quarter and, where the row needs it, the
// chunk's weight beside its own largest. The second has a work-group for every row.
// Without filters it finds the chunk by the chunks' weights and reads only that one. The
// k best lie in the k quarters with the largest keys, so with filters it reads those (64
// for top_p alone) and ranks the few elements that reach the last one's. Where that is
// not enough (a large k, a share that needs more) it reads the row again: sums of 2048
// steps of the logit, passes over what the step that was found holds, and one for the
// chunks' kept weights. With few rows these take launches of their own, in which all CUs
// share the rows, and which end at once where no row needs them.
//
// A draw lands where sums of up to 2^17 weights say, so weights have 2^-42 and better:
// 2^x in 64 bits from a table of 256 powers and three terms. Sums that several lanes
// form in any order are whole numbers of 2^-shift; the others are 64-bit numbers in a
// fixed order. No result depends on the order of the work.
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
constexpr int kShortList = 512;             // of which every element is ranked
constexpr int kList = 2048;                 // elements of a list
constexpr int kShareOpened = 64;            // opened for a share alone
constexpr int kOctaves = 50;                // weights below 2^-50 do not count
constexpr int kTable = 256;

// ---------------------------------------------------------------- lanes
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
template <typename T>
__device__ __forceinline__ void LoadKeys(const SampleParams& p, std::int64_t row, int q,
                                         unsigned (&key)[kRun]) {
  float z[kRun];
  LoadLogits<T>(p, row, q, z);
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    key[i] = KeyOf(z[i]);
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
  __device__ __forceinline__ double operator()(unsigned key) const {
    const double w = Raw(LogitOf(key));
    return (key != 0) & (w >= 0x1p-50) ? w : 0.0;
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
  // Whether the sums of the row's steps may be asked for.
  __device__ __forceinline__ bool Searches(int quarters) const {
    return !lost && !greedy &&
           (top_k > min(kMostOpened, quarters) || (top_k == 0 && top_p < 1.0F));
  }
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

// N elements a lane, of which `used` registers are in use in some lane.
template <int N>
struct Held {
  unsigned key[N];
  u64 weight[N];
  int used;
  __device__ __forceinline__ int Count(unsigned t) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= used)
        break;
      n += __popcll(__ballot(key[i] >= t));
    }
    return n;
  }
  __device__ __forceinline__ u64 Weight(unsigned t) const {
    u64 n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= used)
        break;
      n += key[i] >= t ? weight[i] : 0;
    }
    return WaveSum64(n);
  }
  __device__ __forceinline__ unsigned Least() const {  // 1 or more
    unsigned n = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= used)
        break;
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
  // Of all that is held, or the prefix of weight ShareOf(top_p, *whole) of it where the
  // row holds more; false where that does not reach.
  __device__ __forceinline__ bool Select(const Settings& s, const Weigher& w, unsigned best,
                                         int shift, const u64* whole, Kept* kept) const {
    const unsigned least = Least();
    kept->t = least;
    kept->need = kAll;
    kept->weight = Weight(1);
    if (s.top_k > 0 && Count(1) > s.top_k) {
      kept->t = Search(least, best, [&](unsigned t) { return Count(t) >= s.top_k; });
      const unsigned above = kept->t + 1;
      kept->need = s.top_k - Count(above);
      kept->weight = Weight(above) + kept->need * UnitsOf(w(kept->t), shift);
    }
    if (s.top_p < 1.0F) {
      const u64 want = ShareOf(s.top_p, whole != nullptr ? *whole : kept->weight);
      if (kept->weight < want)
        return false;
      const unsigned low = kept->t;
      u64 above = Weight(low + 1);
      if (above >= want) {
        kept->t = Search(low + 1, best, [&](unsigned t) { return Weight(t) >= want; });
        kept->need = kAll;
        above = Weight(kept->t + 1);
      }
      const u64 each = UnitsOf(w(kept->t), shift);
      if (each > 0) {
        kept->need = min(kept->need, (want - above + each - 1) / each);
        kept->need = min(kept->need, static_cast<u64>(Count(kept->t) - Count(kept->t + 1)));
        kept->weight = above + kept->need * each;
      }
    }
    if (s.min_p > 0.0F) {
      const unsigned t = KeyOfShare(w, best, s.min_p);
      if (t > kept->t) {
        kept->t = t;
        kept->need = kAll;
        kept->weight = Weight(t);
      }
    }
    return true;
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
// A wave a row of up to 512 Q tokens. With a top_k of 64 or less, the lanes' largest keys
// give a floor that the k best reach, and the few elements that do go through LDS, in the
// row's order, to two a lane.
constexpr int kFew = 2 * kWave;

template <typename T, int Q>
__global__ __launch_bounds__(kThreads) void SmallKernel(SampleParams p, int shift) {
  constexpr int N = Q * kRun;
  __shared__ double powers[kTable];
  __shared__ u64 few[kWaves][kFew];  // key, index
  FillTable(powers);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int row = blockIdx.x * kWaves + wave;
  Held<N> held;
  held.used = N;
  Settings s{};
  if (row < p.rows) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      unsigned key[kRun];
      LoadKeys<T>(p, row, q, key);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        held.key[q * kRun + i] = key[i];
    }
  }
  __syncthreads();
  if (row >= p.rows)
    return;
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    most = max(most, held.key[i]);
  const unsigned best = WaveMaxKey(most);
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (lane == 0)
      p.tokens[row] = -1;
    return;
  }
  const Weigher w = WeigherOf(powers, best, s.greedy ? 1.0F : s.temperature);
  Kept kept{best, 1, 1};
  u64 left, need;
  int of, place;
  if (!s.greedy && s.top_k > 0 && s.top_k <= kWave) {
    const unsigned floor = Held<1>::Search(1, best, [&](unsigned t) {
      return __popcll(__ballot(most >= t)) >= s.top_k;
    });
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
      Held<2> best_few;
      best_few.used = 2;
      int index[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u64 e = 2 * lane + i < listed ? few[wave][2 * lane + i] : 0;
        best_few.key[i] = static_cast<unsigned>(e >> 32);
        index[i] = static_cast<int>(e);
        best_few.weight[i] = UnitsOf(w(best_few.key[i]), shift);
      }
      best_few.Select(s, w, best, shift, nullptr, &kept);
      left = TargetOf(s.u, kept.weight);
      need = kept.need;
      if (DrawOf(best_few.key, best_few.weight, kept.t, &need, &left, &of, &place)) {
        const int token = place == 0 ? index[0] : index[1];
        if (lane == of)
          p.tokens[row] = token;
      }
      return;
    }
  }
  if (s.greedy) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      held.weight[i] = held.key[i] == best;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      held.weight[i] = UnitsOf(w(held.key[i]), shift);
    held.Select(s, w, best, shift, nullptr, &kept);
  }
  left = TargetOf(s.greedy ? 0.0F : s.u, kept.weight);
  need = kept.need;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    unsigned key[kRun];
    u64 weight[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      key[i] = held.key[q * kRun + i];
      weight[i] = held.weight[q * kRun + i];
    }
    if (DrawOf(key, weight, kept.t, &need, &left, &of, &place)) {
      if (lane == of)
        p.tokens[row] = RunStart(q, p.vocab) + place;
      return;
    }
  }
}

// ---------------------------------------------------------------- large rows
// A row's part of the workspace: the chunks' weights, their equals of a threshold, the
// quarters' largest keys.
struct Work {
  double* weight;
  unsigned* equal;
  unsigned* most;
};
// What a row goes on with in the launches of its own passes, and their sums.
struct RowState {
  enum : unsigned { kDone, kSearch, kPick };
  unsigned status, t, best, spare;
  u64 need;
  unsigned counts[kList];
  u64 weights[kList];
};
constexpr int kSplitRows = 256;
__host__ __device__ constexpr std::int64_t WorkWords(std::int64_t chunks) {
  return (chunks * (2 + 1 + kQuarters) + 3) / 4 * 4;
}
__device__ __forceinline__ RowState* StateOf(const SampleParams& p, int row, int chunks) {
  return reinterpret_cast<RowState*>(p.work + WorkWords(chunks) * p.rows) + row;
}
__device__ __forceinline__ Work WorkOf(const SampleParams& p, int row, int chunks) {
  double* const base = reinterpret_cast<double*>(p.work + WorkWords(chunks) * row);
  unsigned* const equal = reinterpret_cast<unsigned*>(base + chunks);
  return {base, equal, equal + chunks};
}

// The largest key of every quarter of a chunk, and the chunk's weight beside the
// chunk's own largest.
template <typename T>
__global__ __launch_bounds__(kThreads) void ChunkKernel(SampleParams p, int chunks, int groups,
                                                        bool split) {
  __shared__ double powers[kTable];
  __builtin_assume(p.vocab > kChunk);
  FillTable(powers);
  const int lane = threadIdx.x % kWave;
  const int row = blockIdx.x / groups;
  const int chunk = (blockIdx.x - row * groups) * kWaves + threadIdx.x / kWave;
  float z[kQuarters][kRun];
  Settings s{};
  if (chunk < chunks) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
      LoadLogits<T>(p, row, chunk * kQuarters + q, z[q]);
  }
  if (split && s.Searches((p.vocab - 1) / kQuarter + 1)) {  // the sums that the next launch adds to
    RowState* const state = StateOf(p, row, chunks);
    const int part = blockIdx.x - row * groups;
    for (int i = part * kThreads + threadIdx.x; i < kList; i += groups * kThreads) {
      state->counts[i] = 0;
      state->weights[i] = 0;
    }
  }
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

struct RowShared {
  double powers[kTable];
  u64 weights[kList];  // of a pass's bins; as 64-bit numbers, the chunks'
  unsigned counts[kList];
  unsigned most[kMostQuarters];
  u64 list[kList];     // key, index
  unsigned short open[kMostQuarters];
  u64 unit[kShortList];    // the list's weights
  u64 before[kShortList];
  int rank[kShortList];
  u64 slots[kRowWaves], count_slots[kRowWaves];
  unsigned listed, opened, t;
  int bin;
  u64 above_weight, above_count;
};

// v is the same in every lane of a wave.
template <int WAVES = kRowWaves, typename V, typename F>
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

// What a search goes over: the row, or the list of all its keys from some key on.
struct Source {
  bool list;
  int count;
};

// Calls f(key, index) for the elements, a wave a chunk of the row.
template <typename T, typename F>
__device__ __forceinline__ void EachKey(const SampleParams& p, int row, int chunks,
                                        const RowShared& sh, const Source& from, F&& f) {
  if (from.list) {
    for (int i = threadIdx.x; i < from.count; i += kRowThreads)
      f(static_cast<unsigned>(sh.list[i] >> 32), static_cast<int>(sh.list[i]));
    return;
  }
  for (int c = threadIdx.x / kWave; c < chunks; c += kRowWaves) {
    float z[kQuarters][kRun];
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
      LoadLogits<T>(p, row, c * kQuarters + q, z[q]);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q) {
      const int start = RunStart(c * kQuarters + q, p.vocab);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        f(KeyOf(z[q][i]), start + i);
    }
  }
}

// The list of the row's keys from `floor` to `high`; false where it does not hold them.
// Quarters without any are not read. The whole work-group calls this.
template <typename T>
__device__ __forceinline__ bool Gather(const SampleParams& p, int row, int quarters,
                                       RowShared& sh, const unsigned* most, unsigned floor,
                                       unsigned high) {
  constexpr int kAtOnce = 4;  // quarters' loads of a wave
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x == 0)
    sh.listed = 0;
  for (int first = 0; first < quarters; first += kMostQuarters) {
    if (threadIdx.x == 0)
      sh.opened = 0;
    __syncthreads();
    const int count = min(quarters - first, kMostQuarters);
    for (int q = threadIdx.x; q < count; q += kRowThreads)
      if (most[first + q] >= floor)
        sh.open[atomicAdd(&sh.opened, 1u)] = static_cast<unsigned short>(q);
    __syncthreads();
    const int opened = static_cast<int>(sh.opened);
    for (int o = wave; o < opened; o += kAtOnce * kRowWaves) {
      float z[kAtOnce][kRun];
      int q[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        q[i] = first + sh.open[min(o + i * kRowWaves, opened - 1)];
        LoadLogits<T>(p, row, q[i], z[i]);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (o + i * kRowWaves >= opened)
          break;
        const int start = RunStart(q[i], p.vocab);
#pragma unroll
        for (int e = 0; e < kRun; ++e) {
          const unsigned key = KeyOf(z[i][e]);
          if (key >= floor && key <= high) {
            const unsigned at = atomicAdd(&sh.listed, 1u);
            if (at < kList)
              sh.list[at] = static_cast<u64>(key) << 32 | static_cast<unsigned>(start + e);
          }
        }
      }
    }
    __syncthreads();
  }
  return sh.listed <= kList;
}

// 2048 equal steps of the logit from the best down to the smallest weight that counts.
struct Steps {
  float top, scale;
  __device__ __forceinline__ int operator()(unsigned key) const {
    const float at = fminf(top - LogitOf(key), 3e38F) * scale;
    return at < static_cast<float>(kList) ? static_cast<int>(at) : kList;
  }
  // The smallest key of a step up to `last`; 64 keys at once.
  __device__ __forceinline__ unsigned Least(unsigned best, int last) const {
    unsigned low = kKeyOfMinusInf, high = best;
    while (high - low > 1) {
      const unsigned step = (high - low + kWave - 1) / kWave;
      const unsigned key = min(low + step * (threadIdx.x % kWave + 1), high);
      const int at = __builtin_ctzll(__ballot(key == high || (*this)(key) <= last));
      high = min(low + step * (at + 1), high);
      low += step * at;
    }
    return high;
  }
};
__device__ __forceinline__ Steps StepsOf(const Weigher& w) {
  return {static_cast<float>(w.top),
          fminf(static_cast<float>(w.per * (static_cast<double>(kList) / (kOctaves * kTable))),
                1e30F)};
}

// The key at which the count of keys (or their weight) reaches `want`, from the top: sums
// of the logit's steps (from `state`, or a pass over the elements), then of equal ranges
// of the keys in the step that was found, until that is one key. Where the first sums
// leave few elements the passes go over a list, of all from that step up if it holds
// them. Below `floor` nothing counts. The whole work-group calls this; the result is in
// sh.t, sh.above_count and sh.above_weight.
template <typename T, bool WEIGHT>
__device__ __forceinline__ void RowSearch(const SampleParams& p, int row, int chunks,
                                          int quarters, const unsigned* most, RowShared& sh,
                                          Source* from, const RowState* state, const Weigher& w,
                                          int shift, unsigned best, unsigned floor, u64 want) {
  constexpr int kBins = kList;
  const int tid = threadIdx.x, lane = tid % kWave;
  u64 above_weight = 0, above_count = 0;
  // The bin in which the sums of the bins (0 is the top one) reach: two bins a thread.
  const auto find = [&] {
    static_assert(kBins == 2 * kRowThreads, "two bins a thread");
    __syncthreads();
    const u64 w0 = sh.weights[2 * tid], w1 = sh.weights[2 * tid + 1];
    const unsigned c0 = sh.counts[2 * tid], c1 = sh.counts[2 * tid + 1];
    u64 weight_to = WaveScan(w0 + w1);
    u64 count_to = WaveScan(static_cast<unsigned>(c0 + c1));
    if (lane == kWave - 1) {
      sh.slots[tid / kWave] = weight_to;
      sh.count_slots[tid / kWave] = count_to;
    }
    __syncthreads();
    weight_to += above_weight;
    count_to += above_count;
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) {
      const bool before = i < tid / kWave;
      weight_to += before ? sh.slots[i] : 0;
      count_to += before ? sh.count_slots[i] : 0;
    }
    const u64 weight = weight_to - w0 - w1, count = count_to - c0 - c1;
    const u64 to = WEIGHT ? weight_to : count_to, from_here = WEIGHT ? weight : count;
    // The last bin takes what fewer keys or the sums' rounding leave.
    if ((to >= want && (from_here < want || tid == 0)) || (tid == kRowThreads - 1 && to < want)) {
      const bool second = (WEIGHT ? weight + w0 : count + c0) < want;
      sh.bin = 2 * tid + second;
      sh.above_weight = weight + (second ? w0 : 0);
      sh.above_count = count + (second ? c0 : 0);
    }
    __syncthreads();
    above_weight = sh.above_weight;
    above_count = sh.above_count;
    return sh.bin;
  };
  const auto pass = [&](const Source& source, auto&& bin_of) {
    __syncthreads();
    for (int i = tid; i < kBins; i += kRowThreads) {
      sh.weights[i] = 0;
      sh.counts[i] = 0;
    }
    __syncthreads();
    EachKey<T>(p, row, chunks, sh, source, [&](unsigned key, int) {
      const int bin = bin_of(key);
      if (key >= floor && bin < kBins) {
        atomicAdd(&sh.counts[bin], 1u);
        if constexpr (WEIGHT)
          atomicAdd(&sh.weights[bin], UnitsOf(w(key), shift));
      }
    });
    return find();
  };
  const Steps steps = StepsOf(w);
  int first;
  if (state != nullptr && !from->list) {
    __syncthreads();
    for (int i = tid; i < kBins; i += kRowThreads) {
      sh.weights[i] = state->weights[i];
      sh.counts[i] = state->counts[i];
    }
    first = find();
  } else {
    first = pass(*from, steps);
  }
  const unsigned held = sh.counts[first];
  unsigned low = max(steps.Least(best, first), floor);
  unsigned high = first == 0 ? best : steps.Least(best, first - 1) - 1;
  Source source = *from;
  if (!from->list && held <= kList && low < high) {
    const bool all = above_count + held <= kList;
    source.list = Gather<T>(p, row, quarters, sh, most, low, all ? best : high);
    source.count = static_cast<int>(sh.listed);
    if (all)
      *from = source;
  }
  while (low < high) {
    const int bits = 32 - __builtin_clz(high - low);
    const int down = bits > 11 ? bits - 11 : 0;
    const int bin = pass(source, [&](unsigned key) {
      return key >= low && key <= high ? static_cast<int>((high - key) >> down) : kBins;
    });
    high -= min(static_cast<unsigned>(bin) << down, high - low);
    low = max(low, down == 0 ? high : high - min(high, (1u << down) - 1));
  }
  __syncthreads();
  if (tid == 0)
    sh.t = high;
  __syncthreads();
}

// For every element of a list, what `ahead` of it others count and weigh, added to
// sh.rank and sh.before: a wave has 64 elements and a part of the others.
template <typename F>
__device__ __forceinline__ void RankList(RowShared& sh, int listed, F&& ahead) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int groups = (listed + kWave - 1) / kWave, parts = kRowWaves / groups;
  const int part = wave / groups, e = wave % groups * kWave + lane;
  if (part >= parts)
    return;
  const u64 mine = sh.list[min(e, listed - 1)];
  int rank = 0;
  u64 before = 0;
  for (int i = part; i < listed; i += parts) {
    const bool in = ahead(sh.list[i], mine);
    rank += in;
    before += in ? sh.unit[i] : 0;
  }
  if (e < listed) {
    atomicAdd(&sh.rank[e], rank);
    atomicAdd(&sh.before[e], before);
  }
}

// The draw from a short list, an element a thread; false where the list does not hold the
// share. The whole work-group calls this.
__device__ __forceinline__ bool DrawFromList(const SampleParams& p, int row, RowShared& sh,
                                             int listed, const Settings& s, const Weigher& w,
                                             int shift, double all) {
  static_assert(kShortList <= kRowThreads && kShortList <= kRowWaves * kWave, "elements");
  const int e = threadIdx.x;
  const bool there = e < listed, share = s.top_p < 1.0F;
  const auto total = [&](u64 v) {
    return RowJoin(WaveSum64(v), sh.slots, [](u64 a, u64 b) { return a + b; });
  };
  u64 whole = static_cast<u64>(ldexp(all, shift));
  if (s.top_k > 0)  // few elements take finer units, where they are all that counts
    shift = 51;
  const u64 element = there ? sh.list[e] : 0;
  const double weight = w(static_cast<unsigned>(element >> 32));
  const u64 unit = UnitsOf(weight, shift);
  if (share && s.top_k == 0 && total(unit) < ShareOf(s.top_p, whole))
    return false;
  if (e < kShortList) {
    sh.unit[e] = unit;
    sh.rank[e] = 0;
    sh.before[e] = 0;
  }
  __syncthreads();
  // Ahead are larger keys and equal ones of smaller index.
  RankList(sh, listed, [](u64 other, u64 mine) {
    return (other ^ 0xFFFFFFFFu) > (mine ^ 0xFFFFFFFFu);
  });
  __syncthreads();
  const int rank = there ? sh.rank[e] : kList;
  const u64 before = there ? sh.before[e] : 0;
  const int most = s.top_k > 0 ? s.top_k : listed;
  if (s.top_k > 0 && share)
    whole = total(rank < most ? unit : 0);
  const double least = fmin(static_cast<double>(s.min_p), 1.0);
  const bool in = rank < most && (!share || before < ShareOf(s.top_p, whole)) && weight >= least;
  const u64 kept = in || rank == 0 ? unit : 0;
  const u64 target = TargetOf(s.u, total(kept));
  if (there) {
    sh.unit[e] = kept;
    sh.before[e] = 0;
  }
  __syncthreads();
  RankList(sh, listed, [](u64 other, u64 mine) {
    return static_cast<unsigned>(other) < static_cast<unsigned>(mine);
  });
  __syncthreads();
  if (there && sh.before[e] <= target && target < sh.before[e] + kept)
    p.tokens[row] = static_cast<int>(element);
  return true;
}

// The chunk's kept weight: above the threshold, and how many equal it. A wave's.
template <typename T>
__device__ __forceinline__ void KeptOfChunk(const SampleParams& p, int row, int c, unsigned t,
                                            const Weigher& w, double* weight, unsigned* equals) {
  double sum = 0.0;
  unsigned equal = 0;
  float z[kQuarters][kRun];
#pragma unroll
  for (int q = 0; q < kQuarters; ++q)
    LoadLogits<T>(p, row, c * kQuarters + q, z[q]);
#pragma unroll
  for (int q = 0; q < kQuarters; ++q)
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const unsigned key = KeyOf(z[q][i]);
      if (key > t)
        sum += w(key);
      equal += key == t;
    }
  sum = WaveSum64(sum);
  const u64 n = WaveSum64(static_cast<u64>(equal));
  if (threadIdx.x % kWave == 0) {
    *weight = sum;
    *equals = static_cast<unsigned>(n);
  }
}

// The draw by the chunks' kept weights: one wave finds the chunk, 64 at a time, then the
// place in it. Without a threshold (t is 0) `all` is what is kept.
template <typename T>
__device__ __forceinline__ void Pick(const SampleParams& p, int row, int chunks,
                                     const double* weights, const unsigned* equals,
                                     const Settings& s, const Weigher& w, unsigned t, u64 need0,
                                     double all) {
  const int lane = threadIdx.x % kWave;
  const bool chunked = t == 0;
  const double each = chunked ? 0.0 : w(t);
  // The kept weight of the lane's chunk and the equals before it, of 64 chunks with `need`
  // equals left.
  const auto chunk_weight = [&](int c, u64 need, u64* equal_to, u64* equal_before) {
    const unsigned equal = c < chunks && !chunked ? equals[c] : 0;
    *equal_to = chunked ? 0 : WaveScan(static_cast<u64>(equal));
    *equal_before = *equal_to - equal;
    const u64 in = need > *equal_before ? min(need - *equal_before, static_cast<u64>(equal)) : 0;
    return (c < chunks ? weights[c] : 0.0) + static_cast<double>(in) * each;
  };
  const auto last_lane = [](double v) {
    return __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, v), kWave - 1));
  };
  u64 need = need0, equal_to, equal_before;
  double total = all;
  if (!chunked) {
    total = 0.0;
    for (int c0 = 0; c0 < chunks; c0 += kWave) {
      total += WaveSum64(chunk_weight(c0 + lane, need, &equal_to, &equal_before));
      need -= min(need, Lane64(equal_to, kWave - 1));
    }
  }
  double left = static_cast<double>(fminf(fmaxf(s.u, 0.0F), 1.0F)) * total;
  if (!(left < total))
    left = total * (1.0 - 0x1p-53);
  need = need0;
  bool done = false;
  double before = 0.0;
  int last = 0;  // the chunk; the last one that keeps any where rounding leaves none
  double last_before = 0.0;
  u64 last_need = 0;
  for (int c0 = 0; c0 < chunks && !done; c0 += kWave) {
    const double mine = chunk_weight(c0 + lane, need, &equal_to, &equal_before);
    const double to = before + WaveScan(mine);
    const u64 hit = __ballot(mine > 0.0 && to > left);
    const u64 any = __ballot(mine > 0.0);
    if (any != 0) {
      const int l = hit != 0 ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
      last = c0 + l;
      last_before = __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, to - mine), l));
      last_need = need - min(need, Lane64(equal_before, l));
    }
    done = hit != 0;
    before = last_lane(to);
    need -= min(need, Lane64(equal_to, kWave - 1));
  }
  left -= last_before;
  need = last_need;
  unsigned key[kQuarters][kRun];
#pragma unroll
  for (int q = 0; q < kQuarters; ++q)
    LoadKeys<T>(p, row, last * kQuarters + q, key[q]);
  int token = -1, most_of = -1;  // the last kept one, where rounding leaves none
#pragma unroll
  for (int q = 0; q < kQuarters; ++q) {
    if (token >= 0)
      break;
    unsigned equal = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      equal += !chunked && key[q][i] == t;
    const unsigned equals_to = __ballot(equal != 0) != 0 ? WaveScan(equal) : 0;
    u64 seen = equals_to - equal;
    double to_place[kRun], mine = 0.0;
    int end = -1;  // the lane's last kept one
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const bool in = chunked || key[q][i] > t || (key[q][i] == t && seen++ < need);
      const double weight = in ? w(key[q][i]) : 0.0;
      end = weight > 0.0 ? i : end;
      mine += weight;
      to_place[i] = mine;
    }
    const double to = WaveScan(mine);
    const u64 hit = __ballot(mine > 0.0 && to > left);
    const u64 any = __ballot(mine > 0.0);
    int place = end;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const double before_it = i > 0 ? to_place[i - 1] : 0.0;
      place = to_place[i] > before_it && (to - mine) + to_place[i] > left ? i : place;
    }
    place += RunStart(last * kQuarters + q, p.vocab);
    if (any != 0) {
      most_of = __builtin_amdgcn_readlane(place, hit != 0 ? __builtin_ctzll(hit)
                                                          : 63 - __builtin_clzll(any));
      token = hit != 0 ? most_of : -1;
    }
    left -= last_lane(to);
    need -= min(need, static_cast<u64>(__builtin_amdgcn_readlane(equals_to, kWave - 1)));
  }
  if (lane == 0)
    p.tokens[row] = token >= 0 ? token : most_of;
}

// The sums of the logit's steps of `row`'s chunks from `first` on, by a work-group.
constexpr int kStepChunks = 16;  // of a work-group
template <typename T>
__device__ __forceinline__ void AddSteps(const SampleParams& p, int row, int chunks, int quarters,
                                         int shift, int first, const Settings& s, RowShared& sh) {
  RowState* const state = StateOf(p, row, chunks);
  const Work work = WorkOf(p, row, chunks);
  unsigned best = 0;
  for (int i = threadIdx.x; i < quarters; i += kRowThreads)
    best = max(best, work.most[i]);
  for (int i = threadIdx.x; i < kList; i += kRowThreads) {
    sh.counts[i] = 0;
    sh.weights[i] = 0;
  }
  best = RowJoin(WaveMaxKey(best), sh.slots, [](unsigned a, unsigned b) { return max(a, b); });
  if (best == 0 || best >= kKeyOfInf)
    return;
  const Weigher w = WeigherOf(sh.powers, best, s.temperature);
  const Steps steps = StepsOf(w);
  const bool share = s.top_p < 1.0F;
  const int c = first + static_cast<int>(threadIdx.x / kWave);
  static_assert(kStepChunks == kRowWaves, "a wave a chunk");
  if (c < chunks) {
    float z[kQuarters][kRun];
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
      LoadLogits<T>(p, row, c * kQuarters + q, z[q]);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const unsigned key = KeyOf(z[q][i]);
        const int step = steps(key);
        if (key != 0 && step < kList) {
          atomicAdd(&sh.counts[step], 1u);
          if (share)
            atomicAdd(&sh.weights[step], UnitsOf(w(key), shift));
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

// kWhole: a row from the chunks' numbers to its token. Else the row's passes are spread
// over work-groups and launches of their own: kFirst does what needs none, while other
// work-groups sum the steps of rows that may search, kSearch finds the threshold from
// the sums, kPick draws from the chunks' kept weights.
// kPlain: rows of which none has a filter.
enum class Phase { kPlain, kWhole, kFirst, kSearch, kPick };
constexpr int ThreadsOf(Phase phase) {
  return phase == Phase::kPlain ? kThreads : phase == Phase::kPick ? kWave : kRowThreads;
}

template <typename T, Phase PHASE>
__global__ __launch_bounds__(ThreadsOf(PHASE)) void RowKernel(SampleParams p, int chunks, int quarters,
                                                         int shift) {
  __shared__ RowShared sh;
  __builtin_assume(p.vocab > kChunk);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int row = blockIdx.x % p.rows;
  if (PHASE == Phase::kFirst && static_cast<int>(blockIdx.x) >= p.rows) {
    const Settings s = SettingsOf(p, row);
    if (!s.Searches(quarters))
      return;
    FillTable(sh.powers);
    AddSteps<T>(p, row, chunks, quarters, shift,
                (static_cast<int>(blockIdx.x) / p.rows - 1) * kStepChunks, s, sh);
    return;
  }
  constexpr int kGroup = ThreadsOf(PHASE), kGroupWaves = kGroup / kWave;
  constexpr bool kOwn = PHASE == Phase::kPlain || PHASE == Phase::kWhole;
  RowState* const state = kOwn ? nullptr : StateOf(p, row, chunks);
  if (PHASE == Phase::kSearch && state->status != RowState::kSearch)
    return;
  if (PHASE == Phase::kPick && state->status != RowState::kPick)
    return;
  const Settings s = SettingsOf(p, row);
  const Work work = WorkOf(p, row, chunks);
  FillTable(sh.powers);
  // The chunks' and quarters' numbers, in LDS where they fit.
  double* const weights =
      chunks <= kList ? reinterpret_cast<double*>(sh.weights) : work.weight;
  unsigned* const equals = chunks <= kList ? sh.counts : work.equal;
  const bool ranked = quarters <= kMostQuarters;
  const unsigned* const most = ranked ? sh.most : work.most;
  if (PHASE == Phase::kFirst && tid == 0)
    state->status = RowState::kDone;

  if constexpr (PHASE == Phase::kPick) {
    __syncthreads();
    if (wave == 0)
      Pick<T>(p, row, chunks, work.weight, work.equal, s,
              WeigherOf(sh.powers, state->best, s.temperature), state->t, state->need, 0.0);
    return;
  }
  unsigned best = 0;
  for (int i = tid; i < quarters; i += kGroup) {
    const unsigned m = work.most[i];
    if (ranked)
      sh.most[i] = m;
    best = max(best, m);
  }
  best = RowJoin<kGroupWaves>(WaveMaxKey(best), sh.slots, [](unsigned a, unsigned b) { return max(a, b); });
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (tid == 0)
      p.tokens[row] = -1;
    return;
  }
  if (s.greedy) {
    unsigned first = ~0u;
    for (int i = tid; i < quarters && first == ~0u; i += kGroup)
      if (most[i] == best)
        first = i;
    first = RowJoin<kGroupWaves>(WaveMinKey(first), sh.slots,
                    [](unsigned a, unsigned b) { return min(a, b); });
    if (wave == 0) {
      unsigned key[kRun];
      LoadKeys<T>(p, row, static_cast<int>(first), key);
      unsigned token = ~0u;
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i)
        token = key[i] == best ? RunStart(static_cast<int>(first), p.vocab) + i : token;
      token = WaveMinKey(token);
      if (lane == 0)
        p.tokens[row] = static_cast<int>(token);
    }
    return;
  }

  const Weigher w = WeigherOf(sh.powers, best, s.temperature);
  const bool share = s.top_p < 1.0F;
  // The whole row's weight, where the first launch left the chunks'.
  double all = 0.0;
  if (s.top_k == 0) {
    for (int i = tid; i < chunks; i += kGroup) {
      unsigned top = 0;
      for (int q = i * kQuarters; q < min((i + 1) * kQuarters, quarters); ++q)
        top = max(top, most[q]);
      const double sum = work.weight[i] * w(top);
      weights[i] = sum;
      all += sum;
    }
    all = RowJoin<kGroupWaves>(WaveSum64(all), sh.slots, [](double a, double b) { return a + b; });
  }
  if (PHASE == Phase::kPlain || (s.top_k == 0 && !share && !(s.min_p > 0.0F))) {
    __threadfence_block();
    __syncthreads();
    if (wave == 0)
      Pick<T>(p, row, chunks, weights, equals, s, w, 0, 0, all);
    return;
  }

  if constexpr (PHASE != Phase::kPlain && PHASE != Phase::kPick) {
    Kept kept{1, kAll, 0};
    Source from{false, 0};
    bool known = s.top_k == 0 && !share;  // min_p says the threshold itself
    if (known)
      kept.t = KeyOfShare(w, best, s.min_p);
    const int opened = s.top_k > 0 ? s.top_k : kShareOpened;
    if (PHASE != Phase::kSearch && ranked && (known || (opened <= kMostOpened && opened <= quarters))) {
      unsigned floor = kept.t;
      if (!known) {
        // What reaches the last of the loudest quarters.
        Held<8> loud;  // of up to 262144 tokens; every wave by itself
        loud.used = min((quarters + kWave - 1) / kWave, 8);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          loud.key[i] = i * kWave + lane < quarters ? sh.most[i * kWave + lane] : 0;
        floor = Held<8>::Search(1, best, [&](unsigned t) {
          int n = loud.Count(t);
          for (int i = 8 * kWave; i < quarters; i += kWave)
            n += __popcll(__ballot(i + lane < quarters && sh.most[i + lane] >= t));
          return n >= opened;
        });
      }
      const bool fits = Gather<T>(p, row, quarters, sh, most, floor, best);
      const int listed = static_cast<int>(sh.listed);
      if (listed <= kShortList && DrawFromList(p, row, sh, listed, s, w, shift, all))
        return;
      if (fits && (known || s.top_k > 0))
        from = Source{true, listed};
    }
    if (PHASE == Phase::kFirst && !from.list) {
      // The row's passes are the next launches.
      if (tid == 0) {
        state->status = known ? RowState::kPick : RowState::kSearch;
        state->best = best;
        state->t = kept.t;
        state->need = kept.need;
      }
      return;
    }

    if (!known) {
      const RowState* const sums =
          PHASE == Phase::kSearch && s.Searches(quarters) ? state : nullptr;
      u64 whole = s.top_k == 0 ? static_cast<u64>(ldexp(all, shift)) : 0;
      if (s.top_k > 0) {
        RowSearch<T, false>(p, row, chunks, quarters, most, sh, &from, sums, w, shift, best, 1,
                            s.top_k);
        kept.t = sh.t;
        kept.need = s.top_k - sh.above_count;  // of those that there are
        if (share) {
          // The weight of what top_k keeps.
          u64 sum = 0, equal = 0;
          EachKey<T>(p, row, chunks, sh, from, [&](unsigned key, int) {
            if (key > kept.t)
              sum += UnitsOf(w(key), shift);
            equal += key == kept.t;
          });
          const auto add = [](u64 a, u64 b) { return a + b; };
          whole = RowJoin(WaveSum64(sum), sh.slots, add);
          kept.need = min(kept.need, RowJoin(WaveSum64(equal), sh.slots, add));
          whole += kept.need * UnitsOf(w(kept.t), shift);
        }
      }
      if (share) {
        const u64 want = ShareOf(s.top_p, whole);
        RowSearch<T, true>(p, row, chunks, quarters, most, sh, &from, sums, w, shift, best, kept.t,
                           want);
        const u64 each = UnitsOf(w(sh.t), shift);
        const u64 need = each > 0 && want > sh.above_weight
                             ? (want - sh.above_weight + each - 1) / each
                             : kAll;
        kept.need = sh.t > kept.t ? need : min(kept.need, need);
        kept.t = max(sh.t, kept.t);
      }
      if (s.min_p > 0.0F) {
        const unsigned t = KeyOfShare(w, best, s.min_p);
        if (t > kept.t) {
          kept.t = t;
          kept.need = kAll;
        }
      }
    }
    // The chunks' kept weights.
    __syncthreads();
    if (from.list && chunks <= kList) {
      for (int i = tid; i < chunks; i += kRowThreads) {
        sh.weights[i] = 0;
        equals[i] = 0;
      }
      __syncthreads();
      EachKey<T>(p, row, chunks, sh, from, [&](unsigned key, int index) {
        if (key > kept.t)
          atomicAdd(&sh.weights[index / kChunk], UnitsOf(w(key), shift));
        else if (key == kept.t)
          atomicAdd(&equals[index / kChunk], 1u);
      });
      __syncthreads();
      for (int i = tid; i < chunks; i += kRowThreads)
        weights[i] = ldexp(static_cast<double>(sh.weights[i]), -shift);
    } else if (PHASE == Phase::kSearch) {
      if (tid == 0) {
        state->status = RowState::kPick;
        state->t = kept.t;
        state->need = kept.need;
      }
      return;
    } else {
      for (int c = wave; c < chunks; c += kRowWaves)
        KeptOfChunk<T>(p, row, c, kept.t, w, weights + c, equals + c);
    }
    if (PHASE == Phase::kSearch && tid == 0)
      state->status = RowState::kDone;
    __threadfence_block();
    __syncthreads();
    if (wave == 0)
      Pick<T>(p, row, chunks, weights, equals, s, w, kept.t, kept.need, 0.0);
  }
}

// The chunks' kept weights of the rows that have their threshold.
template <typename T>
__global__ __launch_bounds__(kThreads) void KeptKernel(SampleParams p, int chunks, int groups) {
  __shared__ double powers[kTable];
  __builtin_assume(p.vocab > kChunk);
  const int row = blockIdx.x / groups;
  const RowState* const state = StateOf(p, row, chunks);
  if (state->status != RowState::kPick)
    return;
  const Settings s = SettingsOf(p, row);
  const Work work = WorkOf(p, row, chunks);
  FillTable(powers);
  __syncthreads();
  const int c = (blockIdx.x - row * groups) * kWaves + threadIdx.x / kWave;
  if (c < chunks)
    KeptOfChunk<T>(p, row, c, state->t, WeigherOf(powers, state->best, s.temperature),
                   work.weight + c, work.equal + c);
}

// Whether the rows' passes are launches of their own: where the rows do not fill the
// device by themselves.
bool SplitRows(std::int64_t rows, std::int64_t chunks) {
  return rows <= kSplitRows && chunks <= kList;
}

int ChunksOf(int vocab) { return vocab <= kChunk ? 0 : (vocab - 1) / kChunk + 1; }

}  // namespace

std::int64_t SampleWorkBytes(std::int64_t rows, std::int64_t vocab) {
  const std::int64_t chunks = ChunksOf(static_cast<int>(vocab));
  if (chunks == 0)
    return 0;
  return rows * (WorkWords(chunks) * static_cast<std::int64_t>(sizeof(unsigned)) +
                 (SplitRows(rows, chunks) ? static_cast<std::int64_t>(sizeof(RowState)) : 0));
}

void LaunchSample(const SampleParams& p, DType type, hipStream_t stream) {
  Require(p.rows >= 1 && p.vocab >= 1, "sample: empty shape");
  int bits = 0;
  while ((std::int64_t{1} << bits) < p.vocab)
    ++bits;
  const int shift = 62 - bits < 51 ? 62 - bits : 51;
  const int chunks = ChunksOf(p.vocab);
  const int groups = (chunks + kWaves - 1) / kWaves;
  Require(static_cast<std::int64_t>(p.rows) * groups < (1 << 23), "rows times vocab too large");
  const int quarters = (p.vocab + kQuarter - 1) / kQuarter;
  WithType(type, [&](auto t) {
    using T = decltype(t);
    const auto small = [&](auto q) {
      Dispatch(SmallKernel<T, q()>, dim3((p.rows + kWaves - 1) / kWaves), dim3(kThreads), 0,
               stream, true, true, p, shift);
    };
    if (quarters == 1) {
      small(std::integral_constant<int, 1>());
    } else if (quarters == 2) {
      small(std::integral_constant<int, 2>());
    } else if (quarters == 3) {
      small(std::integral_constant<int, 3>());
    } else if (quarters <= kQuarters && chunks == 0) {
      small(std::integral_constant<int, kQuarters>());
    } else {
      // A row may need a threshold where any setting may ask for one.
      const bool filtered = p.top_ks != nullptr || p.top_ps != nullptr || p.min_ps != nullptr ||
                            p.top_k > 0 || p.top_p < 1.0F || p.min_p > 0.0F;
      // Where every row has one small k its list is short, but for many equals.
      const bool listed = p.top_ks == nullptr && p.top_k > 0 && p.top_k <= kMostOpened &&
                          p.top_k <= quarters;
      const bool split = filtered && !listed && SplitRows(p.rows, chunks);
      Dispatch(ChunkKernel<T>, dim3(p.rows * groups), dim3(kThreads), 0, stream, true, false, p,
               chunks, groups, split);
      const auto rows = [&](auto kernel, int groups_each, int threads, bool last) {
        Dispatch(kernel, dim3(p.rows * groups_each), dim3(threads), 0, stream, false, last, p,
                 chunks, quarters, shift);
      };
      if (!filtered) {
        rows(RowKernel<T, Phase::kPlain>, 1, kThreads, true);
      } else if (!split) {
        rows(RowKernel<T, Phase::kWhole>, 1, kRowThreads, true);
      } else {
        rows(RowKernel<T, Phase::kFirst>, 1 + (chunks + kStepChunks - 1) / kStepChunks,
             kRowThreads, false);
        rows(RowKernel<T, Phase::kSearch>, 1, kRowThreads, false);
        Dispatch(KeptKernel<T>, dim3(p.rows * groups), dim3(kThreads), 0, stream, false, false, p,
                 chunks, groups);
        rows(RowKernel<T, Phase::kPick>, 1, kWave, true);
      }
    }
  });
  Check(hipGetLastError(), "sample launch");
}

}  // namespace ovg
