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
// for top_p alone) and selects among the few elements that reach the last one's. Where
// that is not enough (a large k, a share that needs more) it reads the row again: three
// passes over 11, 11 and 10 bits of the keys with sums in LDS, and one for the chunks'
// kept weights.
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
constexpr int kRowThreads = 512;            // of a row's work-group in the second launch
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kMostQuarters = 2048;         // that are ranked
constexpr int kMostOpened = 256;            // quarters that are read for a list
constexpr int kList = 512;                  // elements of it
constexpr int kShareOpened = 64;            // opened for a share alone
constexpr double kLeast = -50.0;            // log2 of the smallest weight that counts
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
// The lanes' sums up to and with themselves.
template <typename V>
__device__ __forceinline__ V WaveScan(V v) {
  const int lane = threadIdx.x % kWave;
  for (int offset = 1; offset < kWave; offset *= 2) {
    const V before = __shfl_up(v, offset);
    v = lane >= offset ? v + before : v;
  }
  return v;
}

// ---------------------------------------------------------------- keys
// Keys order logits as unsigned numbers; 0 is what cannot be drawn.
constexpr unsigned kKeyOfInf = 0xFF800000u;  // and NaN from here on
constexpr unsigned kKeyOfMinusInf = 0x007FFFFFu;
__device__ __forceinline__ unsigned KeyOf(float z) {
  if (z != z)
    return ~0u;
  const unsigned bits = __float_as_uint(z + 0.0F);  // one zero
  const unsigned key = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return key <= kKeyOfMinusInf ? 0 : key;
}
__device__ __forceinline__ float LogitOf(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// The lane's run of keys at d .. d + 7: 0 before `d` where the row's end moved the run
// forward (RunStart), and for the masked token.
__device__ __forceinline__ int RunStart(int d, int vocab) {
  return vocab >= kRun ? min(d, vocab - kRun) : 0;
}
template <typename T>
__device__ __forceinline__ void LoadRun(const T* row, int d, int vocab, float (&v)[kRun]) {
  if (vocab >= kRun) {
    LoadFloats<kRun>(row + RunStart(d, vocab), v);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      v[i] = i < vocab ? static_cast<float>(row[i]) : 0.0F;
  }
}
template <typename T>
__device__ __forceinline__ void LoadKeys(const SampleParams& p, std::int64_t row, int d,
                                         unsigned (&key)[kRun]) {
  float c[kRun], u[kRun];
  LoadRun(static_cast<const T*>(p.logits) + row * p.stride, d, p.vocab, c);
  if (p.uncond != nullptr) {
    LoadRun(static_cast<const T*>(p.uncond) + row * p.uncond_stride, d, p.vocab, u);
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      c[i] = c[i] == -__builtin_inff() ? c[i] : c[i] + p.guidance * (c[i] - u[i]);
  }
  const int start = RunStart(d, p.vocab);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int e = start + i;
    key[i] = e >= d && e < p.vocab && e != p.mask_id ? KeyOf(c[i]) : 0;
  }
}

// ---------------------------------------------------------------- weights
// powers[j] = 2^(j / 256), by the series of e^x.
__device__ __forceinline__ void FillTable(double* powers) {
  for (int j = threadIdx.x; j < kTable; j += blockDim.x) {
    const double x = j * (0.69314718055994530942 / kTable);
    double e = 1.0;
    for (int n = 18; n > 0; --n)
      e = 1.0 + e * x / n;
    powers[j] = e;
  }
}

struct Weigher {
  const double* powers;  // in LDS
  double top, per;       // the largest logit; 256 log2(e) / T
  // 2^((z - top) per / 256): the table's power times three terms of the rest, which is
  // under ln 2 / 512, so that 1.4e-13 is left out.
  __device__ __forceinline__ double operator()(unsigned key) const {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: whole numbers behind it
    constexpr double kA = 0.69314718055994530942 / kTable;
    const double t = (static_cast<double>(LogitOf(key)) - top) * per;
    const double y = t + kMagic;
    const int k = static_cast<int>(__builtin_bit_cast(u64, y));
    const double r = t - (y - kMagic);
    double e = __fma_rn(r, kA * kA * kA / 6, kA * kA / 2);
    e = __fma_rn(r, e, kA);
    e = __fma_rn(r, e, 1.0);
    e *= powers[k & (kTable - 1)];
    u64 bits = __builtin_bit_cast(u64, e);
    bits += static_cast<u64>(static_cast<unsigned>(k >> 8) << 20) << 32;
    return key != 0 && t >= kLeast * kTable ? __builtin_bit_cast(double, bits) : 0.0;
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

// ---------------------------------------------------------------- small rows
// A wave a row of up to 512 Q tokens.
template <typename T, int Q>
__global__ __launch_bounds__(kThreads) void SmallKernel(SampleParams p, int shift) {
  constexpr int N = Q * kRun;
  __shared__ double powers[kTable];
  FillTable(powers);
  const int lane = threadIdx.x % kWave;
  const int row = blockIdx.x * kWaves + threadIdx.x / kWave;
  Held<N> held;
  held.used = N;
  Settings s{};
  if (row < p.rows) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      unsigned key[kRun];
      LoadKeys<T>(p, row, (q * kWave + lane) * kRun, key);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        held.key[q * kRun + i] = key[i];
    }
  }
  __syncthreads();
  if (row >= p.rows)
    return;
  unsigned best = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    best = max(best, held.key[i]);
  best = WaveMaxKey(best);
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (lane == 0)
      p.tokens[row] = -1;
    return;
  }
  const Weigher w = WeigherOf(powers, best, s.greedy ? 1.0F : s.temperature);
  Kept kept{best, 1, 1};
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
  // In the order of the row: quarters, lanes, elements.
  u64 left = TargetOf(s.greedy ? 0.0F : s.u, kept.weight);
  u64 need = kept.need;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const auto run = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        f(i, held.key[q * kRun + i], held.weight[q * kRun + i]);
    };
    u64 equal = 0;
    run([&](int, unsigned key, u64) { equal += key == kept.t; });
    const u64 equal_to = WaveScan(static_cast<unsigned>(equal));
    u64 before = equal_to - equal, mine = 0, seen = before;
    run([&](int, unsigned key, u64 weight) {
      mine += key > kept.t || (key == kept.t && seen++ < need) ? weight : 0;
    });
    const u64 to = WaveScan(mine);
    const u64 hit = __ballot(to > left);
    if (hit != 0) {
      if (lane == __builtin_ctzll(hit)) {
        u64 at = to - mine;
        int token = -1;
        const int start = RunStart((q * kWave + lane) * kRun, p.vocab);
        run([&](int i, unsigned key, u64 weight) {
          at += key > kept.t || (key == kept.t && before++ < need) ? weight : 0;
          if (token < 0 && at > left)
            token = start + i;
        });
        p.tokens[row] = token;
      }
      return;
    }
    left -= Lane64(to, kWave - 1);
    const u64 equals = __builtin_amdgcn_readlane(static_cast<int>(equal_to), kWave - 1);
    need -= min(need, equals);
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
__device__ __forceinline__ Work WorkOf(const SampleParams& p, int row, int chunks) {
  const std::size_t each = static_cast<std::size_t>(chunks) * (2 + 1 + kQuarters);
  double* const base = reinterpret_cast<double*>(p.work + (each + (each & 1)) * row);
  unsigned* const equal = reinterpret_cast<unsigned*>(base + chunks);
  return {base, equal, equal + chunks};
}

// The largest key of every quarter of a chunk, and the chunk's weight beside the
// chunk's own largest.
template <typename T>
__global__ __launch_bounds__(kThreads) void ChunkKernel(SampleParams p, int chunks, int groups) {
  __shared__ double powers[kTable];
  FillTable(powers);
  const int lane = threadIdx.x % kWave;
  const int row = blockIdx.x / groups;
  const int chunk = (blockIdx.x - row * groups) * kWaves + threadIdx.x / kWave;
  unsigned key[kQuarters][kRun];
  Settings s{};
  if (chunk < chunks) {
    s = SettingsOf(p, row);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
      LoadKeys<T>(p, row, chunk * kChunk + (q * kWave + lane) * kRun, key[q]);
  }
  __syncthreads();
  if (chunk >= chunks)
    return;
  const Work work = WorkOf(p, row, chunks);
  unsigned best = 0;
#pragma unroll
  for (int q = 0; q < kQuarters; ++q) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      most = max(most, key[q][i]);
    most = WaveMaxKey(most);
    if (lane == 0)
      work.most[chunk * kQuarters + q] = most;
    best = max(best, most);
  }
  if (!s.Whole() || best >= kKeyOfInf)
    return;
  double sum = 0.0;
  if (best != 0) {
    const Weigher w = WeigherOf(powers, best, s.temperature);
#pragma unroll
    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        sum += w(key[q][i]);
  }
  sum = WaveSum64(sum);
  if (lane == 0)
    work.weight[chunk] = sum;
}

struct RowShared {
  double powers[kTable];
  u64 weights[2048];      // of a pass's bins
  unsigned counts[2048];
  unsigned most[kMostQuarters];
  u64 list[kList];        // index, key
  u64 slots[kRowWaves];
  double sums[kRowWaves];
  unsigned listed;
  Kept kept;
  int mode;
  unsigned t;
  u64 above_weight, above_count;
};

template <typename V, typename F>
__device__ __forceinline__ V RowJoin(V v, V* slots, F&& join) {
  // v is the same in every lane of a wave
  __syncthreads();
  if (threadIdx.x % kWave == 0)
    slots[threadIdx.x / kWave] = v;
  __syncthreads();
  v = slots[0];
  for (int i = 1; i < kRowWaves; ++i)
    v = join(v, slots[i]);
  return v;
}

// Calls f(key, index) for every element of the row, a wave a quarter.
template <typename T, typename F>
__device__ __forceinline__ void EachKey(const SampleParams& p, int row, int quarters, F&& f) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  for (int q = wave; q < quarters; q += kRowWaves) {
    const int d = (q * kWave + lane) * kRun;
    unsigned key[kRun];
    LoadKeys<T>(p, row, d, key);
    const int start = RunStart(d, p.vocab);
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      f(key[i], start + i);
  }
}

// The threshold at which the keys' count (or their weight) reaches `want`, by three
// passes over the row: sums of 2048 bins of the keys that share the bits found so far.
// Below `floor` nothing counts. The whole work-group calls this.
template <typename T, bool WEIGHT>
__device__ __forceinline__ void RowSearch(const SampleParams& p, int row, int quarters,
                                          RowShared& sh, const Weigher& w, int shift,
                                          unsigned floor, u64 want) {
  const int tid = threadIdx.x;
  unsigned prefix = 0;
  u64 above_weight = 0, above_count = 0;
  for (int level = 0; level < 3; ++level) {
    const int low = level == 0 ? 21 : level == 1 ? 10 : 0;
    const int bins = level == 2 ? 1024 : 2048;
    const int high = low + (level == 2 ? 10 : 11);  // bits of the prefix begin here
    for (int i = tid; i < 2048; i += kRowThreads) {
      sh.weights[i] = 0;
      sh.counts[i] = 0;
    }
    __syncthreads();
    EachKey<T>(p, row, quarters, [&](unsigned key, int) {
      if (key >= floor && (level == 0 || key >> high == prefix >> high)) {
        const int bin = (key >> low) & (bins - 1);
        atomicAdd(&sh.counts[bin], 1u);
        if constexpr (WEIGHT)
          atomicAdd(&sh.weights[bin], UnitsOf(w(key), shift));
      }
    });
    __syncthreads();
    // The first wave sums from the top, 32 bins a lane (16 in the last pass).
    if (tid < kWave) {
      const int each = bins / kWave, top = bins - 1 - tid * each;
      u64 weight = 0, count = 0;
      for (int i = 0; i < each; ++i) {
        weight += sh.weights[top - i];
        count += sh.counts[top - i];
      }
      const u64 weight_to = WaveScan(weight), count_to = WaveScan(count);
      const u64 at = WEIGHT ? above_weight + weight_to : above_count + count_to;
      const u64 hit = __ballot(at >= want);
      // Fixed-point shares round up to what there is, so some lane is hit; the last one
      // takes what rounding leaves.
      const int owner = hit != 0 ? __builtin_ctzll(hit) : kWave - 1;
      if (tid == owner) {
        u64 aw = above_weight + weight_to - weight, ac = above_count + count_to - count;
        int bin = top;
        for (int i = 0; i < each - 1; ++i, --bin) {
          const u64 next = WEIGHT ? aw + sh.weights[bin] : ac + sh.counts[bin];
          if (next >= want)
            break;
          aw += sh.weights[bin];
          ac += sh.counts[bin];
        }
        sh.t = prefix | static_cast<unsigned>(bin) << low;
        sh.above_weight = aw;
        sh.above_count = ac;
      }
    }
    __syncthreads();
    prefix = sh.t;
    above_weight = sh.above_weight;
    above_count = sh.above_count;
  }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void RowKernel(SampleParams p, int chunks, int quarters,
                                                         int row_shift) {
  __shared__ RowShared sh;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int row = blockIdx.x;
  const Settings s = SettingsOf(p, row);
  const Work work = WorkOf(p, row, chunks);
  FillTable(sh.powers);
  if (tid == 0)
    sh.listed = 0;

  unsigned best = 0;
  for (int i = tid; i < quarters; i += kRowThreads) {
    const unsigned most = work.most[i];
    if (i < kMostQuarters)
      sh.most[i] = most;
    best = max(best, most);
  }
  best = static_cast<unsigned>(RowJoin(static_cast<u64>(WaveMaxKey(best)), sh.slots,
                                       [](u64 a, u64 b) { return a > b ? a : b; }));
  if (best == 0 || best >= kKeyOfInf || s.lost) {
    if (tid == 0)
      p.tokens[row] = -1;
    return;
  }
  if (s.greedy) {
    u64 first = ~u64{0};
    for (int i = tid; i < quarters && first == ~u64{0}; i += kRowThreads)
      if (work.most[i] == best)
        first = i;
    first = WaveMinKey(static_cast<unsigned>(min(first, u64{0xFFFFFFFFu})));
    first = RowJoin(first, sh.slots, [](u64 a, u64 b) { return min(a, b); });
    if (wave == 0) {
      const int d = (static_cast<int>(first) * kWave + lane) * kRun;
      unsigned key[kRun];
      LoadKeys<T>(p, row, d, key);
      int token = 0x7FFFFFFF;
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i)
        token = key[i] == best ? RunStart(d, p.vocab) + i : token;
      token = static_cast<int>(WaveMinKey(static_cast<unsigned>(token)));
      if (lane == 0)
        p.tokens[row] = token;
    }
    return;
  }

  const Weigher w = WeigherOf(sh.powers, best, s.temperature);
  const bool share = s.top_p < 1.0F;
  // The whole row's weight, where the first launch left the chunks'.
  double all = 0.0;
  if (s.top_k == 0) {
    for (int i = tid; i < chunks; i += kRowThreads) {
      const unsigned* most = work.most + i * kQuarters;
      unsigned top = 0;
      for (int q = 0; q < kQuarters; ++q)
        top = max(top, i * kQuarters + q < quarters ? most[q] : 0);
      const double sum = work.weight[i] * w(top);
      work.weight[i] = sum;
      all += sum;
    }
    all = RowJoin(WaveSum64(all), sh.sums, [](double a, double b) { return a + b; });
  }

  Kept kept{1, kAll, 0};
  bool chunked = s.top_k == 0 && !share && !(s.min_p > 0.0F);  // the chunks' weights are it
  const bool ranked = quarters <= kMostQuarters;
  const int opened = s.top_k > 0 ? s.top_k : kShareOpened;
  if (!chunked && ranked && (s.top_k > 0 || share) && opened <= kMostOpened &&
      opened <= quarters) {
    // The list: what reaches the last of the loudest quarters.
    unsigned floor = 0;
    {
      int n = 0;
      unsigned low = 1, high = best;
      while (low < high) {  // every wave by itself
        const unsigned mid = low + (high - low + 1) / 2;
        n = 0;
        for (int i = 0; i < quarters; i += kWave)
          n += __popcll(__ballot(i + lane < quarters && sh.most[i + lane] >= mid));
        if (n >= opened)
          low = mid;
        else
          high = mid - 1;
      }
      floor = low;
    }
    for (int q = wave; q < quarters; q += kRowWaves) {
      if (sh.most[q] < floor)
        continue;
      const int d = (q * kWave + lane) * kRun;
      unsigned key[kRun];
      LoadKeys<T>(p, row, d, key);
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (key[i] >= floor) {
          const unsigned at = atomicAdd(&sh.listed, 1u);
          if (at < kList)
            sh.list[at] = static_cast<u64>(key[i]) << 32 |
                          static_cast<unsigned>(RunStart(d, p.vocab) + i);
        }
    }
    __syncthreads();
    const int listed = static_cast<int>(sh.listed);
    if (listed <= kList) {
      if (wave == 0) {
        constexpr int N = kList / kWave;
        // Few elements are finer units, where the list is all that counts.
        const int shift = s.top_k > 0 ? 51 : row_shift;
        Held<N> held;
        unsigned index[N];
        held.used = (listed + kWave - 1) / kWave;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int at = i * kWave + lane;
          const u64 e = at < listed ? sh.list[at] : 0;
          held.key[i] = static_cast<unsigned>(e >> 32);
          index[i] = static_cast<unsigned>(e);
          held.weight[i] = UnitsOf(w(held.key[i]), shift);
        }
        const u64 whole = static_cast<u64>(ldexp(all, shift));
        Kept k;
        const bool done = held.Select(s, w, best, shift, s.top_k > 0 ? nullptr : &whole, &k);
        if (lane == 0) {
          sh.mode = done;
          sh.kept = k;
        }
        if (done) {
          // The equals that are kept are those up to some index, and so is the draw.
          const auto up_to = [&](auto&& value) {
            unsigned low = 0, high = p.vocab - 1;  // the first index that reaches
            while (low < high) {
              const unsigned mid = (low + high) / 2;
              if (value(mid))
                high = mid;
              else
                low = mid + 1;
            }
            return low;
          };
          unsigned last = p.vocab;
          if (k.need != kAll)
            last = up_to([&](unsigned m) {
              u64 n = 0;
#pragma unroll
              for (int i = 0; i < N; ++i)
                n += __popcll(__ballot(held.key[i] == k.t && index[i] <= m));
              return n >= k.need;
            });
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (!(held.key[i] > k.t || (held.key[i] == k.t && index[i] <= last)))
              held.weight[i] = 0;
          const u64 target = TargetOf(s.u, k.weight);
          const unsigned token = up_to([&](unsigned m) {
            u64 n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
              n += index[i] <= m ? held.weight[i] : 0;
            return WaveSum64(n) > target;
          });
          if (lane == 0)
            p.tokens[row] = static_cast<int>(token);
        }
      }
      __syncthreads();
      if (sh.mode)
        return;
    }
  }

  const int shift = row_shift;
  if (!chunked) {
    // The thresholds from passes over the row.
    u64 whole = s.top_k == 0 ? static_cast<u64>(ldexp(all, shift)) : 0;
    if (s.top_k > 0) {
      RowSearch<T, false>(p, row, quarters, sh, w, shift, 1, s.top_k);
      if (sh.t != 0) {
        kept.t = sh.t;
        kept.need = s.top_k - sh.above_count;
      }
    }
    if (share) {
      if (s.top_k > 0) {
        // The weight of what top_k keeps.
        u64 sum = 0;
        EachKey<T>(p, row, quarters, [&](unsigned key, int) {
          sum += key > kept.t ? UnitsOf(w(key), shift) : 0;
        });
        whole = RowJoin(WaveSum64(sum), sh.slots, [](u64 a, u64 b) { return a + b; }) +
                kept.need * UnitsOf(w(kept.t), shift);
      }
      const u64 want = ShareOf(s.top_p, whole);
      __syncthreads();
      RowSearch<T, true>(p, row, quarters, sh, w, shift, kept.t, want);
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
    // The chunks' kept weights: above the threshold, and how many equal it.
    __syncthreads();
    for (int c = wave; c < chunks; c += kRowWaves) {
      double sum = 0.0;
      unsigned equal = 0;
      for (int q = 0; q < kQuarters; ++q) {
        if (work.most[c * kQuarters + q] < kept.t)
          continue;
        unsigned key[kRun];
        LoadKeys<T>(p, row, c * kChunk + (q * kWave + lane) * kRun, key);
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          if (key[i] > kept.t)
            sum += w(key[i]);
          equal += key[i] == kept.t;
        }
      }
      sum = WaveSum64(sum);
      const u64 equals = WaveSum64(static_cast<u64>(equal));
      if (lane == 0) {
        work.weight[c] = sum;
        work.equal[c] = static_cast<unsigned>(equals);
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  if (wave != 0)
    return;
  // The first wave finds the chunk, 64 at a time, then the place in it.
  const double each = chunked ? 0.0 : w(kept.t);
  u64 need = chunked ? 0 : kept.need;
  const auto chunk_weight = [&](int c, u64* equal_before) {
    // Of chunk c (lanes' own, neighbouring ones), with the equals kept before it.
    const bool there = c < chunks;
    const unsigned equal = there && !chunked ? work.equal[c] : 0;
    const u64 to = WaveScan(static_cast<u64>(equal));
    *equal_before = to;
    const u64 before = to - equal;
    const u64 kept_equal = need > before ? min(need - before, static_cast<u64>(equal)) : 0;
    return (there ? work.weight[c] : 0.0) + static_cast<double>(kept_equal) * each;
  };
  double total = 0.0;
  for (int c0 = 0; c0 < chunks; c0 += kWave) {
    u64 equal_to;
    total += WaveSum64(chunk_weight(c0 + lane, &equal_to));
    need -= min(need, Lane64(equal_to, kWave - 1));
  }
  const double u = fminf(fmaxf(s.u, 0.0F), 1.0F);
  double left = u * total;
  if (!(left < total))
    left = total * (1.0 - 0x1p-53);
  need = chunked ? 0 : kept.need;
  bool done = false;
  double before = 0.0;
  int last = 0;  // the chunk; the last one that keeps any where rounding leaves none
  double last_before = 0.0;
  u64 last_need = 0;
  for (int c0 = 0; c0 < chunks && !done; c0 += kWave) {
    u64 equal_to;
    const double mine = chunk_weight(c0 + lane, &equal_to);
    const double to = before + WaveScan(mine);
    const u64 hit = __ballot(mine > 0.0 && to > left);
    const u64 any = __ballot(mine > 0.0);
    const u64 equal_before =
        equal_to - (c0 + lane < chunks && !chunked ? work.equal[c0 + lane] : 0);
    if (any != 0) {
      const int l = hit != 0 ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
      last = c0 + l;
      last_before = __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, to - mine), l));
      last_need = need - min(need, Lane64(equal_before, l));
    }
    done = hit != 0;
    before = __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, to), kWave - 1));
    need -= min(need, Lane64(equal_to, kWave - 1));
  }
  left -= last_before;
  need = last_need;
  int token = -1, most = -1;  // the last kept one, where rounding leaves none
  for (int q = 0; q < kQuarters && token < 0; ++q) {
    const int d = last * kChunk + (q * kWave + lane) * kRun;
    unsigned key[kRun];
    LoadKeys<T>(p, row, d, key);
    unsigned equal = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      equal += !chunked && key[i] == kept.t;
    const unsigned equal_to = WaveScan(equal);
    u64 seen = equal_to - equal;
    double weight[kRun], mine = 0.0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const bool in = chunked || key[i] > kept.t || (key[i] == kept.t && seen++ < need);
      weight[i] = in ? w(key[i]) : 0.0;
      mine += weight[i];
    }
    const double to = WaveScan(mine);
    const u64 hit = __ballot(mine > 0.0 && to > left);
    const u64 any = __ballot(mine > 0.0);
    const int owner = hit != 0 ? __builtin_ctzll(hit) : any != 0 ? 63 - __builtin_clzll(any) : -1;
    int place = -1, end = -1;
    double sum = to - mine;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      sum += weight[i];
      end = weight[i] > 0.0 ? i : end;
      place = place < 0 && weight[i] > 0.0 && sum > left ? i : place;
    }
    place = RunStart(d, p.vocab) + (place < 0 ? end : place);
    if (owner >= 0) {
      most = __builtin_amdgcn_readlane(place, owner);
      if (hit != 0)
        token = most;
    }
    left -= __builtin_bit_cast(double, Lane64(__builtin_bit_cast(u64, to), kWave - 1));
    need -= min(need, static_cast<u64>(__builtin_amdgcn_readlane(equal_to, kWave - 1)));
  }
  if (lane == 0)
    p.tokens[row] = token >= 0 ? token : most;
}

int ChunksOf(int vocab) { return vocab <= kChunk ? 0 : (vocab - 1) / kChunk + 1; }

}  // namespace

std::int64_t SampleWorkBytes(std::int64_t rows, std::int64_t vocab) {
  std::int64_t each = ChunksOf(static_cast<int>(vocab)) * std::int64_t{2 + 1 + kQuarters};
  each += each & 1;
  return rows * each * static_cast<std::int64_t>(sizeof(unsigned));
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
    } else if (quarters <= kQuarters && chunks == 0) {
      small(std::integral_constant<int, kQuarters>());
    } else {
      Dispatch(ChunkKernel<T>, dim3(p.rows * groups), dim3(kThreads), 0, stream, true, false, p,
               chunks, groups);
      Dispatch(RowKernel<T>, dim3(p.rows), dim3(kRowThreads), 0, stream, false, true, p, chunks,
               quarters, shift);
    }
  });
  Check(hipGetLastError(), "sample launch");
}

}  // namespace ovg
