// Log probabilities of given tokens with the entropy and the best
// alternatives of their distributions, in one pass over the logits.
//
//   z = c, or c + g (c - u) with unconditional logits, each step rounded to
//   float32 (c = -inf stays -inf, the token being impossible)
//   Z = log sum exp z, log p(token) = z[token] - Z, H = Z - sum p z
//
// A lane keeps the maximum m of what it has seen, s = sum exp(z - m) and
// t = sum exp(z - m) log2 exp(z - m), so that H = log s - ln 2 t / s needs no
// second pass; lanes, waves and splits of a row are joined at the end, in a
// fixed order.
//
// For the alternatives a lane keeps the three loudest of its runs of 16 elements,
// by their largest element, which costs 13 operations a run. The row's `top` best
// elements lie in its `top` loudest runs (equal ones by place: whatever lies in
// another run has the loudest elements of those before it), so at the end a wave
// picks that many runs, fetches them again and ranks the few elements that reach
// the last one's loudest. A lane that has given its three gets the next three from
// its segments, which the wave asks for again. A row of one segment is ranked from
// its registers. Where more than 64 elements reach the value, a higher one is looked
// for by halves (14701 rows of 98 elements, 17 listed: 36 us, 95 without). Only where
// over 64 are equal there, or the rows of the two tensors do not lie alike, does the
// wave search all its elements once more, with a sorted list in its lanes.
//
// Elements come as 16-byte loads, 16 elements in a row to a lane, a segment of 1024
// to a wave; the up to 14 before a row's first 16-byte border and behind its last are
// one more load each of single elements. A row belongs to one wave up to 2048
// elements (four rows to a work-group), else to the four waves of a work-group, and
// where there are too few rows for the device to several of those, whose states a
// second kernel joins.
//
// Bound: memory for large vocabularies, 1000 rows of 151936 bf16 logits (304 MB) 61 us,
// 5.0 TB/s, where a large copy reaches 5.05. For small ones the chain of a wave's
// dependent steps: 2000 guided rows of 1025 float32 logits (16 MB) 8.9 us, of which two
// trips to memory, the joins of 64 lanes and the ranking are 6.
#include <algorithm>

#include "cache.hpp"

#pragma clang fp contract(off)

namespace ovg {
namespace {

constexpr int kWaves = 4;
constexpr int kElements = 16;  // a lane's elements of a segment
constexpr int kSegment = kElements * kWave;
constexpr float kLog2e = 1.44269504088896341F;
constexpr float kLn2 = 0.693147180559945309F;

__device__ __forceinline__ float Inf() { return __builtin_inff(); }

template <int CTRL>
__device__ __forceinline__ int Dpp(int v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ float LaneOf(float v, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Whole numbers in the order of the floats; 0 is below them all. -0 and +0 are one.
__device__ __forceinline__ unsigned OrderOf(float v) {
  const unsigned u = __float_as_uint(v + 0.0F);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ValueOf(unsigned order) {
  if (order == 0)
    return -Inf();
  return __uint_as_float((order & 0x80000000u) != 0 ? order & 0x7FFFFFFFu : ~order);
}

// The wave's maximum of whole numbers: within rows of 16 lanes, then across them.
template <int CTRL>
__device__ __forceinline__ unsigned DppMaxOf(unsigned v) {
  return max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF,
                                                               0xF, true)));
}
__device__ __forceinline__ unsigned WaveMaxOf(unsigned v) {
  v = DppMaxOf<0xB1>(v);
  v = DppMaxOf<0x4E>(v);
  v = DppMaxOf<0x141>(v);
  v = DppMaxOf<0x140>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(max(b[0], b[1]));
}

// The `top` best so far: lane j holds the j-th's order and index, (0, -1) where
// there is none, and what lies behind the last is below it. The last one is kept
// apart, the same in every lane.
struct Alternatives {
  unsigned order;
  int index;
  int top;
  unsigned floor;
  int floor_index;
  __device__ __forceinline__ explicit Alternatives(int top_)
      : order(0), index(-1), top(top_), floor(0), floor_index(-1) {}
  __device__ __forceinline__ bool Takes(unsigned o, int i) const {
    return o > floor || (o == floor && o != 0 && i < floor_index);
  }
  // What it takes, the same in every lane.
  __device__ __forceinline__ void Insert(unsigned o, int i, int lane) {
    const int at = __popcll(__ballot(order > o || (order == o && index < i)));
    const unsigned up = static_cast<unsigned>(Dpp<0x138>(static_cast<int>(order)));
    const int up_index = Dpp<0x138>(index);  // wave_shr: 1
    order = lane == at ? o : lane > at ? up : order;
    index = lane == at ? i : lane > at ? up_index : index;
    floor = __builtin_amdgcn_readlane(order, top - 1);
    floor_index = __builtin_amdgcn_readlane(index, top - 1);
  }
  // Another sorted list, lane k holding its k-th.
  __device__ __forceinline__ void Merge(unsigned o, int i, int lane) {
    for (int k = 0; k < top; ++k) {
      const unsigned one = __builtin_amdgcn_readlane(o, k);
      const int at = __builtin_amdgcn_readlane(i, k);
      if (!Takes(one, at))
        return;  // nor does it take any behind
      Insert(one, at, lane);
    }
  }
};

struct Sums {
  float m, s, t;
  // The same sums relative to another maximum. The difference from a mask of the type's
  // lowest value, or its product with s, would be -infinity, which f, 0 from -150 down,
  // makes a NaN.
  __device__ __forceinline__ void Move(float to) {
    const float d = m == -Inf() ? 0.0F : fmaxf((m - to) * kLog2e, -1000.0F);
    const float f = __builtin_amdgcn_exp2f(d);
    t = (t + s * d) * f;
    s = s * f;
    m = to;
  }
  // The wave's, in every lane.
  __device__ __forceinline__ void JoinWave() {
    const float top = WaveMaxFast(m);
    Move(top == -Inf() ? m : top);
    m = top;
    s = WaveSumFast(s);
    t = WaveSumFast(t);
  }
};

__device__ __forceinline__ float Guide(float c, float u, float g) {
  const float d = c - u;
  const float z = c + g * d;
  return c == -Inf() ? c : z;
}

template <typename T>
struct Row {
  const T* c;
  const T* u;  // null without guidance
  float g;
  __device__ __forceinline__ float At(int i) const {
    const float x = static_cast<float>(c[i]);
    return u == nullptr ? x : Guide(x, static_cast<float>(u[i]), g);
  }
};

// A lane's elements of a segment, -inf for none.
typedef float segment_t __attribute__((ext_vector_type(kElements)));

// Takes the first COUNT of a segment's elements into the list; index_of(e) is the
// e-th's, -1 for one that is not to be listed. peak: the lane's largest.
template <int COUNT, typename F>
__device__ __forceinline__ void Search(const segment_t& z, float peak, F&& index_of,
                                       int lane, Alternatives* best) {
  constexpr float kLowest = -3.402823466e38F;
  unsigned floor = best->floor;
  if (!__any(peak >= fmaxf(ValueOf(floor), kLowest)))
    return;
  if (floor == 0 && COUNT > 1) {
    // The list is not full: the top-th largest of the lanes' own largest stands in.
    // That many elements reach it, so nothing below it is listed.
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < COUNT; ++e)
      mine = z[e] >= kLowest && index_of(e) >= 0 ? max(mine, OrderOf(z[e])) : mine;
    for (int k = 0; k < best->top; ++k) {
      floor = WaveMaxOf(mine);
      if (floor == 0)
        break;
      const unsigned long long have = __ballot(mine == floor);
      mine = lane == __ffsll(have) - 1 ? 0u : mine;
    }
  }
  // A bit for each element that may be listed. Taken one after the other, the list's
  // last value rises; when it turns one away the bits are drawn anew by value and
  // index, so that equal values do not queue.
  const float least = fmaxf(ValueOf(floor), kLowest);
  unsigned bits = 0;
#pragma unroll
  for (int e = 0; e < COUNT; ++e)
    bits |= z[e] >= least && index_of(e) >= 0 ? 1u << e : 0u;
  for (unsigned long long lanes = __ballot(bits != 0); lanes != 0;) {
    const int who = __ffsll(lanes) - 1;
    const int e = __ffs(__builtin_amdgcn_readlane(bits, who)) - 1;
    const unsigned order = OrderOf(LaneOf(z[e], who));
    const int index = __builtin_amdgcn_readlane(index_of(e), who);
    if (best->Takes(order, index)) {
      best->Insert(order, index, lane);
      if (lane == who)
        bits &= bits - 1;
    } else {
      const float last = ValueOf(best->floor);
#pragma unroll
      for (int e2 = 0; e2 < COUNT; ++e2)
        if (!(z[e2] > last || (z[e2] == last && index_of(e2) < best->floor_index)))
          bits &= ~(1u << e2);
    }
    lanes = __ballot(bits != 0);
  }
}

// Takes a segment, of which the lane's largest element is `peak`, into the sums.
template <int COUNT>
__device__ __forceinline__ void Add(const segment_t& z, float peak, Sums* sums) {
  if (peak > sums->m)
    sums->Move(peak);
  const float from = sums->m == -Inf() ? 0.0F : sums->m;
#pragma unroll
  for (int e = 0; e < COUNT; ++e) {
    const float d = (z[e] - from) * kLog2e;
    const float x = __builtin_amdgcn_exp2f(d);
    sums->s += x;
    // 0 * -inf stays 0; a NaN is x's already.
    sums->t = __builtin_fmaf(x, fmaxf(d, -1000.0F), sums->t);
  }
}

__device__ __forceinline__ float Peak(const segment_t& z) {
  float peak = z[0];
#pragma unroll
  for (int e = 1; e < kElements; ++e)
    peak = fmaxf(peak, z[e]);
  return peak;
}

struct Entry {
  unsigned order;
  int index;
};

// Between a wave's own writes to LDS and its reads of what other lanes wrote: LDS
// takes a wave's accesses in order, so only the compiler has to keep theirs.
__device__ __forceinline__ void WaveFence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// An order that `least` to `most` things reach, by halves from `low`, which more
// reach or as many, up to `high`, which none does; count(order), the same in every
// lane, says how many reach one. Where equal ones leave none such, the highest that
// `least` reach.
template <typename F>
__device__ __forceinline__ unsigned Between(unsigned low, unsigned high, int least, int most,
                                            F&& count) {
#pragma unroll 1
  while (high - low > 1) {
    const unsigned middle = low + (high - low) / 2;
    const int reach = count(middle);
    if (reach >= least) {
      low = middle;
      if (reach <= most)
        break;
    } else {
      high = middle;
    }
  }
  return low;
}

// The list of what is in a wave's COUNT elements a lane (index_of(e): -1 for one
// that is not to be listed): those that reach `known` are gathered in `slots` (64,
// the wave's own) and each finds its place by counting the ones before it. known: an
// order that `top` elements at least reach, or less than all; where over 64 reach it,
// one that fewer do is looked for. False where there is none.
template <int COUNT, typename Z, typename F>
__device__ __forceinline__ bool Rank(const Z& z, F&& index_of, unsigned known, int lane,
                                     Entry* slots, Alternatives* best) {
  constexpr float kLowest = -3.402823466e38F;
  int count;
  for (bool again = false;; again = true) {
    const float least = fmaxf(ValueOf(known), kLowest);
    count = 0;
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      const int index = index_of(e);
      const bool in = z[e] >= least && index >= 0;
      const unsigned long long all = __ballot(in);
      if (all == 0)
        continue;
      const int at = count + __builtin_amdgcn_mbcnt_hi(
                                 static_cast<unsigned>(all >> 32),
                                 __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(all), 0));
      if (in && at < kWave)
        slots[at] = {OrderOf(z[e]), index};
      count += __popcll(all);
    }
    if (count <= kWave)
      break;
    if (again)
      return false;
    float peak = z[0];
#pragma unroll
    for (int e = 1; e < COUNT; ++e)
      peak = fmaxf(peak, z[e]);
    known = Between(max(known, OrderOf(kLowest)), WaveMaxOf(OrderOf(peak)) + 1, best->top, kWave,
                    [&](unsigned order) {
                      const float value = ValueOf(order);
                      int n = 0;
#pragma unroll
                      for (int e = 0; e < COUNT; ++e)
                        n += __popcll(__ballot(z[e] >= value && index_of(e) >= 0));
                      return n;
                    });
  }
  WaveFence();
  const Entry own = lane < count ? slots[lane] : Entry{0, -1};
  int before = 0;
  for (int j = 0; j < count; ++j) {
    const unsigned order = __builtin_amdgcn_readlane(own.order, j);
    const int index = __builtin_amdgcn_readlane(own.index, j);
    before += order > own.order || (order == own.order && index < own.index) ? 1 : 0;
  }
  WaveFence();
  if (lane < count)
    slots[before] = own;
  WaveFence();
  const Entry mine = lane < min(count, best->top) ? slots[lane] : Entry{0, -1};
  best->order = mine.order;
  best->index = mine.index;
  best->floor = __builtin_amdgcn_readlane(best->order, max(best->top, 1) - 1);
  best->floor_index = __builtin_amdgcn_readlane(best->index, max(best->top, 1) - 1);
  return true;
}

// A lane's three loudest runs, in order, equal ones by place.
struct Runs {
  float peak[3];
  int segment[3];
  __device__ __forceinline__ Runs()
      : peak{-Inf(), -Inf(), -Inf()}, segment{-1, -1, -1} {}
  __device__ __forceinline__ void Add(float p, int s) {
    const bool a = p > peak[0], b = p > peak[1], c = p > peak[2];
    peak[2] = b ? peak[1] : c ? p : peak[2];
    segment[2] = b ? segment[1] : c ? s : segment[2];
    peak[1] = a ? peak[0] : b ? p : peak[1];
    segment[1] = a ? segment[0] : b ? s : segment[1];
    peak[0] = a ? p : peak[0];
    segment[0] = a ? s : segment[0];
  }
  // The largest three of what the wave's lanes hold, into this lane if `here`.
  __device__ __forceinline__ void Largest(Runs from, bool here) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int segment_of;
      const unsigned largest = from.Pop(&segment_of, nullptr);
      if (here) {
        peak[k] = ValueOf(largest);
        segment[k] = segment_of;
      }
    }
  }
  // Takes the loudest run out of the wave's: its order (0: none), segment and lane.
  __device__ __forceinline__ unsigned Pop(int* of_segment, int* of_lane) {
    const unsigned order = peak[0] > -Inf() ? OrderOf(peak[0]) : 0u;
    const unsigned largest = WaveMaxOf(order);
    *of_segment = -1;
    if (largest == 0)
      return 0;
    unsigned long long have = __ballot(order == largest);
    if ((have & (have - 1)) != 0) {
      const unsigned first =
          ~WaveMaxOf(order == largest ? ~static_cast<unsigned>(segment[0]) : 0u);
      have = __ballot(order == largest && static_cast<unsigned>(segment[0]) == first);
    }
    const int who = __ffsll(have) - 1;
    *of_segment = __builtin_amdgcn_readlane(segment[0], who);
    if (of_lane != nullptr)
      *of_lane = who;
    if (static_cast<int>(threadIdx.x & (kWave - 1)) == who) {
      peak[0] = peak[1];
      segment[0] = segment[1];
      peak[1] = peak[2];
      segment[1] = segment[2];
      peak[2] = -Inf();
    }
    return largest;
  }
  // The wave's `top` loudest runs: lane k gets the k-th's segment (-1: none) and lane.
  // The wave took the segments first, first + stride, ..., `seen` of them; a lane
  // that has given all three it kept gets the next three by peak_of(segment, lane),
  // which each lane calls for other segments. Returns the last one's order, 1 where
  // there are fewer than top.
  template <typename F>
  __device__ __forceinline__ unsigned Pick(int top, int first, int stride, int seen, F&& peak_of,
                                           int lane, int* segment_of, int* lane_of) {
    *segment_of = -1;
    *lane_of = 0;
    int given = 0;
    unsigned last = 1;
    for (int k = 0; k < top; ++k) {
      int s, who = 0;
      const unsigned largest = Pop(&s, &who);
      if (largest == 0)
        return 1;
      last = largest;
      if (lane == k) {
        *segment_of = s;
        *lane_of = who;
      }
      given += lane == who ? 1 : 0;
      if (__builtin_amdgcn_readlane(given, who) == 3 && seen > 3 && k + 1 < top) {
        Runs others;
        for (int i0 = 0; i0 < seen; i0 += kWave) {
          const int at = first + min(i0 + lane, seen - 1) * stride;
          float p = peak_of(at, who);
          for (int j = 0; j <= k; ++j)
            if (__builtin_amdgcn_readlane(*lane_of, j) == who &&
                __builtin_amdgcn_readlane(*segment_of, j) == at)
              p = -Inf();
          others.Add(i0 + lane < seen ? p : -Inf(), at);
        }
        Largest(others, lane == who);
        given = lane == who ? 0 : given;
      }
    }
    return last;
  }
};

// The given token's (guided) logit. Asked for first, so that its two dependent
// loads are over when the sums are.
template <typename T>
__device__ __forceinline__ float Chosen(const LogprobParams& p, std::int64_t row,
                                        const Row<T>& from) {
  if (p.logprob == nullptr)
    return 0.0F;
  const int token = p.tokens[row];
  return token >= 0 && token < p.vocab ? from.At(token) : -Inf();
}

// A row's answers from its whole sums and list.
__device__ __forceinline__ void Answer(const LogprobParams& p, std::int64_t row, float chosen,
                                       const Sums& sums, const Alternatives& best, int lane) {
  // No distribution: a NaN or +infinity among the logits, or nothing above -infinity.
  const bool none = !(sums.s > 0.0F && sums.s < Inf());
  const float log_s = logf(sums.s);
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (p.logprob != nullptr)
      p.logprob[row] = none ? nan : chosen - sums.m - log_s;
    if (p.entropy != nullptr)
      p.entropy[row] = none ? nan : log_s - sums.t / sums.s * kLn2;
  }
  if (lane < p.top) {
    p.top_ids[row * p.top + lane] = none ? -1 : best.index;
    p.top_logprobs[row * p.top + lane] = none ? nan : ValueOf(best.order) - sums.m - log_s;
  }
}

// WAVES waves to a row (1: four rows to a work-group), `splits` work-groups.
template <typename T, bool GUIDED, int WAVES>
__global__ __launch_bounds__(kWaves* kWave) void LogprobKernel(LogprobParams p) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kVecs = kElements / kVec;
  typedef T vec __attribute__((ext_vector_type(kVec)));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::int64_t row =
      WAVES == 1 ? static_cast<std::int64_t>(blockIdx.x) * kWaves + wave : blockIdx.x;
  if (row >= p.rows)
    return;
  Row<T> from;
  from.c = static_cast<const T*>(p.logits) + row * p.stride;
  from.u = GUIDED ? static_cast<const T*>(p.uncond) + row * p.uncond_stride : nullptr;
  from.g = p.guidance;
  Sums sums{-Inf(), 0.0F, 0.0F};
  Alternatives best(p.top);

  // [head, head + body) in 16-byte loads, a whole number of them; both tensors' rows
  // have to lie alike.
  const unsigned lie = static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(from.c)) & 15u;
  const bool alike =
      !GUIDED || (static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(from.u)) & 15u) == lie;
  const int head = min(static_cast<int>((16u - lie) & 15u) / static_cast<int>(sizeof(T)), p.vocab);
  const int body = alike ? (p.vocab - head) / kVec * kVec : 0;
  const int of_row = WAVES == 1 ? 0 : static_cast<int>(blockIdx.y) * WAVES + wave;
  const int waves = WAVES == 1 ? 1 : p.splits * WAVES;
  // What is left, one element a lane in turn: the head and the tail, or all of two
  // rows that do not lie alike. The first 64 of it are asked for here.
  const int left = p.vocab - body;
  const auto left_index = [&](int k) { return k < head ? k : k + body; };
  const int left_first = of_row * kWave + lane;
  const float early = left_first < left ? from.At(left_index(left_first)) : -Inf();
  const bool answers = WAVES == 1 || (wave == 0 && p.splits == 1);
  const float chosen = answers ? Chosen(p, row, from) : 0.0F;

  const auto but_mask = [&](int i) { return i == p.mask_id ? -1 : i; };
  vec c[kVecs], u[kVecs];
  const auto load = [&](int base) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int at = head + min(base + lane * kElements + v * kVec, body - kVec);
      c[v] = *reinterpret_cast<const vec*>(from.c + at);
      if (GUIDED)
        u[v] = *reinterpret_cast<const vec*>(from.u + at);
    }
  };
  // What was loaded, as elements base + 16 lane .. + 15 of the body.
  const auto elements = [&](int base, int of_lane) {
    segment_t z;
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float x = static_cast<float>(c[v][e]);
        z[v * kVec + e] = GUIDED ? Guide(x, static_cast<float>(u[v][e]), p.guidance) : x;
      }
    if (__any(base + kSegment > body)) {
#pragma unroll
      for (int e = 0; e < kElements; ++e)
        z[e] = base + of_lane * kElements + e / kVec * kVec < body ? z[e] : -Inf();
    }
    return z;
  };
  Runs runs;
  int seen = 0;
  segment_t held = segment_t(-Inf());  // one wave's last segment
  if (of_row * kSegment < body)
    load(of_row * kSegment);
#pragma unroll 1
  for (int base = of_row * kSegment; base < body; base += waves * kSegment) {
    const segment_t z = elements(base, lane);
    load(base + waves * kSegment);  // past the end the last ones again
    if constexpr (WAVES == 1)
      held = z;
    const float peak = Peak(z);
    Add<kElements>(z, peak, &sums);
    if (p.top > 0) {
      float listed = peak;
      const int hidden = p.mask_id - head - base;  // of the segment
      if (hidden >= 0 && hidden < kSegment) {
        segment_t others = z;
#pragma unroll
        for (int e = 0; e < kElements; ++e)
          others[e] = hidden == lane * kElements + e ? -Inf() : z[e];
        listed = Peak(others);
      }
      runs.Add(listed, base / kSegment);
      ++seen;
    }
  }
  // What is left, one element a lane.
  if (of_row * kWave < left) {
    segment_t z;
    z[0] = early;
    Add<1>(z, early, &sums);
  }
  const bool unlike = left > waves * kWave;  // rows that do not lie alike
#pragma unroll 1
  for (int k = left_first + waves * kWave; unlike && k - lane < left; k += waves * kWave) {
    segment_t z;
    z[0] = k < left ? from.At(left_index(k)) : -Inf();
    Add<1>(z, z[0], &sums);
  }

  __shared__ Entry slots[kWaves][kWave];
  if (p.top > 0) {
    // Run `segment` of lane `of_lane`, into c and u.
    const auto load_run = [&](int segment, int of_lane) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int at = min(segment * kSegment + of_lane * kElements + v * kVec, body - kVec);
        c[v] = *reinterpret_cast<const vec*>(from.c + head + at);
        if (GUIDED)
          u[v] = *reinterpret_cast<const vec*>(from.u + head + at);
      }
    };
    const auto peak_of = [&](int segment, int of_lane) {
      load_run(segment, of_lane);
      segment_t z = elements(segment * kSegment, of_lane);
      const int hidden = p.mask_id - head - segment * kSegment - of_lane * kElements;
#pragma unroll
      for (int e = 0; e < kElements; ++e)
        z[e] = hidden == e ? -Inf() : z[e];
      return Peak(z);
    };
    bool whole = !unlike;
    if (whole) {
      int at = of_row * kSegment + lane * kElements;  // of the body
      unsigned known = 1;
      if (WAVES == 1 && seen <= 1) {
        // All of it is here. As many lanes' own largest reach `known` as are listed.
        const float peak = runs.peak[0];
        const unsigned order = peak > -Inf() ? OrderOf(peak) : 0u;
        const auto reach = [&](unsigned least) { return __popcll(__ballot(order >= least)); };
        const unsigned most = WaveMaxOf(order);
        const unsigned lowest = ~WaveMaxOf(order == 0 ? 0u : ~order);
        if (most != 0 && reach(lowest) >= p.top)
          known = reach(most) >= p.top ? most
                                       : Between(lowest, most, p.top, p.top + 8, reach);
      } else {
        int of_segment, of_lane;
        known = runs.Pick(p.top, of_row, waves, seen, peak_of, lane, &of_segment, &of_lane);
        // The runs again.
        at = of_segment * kSegment + of_lane * kElements;
        if (of_segment >= 0)
          load_run(of_segment, of_lane);
        const segment_t run = elements(of_segment * kSegment, of_lane);
#pragma unroll
        for (int e = 0; e < kElements; ++e)
          held[e] = of_segment >= 0 ? run[e] : -Inf();
      }
      // And the element that was left.
      float z[kElements + 1];
#pragma unroll
      for (int e = 0; e < kElements; ++e)
        z[e] = held[e];
      z[kElements] = early;
      whole = Rank<kElements + 1>(
          z,
          [&](int e) { return but_mask(e < kElements ? head + at + e : left_index(left_first)); },
          known, lane, slots[wave], &best);
    }
    if (!whole) {
      // All the wave's elements once more: the body, then what is left.
#pragma unroll 1
      for (int base = of_row * kSegment; base < body; base += waves * kSegment) {
        load(base);
        const segment_t z = elements(base, lane);
        Search<kElements>(
            z, Peak(z), [&](int e) { return but_mask(head + base + lane * kElements + e); }, lane,
            &best);
      }
#pragma unroll 1
      for (int k = left_first; k - lane < left; k += waves * kWave) {
        segment_t z;
        z[0] = k < left ? from.At(left_index(k)) : -Inf();
        Search<1>(z, z[0], [&](int) { return but_mask(left_index(k)); }, lane, &best);
      }
    }
  }

  sums.JoinWave();
  if constexpr (WAVES > 1) {
    __shared__ Sums shared[WAVES];
    __shared__ Entry lists[WAVES][kMostAlternatives];
    if (lane == 0)
      shared[wave] = sums;
    if (lane < p.top)
      lists[wave][lane] = {best.order, best.index};
    __syncthreads();
    if (wave != 0)
      return;
    float top = -Inf();
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      top = fmaxf(top, shared[w].m);
    sums.Move(top == -Inf() ? sums.m : top);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      Sums part = shared[w];
      part.Move(top == -Inf() ? part.m : top);
      sums.s += part.s;
      sums.t += part.t;
    }
    if (p.top > 0) {
      // Up to 128 entries, two a lane, of which those matter that reach the highest of
      // the lists' last ones.
      constexpr int kEach = WAVES * kMostAlternatives / kWave;
      float z[kEach];
      int index[kEach];
      unsigned known = 1;
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        known = max(known, lists[w][p.top - 1].order);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int w = (e * kWave + lane) / kMostAlternatives, k = lane % kMostAlternatives;
        const Entry entry = lists[w][k];
        z[e] = k < p.top ? ValueOf(entry.order) : -Inf();
        index[e] = entry.index;
      }
      if (!Rank<kEach>(z, [&](int e) { return index[e]; }, known, lane, slots[0], &best)) {
        for (int w = 1; w < WAVES; ++w) {
          const Entry entry = lists[w][lane % kMostAlternatives];
          best.Merge(entry.order, entry.index, lane);
        }
      }
    }
    if (p.splits > 1) {
      float* state = p.states + (row * p.splits + blockIdx.y) * (4 + 2 * p.top);
      if (lane == 0) {
        state[0] = sums.m;
        state[1] = sums.s;
        state[2] = sums.t;
      }
      if (lane < p.top) {
        state[4 + lane] = ValueOf(best.order);
        state[4 + p.top + lane] = __int_as_float(best.index);
      }
      return;
    }
  }
  Answer(p, row, chosen, sums, best, lane);
}

// One wave per row: lane i takes split i's sums, and the splits' lists, element k of
// split s being the (s top + k)-th, are searched as a row's elements are.
template <typename T>
__global__ __launch_bounds__(kWave) void JoinLogprobsKernel(LogprobParams p) {
  const int lane = threadIdx.x;
  const std::int64_t row = blockIdx.x;
  const int state_size = 4 + 2 * p.top;
  const float* states = p.states + row * p.splits * state_size;
  Row<T> from;
  from.c = static_cast<const T*>(p.logits) + row * p.stride;
  from.u = p.uncond == nullptr ? nullptr
                               : static_cast<const T*>(p.uncond) + row * p.uncond_stride;
  from.g = p.guidance;
  const float chosen = Chosen(p, row, from);
  Sums sums{-Inf(), 0.0F, 0.0F};
  Alternatives best(p.top);
  if (lane < p.splits) {
    const float* state = states + lane * state_size;
    sums = {state[0], state[1], state[2]};
  }
  // Element k of split s is the (32 s + k)-th, of up to 512: 8 a lane.
  if (p.top > 0) {
    constexpr int kEach = kMostLogprobSplits * kMostAlternatives / kWave;
    __shared__ Entry slots[kWave];
    float z[kEach];
    int index[kEach];
    unsigned floor = 1;
    if (lane < p.splits)
      floor = max(floor, OrderOf(states[lane * state_size + 4 + p.top - 1]));
    const unsigned known = WaveMaxOf(floor);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int split = e * (kWave / kMostAlternatives) + lane / kMostAlternatives;
      const int k = lane % kMostAlternatives;
      const bool there = split < p.splits && k < p.top;
      const float* state = states + min(split, p.splits - 1) * state_size + 4 + min(k, p.top - 1);
      z[e] = state[0];
      index[e] = there ? __float_as_int(state[p.top]) : -1;
    }
    if (!Rank<kEach>(z, [&](int e) { return index[e]; }, known, lane, slots, &best)) {
      segment_t all;
#pragma unroll
      for (int e = 0; e < kElements; ++e)
        all[e] = e < kEach ? z[e % kEach] : -Inf();
      Search<kElements>(all, Peak(all), [&](int e) { return index[e % kEach]; }, lane, &best);
    }
  }
  sums.JoinWave();
  Answer(p, row, chosen, sums, best, lane);
}

constexpr int kOneWave = 2048;  // elements of a row that one wave takes

template <typename T, bool GUIDED>
void Launch(const LogprobParams& p, hipStream_t stream) {
  const dim3 block(kWaves * kWave);
  const bool last = p.splits == 1;
  if (p.vocab <= kOneWave)
    Dispatch(LogprobKernel<T, GUIDED, 1>, dim3((p.rows + kWaves - 1) / kWaves), block, 0, stream,
             true, last, p);
  else
    Dispatch(LogprobKernel<T, GUIDED, kWaves>, dim3(p.rows, p.splits), block, 0, stream, true,
             last, p);
  if (!last)
    Dispatch(JoinLogprobsKernel<T>, dim3(p.rows), dim3(kWave), 0, stream, false, true, p);
}

}  // namespace

int PlanLogprobs(int rows, int vocab) {
  if (rows == 0 || vocab <= kOneWave)
    return 1;
  const int wanted = (kLogprobGroups + rows - 1) / rows;
  const int most = (vocab + kWaves * kSegment - 1) / (kWaves * kSegment);
  return std::max(1, std::min({wanted, most, kMostLogprobSplits}));
}

void LaunchLogprobs(const LogprobParams& p, DType type, hipStream_t stream) {
  if (p.rows == 0)
    return;
  const bool guided = p.uncond != nullptr;
  if (type == DType::kF16)
    guided ? Launch<_Float16, true>(p, stream) : Launch<_Float16, false>(p, stream);
  else if (type == DType::kBf16)
    guided ? Launch<__bf16, true>(p, stream) : Launch<__bf16, false>(p, stream);
  else
    guided ? Launch<float, true>(p, stream) : Launch<float, false>(p, stream);
  Check(hipGetLastError(), "logprobs launch");
}

}  // namespace ovg
