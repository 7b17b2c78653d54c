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
// fixed order. The best `top` values are a sorted list in the wave's lanes. A
// segment of 1024 elements is searched for entrants only where some lane's
// maximum, which the sums need anyhow, reaches the list's last value; the first
// segment of a wave gives its largest elements one after the other.
//
// Elements come as aligned 16-byte loads; the up to 14 before a row's first
// 16-byte border and behind its last are one more segment of single loads. A row
// belongs to one wave up to 2048 elements (four rows to a work-group), else to
// the four waves of a work-group, and where there are too few rows for the
// device to several of those, whose states a second kernel joins.
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

// (value, index) pairs in descending order, equal values by index.
__device__ __forceinline__ bool Before(float a, int i, float b, int j) {
  return a > b || (a == b && i < j);
}

template <int CTRL>
__device__ __forceinline__ int Dpp(int v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ float LaneOf(float v, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The `top` best so far: lane j holds the j-th, (-inf, -1) where there is none.
struct Alternatives {
  float value;
  int index;
  int top;
  __device__ __forceinline__ float Floor() const { return LaneOf(value, top - 1); }
  __device__ __forceinline__ int FloorIndex() const {
    return __builtin_amdgcn_readlane(index, top - 1);
  }
  // Whether (v, i) belongs into the list.
  __device__ __forceinline__ bool Takes(float v, int i) const {
    return Before(v, i, Floor(), FloorIndex());
  }
  // (v, i), the same in every lane, that belongs into it.
  __device__ __forceinline__ void Insert(float v, int i, int lane) {
    const int at = __popcll(__ballot(lane < top && Before(value, index, v, i)));
    const float up = __builtin_bit_cast(float, Dpp<0x138>(__builtin_bit_cast(int, value)));
    const int up_index = Dpp<0x138>(index);  // wave_shr: 1
    value = lane == at ? v : lane > at ? up : value;
    index = lane == at ? i : lane > at ? up_index : index;
  }
  // Another sorted list: nothing behind the first that does not belong does.
  template <typename V, typename I>
  __device__ __forceinline__ void Merge(V&& value_of, I&& index_of, int lane) {
    for (int k = 0; k < top; ++k) {
      const float v = value_of(k);
      const int i = index_of(k);
      if (!Takes(v, i))
        break;
      Insert(v, i, lane);
    }
  }
};

struct Sums {
  float m, s, t;
  // The same sums relative to another maximum.
  __device__ __forceinline__ void Move(float to) {
    const float d = m == -Inf() ? 0.0F : (m - to) * kLog2e;
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
  return max(b[0], b[1]);
}

// Whole numbers in the order of the floats; 0 is below them all. -0 and +0 are one.
__device__ __forceinline__ unsigned OrderOf(float v) {
  const unsigned u = __float_as_uint(v + 0.0F);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ValueOf(unsigned order) {
  return __uint_as_float((order & 0x80000000u) != 0 ? order & 0x7FFFFFFFu : ~order);
}

// The list of a wave's first segment: `top` times the largest of what is left.
// A lane's elements are in the order of their indices.
template <typename F>
__device__ __forceinline__ void First(const segment_t& z, F&& index_of, int mask_id, int lane,
                                      Alternatives* best) {
  unsigned key[kElements];
#pragma unroll
  for (int e = 0; e < kElements; ++e)
    key[e] = z[e] > -Inf() && index_of(e) != mask_id ? OrderOf(z[e]) : 0u;
  for (int k = 0; k < best->top; ++k) {
    unsigned most = key[0];
#pragma unroll
    for (int e = 1; e < kElements; ++e)
      most = max(most, key[e]);
    const unsigned largest = __builtin_amdgcn_readfirstlane(WaveMaxOf(most));
    if (largest == 0)
      return;
    // Where it is first in each lane that has it, and the first of those.
    int at = kElements;
#pragma unroll
    for (int e = kElements - 1; e >= 0; --e)
      at = key[e] == largest ? e : at;
    const unsigned long long have = __ballot(at < kElements);
    int index = index_of(at);
    int who = __ffsll(have) - 1;
    if ((have & (have - 1)) != 0) {
      const unsigned first = ~WaveMaxOf(at < kElements ? ~static_cast<unsigned>(index) : 0u);
      who = __ffsll(__ballot(at < kElements && static_cast<unsigned>(index) == first)) - 1;
    }
    index = __builtin_amdgcn_readlane(index, who);
    if (lane == k) {
      best->value = ValueOf(largest);
      best->index = index;
    }
    at = lane == who ? at : kElements;
#pragma unroll
    for (int e = 0; e < kElements; ++e)
      key[e] = at == e ? 0u : key[e];
  }
}

// Takes a segment into the sums and the list; index_of(e): its e-th element's.
// `others`: what the list's last value is known to reach in the end.
template <typename F>
__device__ __forceinline__ void Take(const segment_t& z, F&& index_of, float others, int mask_id,
                                     int lane, Sums* sums, Alternatives* best) {
  constexpr int kRun = 4;  // elements that are passed over together
  typedef float peaks_t __attribute__((ext_vector_type(kElements / kRun)));
  peaks_t peaks;
#pragma unroll
  for (int k = 0; k < kElements / kRun; ++k)
    peaks[k] = fmaxf(fmaxf(z[kRun * k], z[kRun * k + 1]), fmaxf(z[kRun * k + 2], z[kRun * k + 3]));
  const float peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
  if (peak > sums->m)
    sums->Move(peak);
  const float from = sums->m == -Inf() ? 0.0F : sums->m;
#pragma unroll
  for (int e = 0; e < kElements; ++e) {
    const float d = (z[e] - from) * kLog2e;
    const float x = __builtin_amdgcn_exp2f(d);
    sums->s += x;
    // 0 * -inf stays 0; a NaN is x's already.
    sums->t = __builtin_fmaf(x, fmaxf(d, -1000.0F), sums->t);
  }
  if (best->top == 0)
    return;
  const float floor = fmaxf(best->Floor(), others);
  if (!__any(peak >= floor && peak > -Inf()))
    return;
  if (LaneOf(best->value, 0) == -Inf()) {
    First(z, index_of, mask_id, lane, best);
    return;
  }
  // Not unrolled: the registers are indexed.
#pragma unroll 1
  for (int e = 0; e < kElements; ++e) {
    if (e % kRun == 0 && !__any(peaks[e / kRun] >= floor)) {
      e += kRun - 1;
      continue;
    }
    const float v = z[e];
    const int i = index_of(e);
    const bool listed = v >= floor && v > -Inf() && i != mask_id;
    unsigned long long todo = __ballot(listed);
    // Asked again after each: the list's last value rises, and with equal values
    // one index after another would be turned away.
    while (todo != 0 && (todo &= __ballot(listed && best->Takes(v, i))) != 0) {
      const int who = __ffsll(todo) - 1;
      todo &= todo - 1;
      best->Insert(LaneOf(v, who), __builtin_amdgcn_readlane(i, who), lane);
    }
  }
}

// The same for one element a lane.
__device__ __forceinline__ void TakeOne(float z, int index, float others, int mask_id, int lane,
                                        Sums* sums, Alternatives* best) {
  if (z > sums->m)
    sums->Move(z);
  const float d = (z - (sums->m == -Inf() ? 0.0F : sums->m)) * kLog2e;
  const float x = __builtin_amdgcn_exp2f(d);
  sums->s += x;
  sums->t = __builtin_fmaf(x, fmaxf(d, -1000.0F), sums->t);
  if (best->top == 0)
    return;
  const bool listed = z >= others && z > -Inf() && index != mask_id;
  unsigned long long todo = __ballot(listed);
  while (todo != 0 && (todo &= __ballot(listed && best->Takes(z, index))) != 0) {
    const int who = __ffsll(todo) - 1;
    todo &= todo - 1;
    best->Insert(LaneOf(z, who), __builtin_amdgcn_readlane(index, who), lane);
  }
}

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
    p.top_logprobs[row * p.top + lane] = none ? nan : best.value - sums.m - log_s;
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
  Alternatives best{-Inf(), -1, p.top};

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

  // The floors of the row's waves. Each is the last value of a full list of some of
  // the row's elements, so nothing below the highest can be listed in the end; it is
  // read without waiting for anyone, an older one only passes over less.
  __shared__ float floors[kWaves];
  if constexpr (WAVES > 1) {
    if (lane == 0)
      floors[wave] = -Inf();
    __syncthreads();
  }
  const auto known = [&]() {
    float f = -Inf();
    if constexpr (WAVES > 1) {
#pragma unroll
      for (int i = 0; i < WAVES; ++i)
        f = fmaxf(f, __hip_atomic_load(&floors[i], __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_WORKGROUP));
    }
    return f;
  };

  vec c[kVecs], u[kVecs];
  const auto load = [&](int base) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int at = head + min(base + (v * kWave + lane) * kVec, body - kVec);
      c[v] = *reinterpret_cast<const vec*>(from.c + at);
      if (GUIDED)
        u[v] = *reinterpret_cast<const vec*>(from.u + at);
    }
  };
  if (of_row * kSegment < body)
    load(of_row * kSegment);
#pragma unroll 1
  for (int base = of_row * kSegment; base < body; base += waves * kSegment) {
    segment_t z;
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float x = static_cast<float>(c[v][e]);
        z[v * kVec + e] = GUIDED ? Guide(x, static_cast<float>(u[v][e]), p.guidance) : x;
      }
    load(base + waves * kSegment);  // past the end the last ones again
    if (base + kSegment > body) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          z[v * kVec + e] =
              base + (v * kWave + lane) * kVec < body ? z[v * kVec + e] : -Inf();
    }
    const float before = best.top > 0 ? best.Floor() : 0.0F;
    Take(z, [&](int e) { return head + base + (e / kVec * kWave + lane) * kVec + e % kVec; },
         known(), p.mask_id, lane, &sums, &best);
    if constexpr (WAVES > 1) {
      const float after = best.top > 0 ? best.Floor() : 0.0F;
      if (after != before && lane == 0)
        __hip_atomic_store(&floors[wave], after, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  if (of_row * kWave < left)
    TakeOne(early, left_index(left_first), known(), p.mask_id, lane, &sums, &best);
#pragma unroll 1
  for (int k0 = (of_row + waves) * kWave; k0 < left; k0 += waves * kSegment) {
    segment_t z;
#pragma unroll
    for (int e = 0; e < kElements; ++e) {
      const int k = k0 + e * waves * kWave + lane;
      z[e] = k < left ? from.At(left_index(k)) : -Inf();
    }
    Take(z, [&](int e) { return left_index(k0 + e * waves * kWave + lane); }, known(), p.mask_id,
         lane, &sums, &best);
  }

  sums.JoinWave();
  if constexpr (WAVES > 1) {
    __shared__ Sums shared[WAVES];
    __shared__ float shared_value[WAVES][kMostAlternatives];
    __shared__ int shared_index[WAVES][kMostAlternatives];
    if (lane == 0)
      shared[wave] = sums;
    if (lane < p.top) {
      shared_value[wave][lane] = best.value;
      shared_index[wave][lane] = best.index;
    }
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
      if (p.top > 0)
        best.Merge([&](int k) { return shared_value[w][k]; },
                   [&](int k) { return shared_index[w][k]; }, lane);
    }
    if (p.splits > 1) {
      float* state = p.states + (row * p.splits + blockIdx.y) * (4 + 2 * p.top);
      if (lane == 0) {
        state[0] = sums.m;
        state[1] = sums.s;
        state[2] = sums.t;
      }
      if (lane < p.top) {
        state[4 + lane] = best.value;
        state[4 + p.top + lane] = __int_as_float(best.index);
      }
      return;
    }
  }
  Answer(p, row, chosen, sums, best, lane);
}

// One wave per row: lane i takes split i's sums.
template <typename T>
__global__ __launch_bounds__(kWave) void JoinLogprobsKernel(LogprobParams p) {
  const int lane = threadIdx.x;
  const std::int64_t row = blockIdx.x;
  const float* states = p.states + row * p.splits * (4 + 2 * p.top);
  Row<T> from;
  from.c = static_cast<const T*>(p.logits) + row * p.stride;
  from.u = p.uncond == nullptr ? nullptr
                               : static_cast<const T*>(p.uncond) + row * p.uncond_stride;
  from.g = p.guidance;
  const float chosen = Chosen(p, row, from);
  Sums sums{-Inf(), 0.0F, 0.0F};
  Alternatives best{-Inf(), -1, p.top};
  if (lane < p.splits) {
    const float* state = states + lane * (4 + 2 * p.top);
    sums = {state[0], state[1], state[2]};
  }
  // Lane k of the s-th list; the next one is on its way while this one is offered.
  float value = lane < p.top ? states[4 + lane] : -Inf();
  int index = lane < p.top ? __float_as_int(states[4 + p.top + lane]) : -1;
  for (int s = 0; s < p.splits && p.top > 0; ++s) {
    const float* next = states + min(s + 1, p.splits - 1) * (4 + 2 * p.top);
    const float next_value = lane < p.top ? next[4 + lane] : -Inf();
    const int next_index = lane < p.top ? __float_as_int(next[4 + p.top + lane]) : -1;
    best.Merge([&](int k) { return LaneOf(value, k); },
               [&](int k) { return __builtin_amdgcn_readlane(index, k); }, lane);
    value = next_value;
    index = next_index;
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
  return std::max(1, std::min({wanted, most, kWave}));
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
