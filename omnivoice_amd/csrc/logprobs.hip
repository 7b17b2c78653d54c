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
// maximum, which the sums need anyhow, reaches the list's last value; for the
// first segment of a wave, whose list is empty, the top-th largest of the lanes'
// maxima stands in (that many elements reach it, so no lower one is listed).
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

// Takes z (element e of this lane at index IndexOf(e), -inf for none) into the
// sums and the list.
template <int N, typename F>
__device__ __forceinline__ void Take(const float (&z)[N], F&& index_of, int mask_id, int lane,
                                     Sums* sums, Alternatives* best) {
  float peak = z[0];
#pragma unroll
  for (int e = 1; e < N; ++e)
    peak = fmaxf(peak, z[e]);
  if (peak > sums->m)
    sums->Move(peak);
  const float from = sums->m == -Inf() ? 0.0F : sums->m;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = (z[e] - from) * kLog2e;
    const float x = __builtin_amdgcn_exp2f(d);
    sums->s += x;
    // 0 * -inf stays 0; a NaN is x's already.
    sums->t = __builtin_fmaf(x, fmaxf(d, -1000.0F), sums->t);
  }
  if (best->top == 0)
    return;
  float floor = best->Floor();
  if (!__any(peak >= floor && peak > -Inf()))
    return;
  if (floor == -Inf()) {
    // The list is not full.
    float mine = -Inf();
#pragma unroll
    for (int e = 0; e < N; ++e)
      mine = index_of(e) == mask_id ? mine : fmaxf(mine, z[e]);
    for (int k = 0; k < best->top; ++k) {
      floor = WaveMaxFast(mine);
      if (floor == -Inf())
        break;
      if (lane == __ffsll(__ballot(mine == floor)) - 1)
        mine = -Inf();
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    // Asked again after each: the list's last value rises, and with equal values
    // one index after another would be turned away.
    const bool listed = z[e] >= floor && z[e] > -Inf() && index_of(e) != mask_id;
    unsigned long long todo = __ballot(listed);
    while ((todo &= __ballot(listed && best->Takes(z[e], index_of(e)))) != 0) {
      const int who = __ffsll(todo) - 1;
      todo &= todo - 1;
      best->Insert(LaneOf(z[e], who), __builtin_amdgcn_readlane(index_of(e), who), lane);
    }
  }
}

// What a row's answers need: its whole sums and list.
template <typename T>
__device__ __forceinline__ void Answer(const LogprobParams& p, std::int64_t row, const Row<T>& from,
                                       const Sums& sums, const Alternatives& best, int lane) {
  // No distribution: a NaN or +infinity among the logits, or nothing above -infinity.
  const bool none = !(sums.s > 0.0F && sums.s < Inf());
  const float log_s = logf(sums.s);
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (p.logprob != nullptr) {
      const int token = p.tokens[row];
      const float z = token >= 0 && token < p.vocab ? from.At(token) : -Inf();
      p.logprob[row] = none ? nan : z - sums.m - log_s;
    }
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
  for (int base = of_row * kSegment; base < body; base += waves * kSegment) {
    float z[kElements];
    vec c[kVecs], u[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int at = base + (v * kWave + lane) * kVec;
      const int safe = head + min(at, body - kVec);
      c[v] = *reinterpret_cast<const vec*>(from.c + safe);
      if (GUIDED)
        u[v] = *reinterpret_cast<const vec*>(from.u + safe);
    }
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const bool there = base + (v * kWave + lane) * kVec < body;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float x = static_cast<float>(c[v][e]);
        const float guided = GUIDED ? Guide(x, static_cast<float>(u[v][e]), p.guidance) : x;
        z[v * kVec + e] = there ? guided : -Inf();
      }
    }
    Take(z, [&](int e) { return head + base + (e / kVec * kWave + lane) * kVec + e % kVec; },
         p.mask_id, lane, &sums, &best);
  }
  // What is left, one element a lane: the head and the tail, or all of two rows
  // that do not lie alike.
  const int left = p.vocab - body;
  for (int base = of_row * kWave; base < left; base += waves * kWave) {
    const int k = base + lane;
    const int at = k < head ? k : k + body;
    const float z[1] = {k < left ? from.At(at) : -Inf()};
    Take(z, [&](int) { return at; }, p.mask_id, lane, &sums, &best);
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
  Answer(p, row, from, sums, best, lane);
}

// One wave per row: lane i takes split i's sums.
template <typename T>
__global__ __launch_bounds__(kWave) void JoinLogprobsKernel(LogprobParams p) {
  const int lane = threadIdx.x;
  const std::int64_t row = blockIdx.x;
  const float* states = p.states + row * p.splits * (4 + 2 * p.top);
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
  Row<T> from;
  from.c = static_cast<const T*>(p.logits) + row * p.stride;
  from.u = p.uncond == nullptr ? nullptr
                               : static_cast<const T*>(p.uncond) + row * p.uncond_stride;
  from.g = p.guidance;
  Answer(p, row, from, sums, best, lane);
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
