// The 8-bit key/value cache and the token log probabilities: parameters and
// launchers of cache_kernels.hip, cache_attention.hip and logprobs.hip.
#ifndef OMNIVOICE_AMD_CACHE_HPP_
#define OMNIVOICE_AMD_CACHE_HPP_

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.hpp"

namespace ovg {

// Element types of the operators' caller tensors (OVG_F16, OVG_BF16, OVG_F32,
// OVG_E4M3).
enum class DType : int { kF16 = 0, kBf16 = 1, kF32 = 2, kE4m3 = 3 };

// A pool of blocks and the sequences of one call. Device pointers; the
// values behind them are not known to the host, so every kernel clamps what
// it reads of them (Span, Page).
struct CacheView {
  unsigned char* data;  // [blocks][kv_heads][2][block_tokens * dim], e4m3 codes
  float* scales;        // [blocks][kv_heads][2]
  const int* tables;    // [count][table_width]
  const int* lengths;   // [count]
  const int* begins;    // [count + 1]
  int blocks, block_shift, kv_heads, dim;
  int count, table_width, rows;
};

// One half (keys 0, values 1) of one head of a block: dim << block_shift codes.
__device__ __forceinline__ unsigned char* HalfOf(const CacheView& c, int page, int head,
                                                 int half) {
  const std::size_t index =
      (static_cast<std::size_t>(page) * c.kv_heads + head) * 2 + half;
  return c.data + index * (static_cast<std::size_t>(c.dim) << c.block_shift);
}
__device__ __forceinline__ std::size_t ScaleIndex(const CacheView& c, int page, int head,
                                                  int half) {
  return (static_cast<std::size_t>(page) * c.kv_heads + head) * 2 + half;
}

// The pool block of a sequence's block `b`, or -1 where the table has none.
__device__ __forceinline__ int PageOf(const CacheView& c, int sequence, int b) {
  if (b < 0 || b >= c.table_width)
    return -1;
  const int page = c.tables[static_cast<std::size_t>(sequence) * c.table_width + b];
  return page >= 0 && page < c.blocks ? page : -1;
}

// A sequence's rows [first, first + count) of the call's tensors, clamped into
// them, and the cache position `start` of the first of these (-count where all of
// them come before position 0, else negative where the sequence is shorter than its
// rows). The rows' last position is length - 1 unless rows were cut off behind.
struct Span {
  int first, count, start, length;
};
// Work items of ragged sequences without a list: sequence i owns the items
// from first_i * scale / tile + slack * i (a whole-number division) up to the next
// one's, at least rows_i * scale / tile + slack of them. Every lane looks at a
// sequence of its own and holds what belongs to it, so that finding an item and its
// span is one trip to memory for up to 64 sequences; where there are more, a trip
// before it leaves a 64th of them. The whole wave calls this; all it returns is the
// same in every lane. count 0: the item is nobody's.
struct Found {
  int sequence, item;  // item: of the sequence
  Span span;
};
__device__ __forceinline__ Found FindItem(const CacheView& c, int scale, int shift, int slack,
                                          int item) {
  const int lane = threadIdx.x & (kWave - 1);
  Found f{0, 0, {0, 0, 0, 0}};
  int low = 0, count = c.count;  // the owner is one of these
  while (count > kWave) {
    const int stride = (count + kWave - 1) / kWave;
    const int i = min(low + lane * stride, c.count - 1);
    const int first = min(max(c.begins[i], 0), c.rows);
    const int base = ((first * scale) >> shift) + slack * i;
    const int below = __popcll(__ballot(lane * stride < count && base <= item));
    if (below == 0)
      return f;
    low += (below - 1) * stride;
    count = min(stride, count - (below - 1) * stride);
  }
  const int i = min(low + lane, c.count - 1);
  const int begin = c.begins[i], end = c.begins[i + 1], length = c.lengths[i];
  const int first = min(max(begin, 0), c.rows);
  const int rows = min(max(end, first), c.rows) - first;
  // Row r is token length - (end - r), also where there are fewer rows than begins says.
  const int start = max(max(length, 0) - max(end, first) + first, -rows);
  const int base = ((first * scale) >> shift) + slack * i;
  const int below = __popcll(__ballot(lane < count && base <= item));
  if (below > 0) {
    const int owner = below - 1;
    f.sequence = low + owner;
    f.item = item - __builtin_amdgcn_readlane(base, owner);
    f.span.first = __builtin_amdgcn_readlane(first, owner);
    f.span.count = __builtin_amdgcn_readlane(rows, owner);
    f.span.length = max(__builtin_amdgcn_readlane(length, owner), 0);
    f.span.start = __builtin_amdgcn_readlane(start, owner);
  }
  return f;
}
inline int ItemBound(const CacheView& c, int scale, int shift, int slack) {
  return ((c.rows * scale) >> shift) + slack * c.count;
}

// ---------------------------------------------------------------- cache
struct CacheWriteParams {
  CacheView cache;
  const void* x[2];  // keys, values [rows][kv_heads][dim], rows `stride` elements apart
  std::int64_t stride[2];
};
void LaunchCacheWrite(const CacheWriteParams& p, DType type, hipStream_t stream);

struct CacheReadParams {
  CacheView cache;
  void* x[2];
  std::int64_t stride[2];
};
void LaunchCacheRead(const CacheReadParams& p, DType type, hipStream_t stream);

struct CacheAttentionParams {
  CacheView cache;
  const void* q;   // [rows][heads][dim], rows q_stride elements apart
  void* out;       // [rows][heads][dim], rows out_stride elements apart
  std::int64_t q_stride, out_stride;
  int group;       // query heads per kv head
  int group_inverse;               // 2^16 / group, rounded up
  unsigned long long group_magic;  // 2^36 / group, rounded up
  bool causal;
  float scale_log2;  // the softmax's scale * log2(e), without its sign:
  bool negate;       // the queries take it
  // The plan's (PlanCacheAttention), and where its splits leave their states:
  // slot ((item * kv_heads + head) * splits + split) * tile rows + row has its
  // row's maximum and sum in partial_m and its output over a power of two (PowerAbove)
  // in partial_o.
  int tile_shift, splits, own_shift;
  int items, first_item;  // tiles in all, and the first of a launch
  float* partial_m;  // [slots][2]
  float* partial_o;  // [slots][dim]
};
// How a call is split: from the shapes that the host knows.
struct CacheAttentionPlan {
  int tile_shift = 4;     // log2 of a work-group's rows
  int splits = 1;         // of each sequence's keys
  int own_shift = 0;      // log2 of a work-group's tiles
  std::size_t slots = 0;  // of the workspace
};
constexpr int kMostSplits = 256;
constexpr int kFewSplits = 8;  // that one group of lanes joins by itself
// Sequences of few rows (16-row tiles) that leave CUs idle are split until every CU
// has a work-group, into 256 keys at least and only from 1024 tokens on: the second
// launch costs what 500 keys do (8 heads, us of the GPU: 500 keys 6.3 whole and 7.4
// in two, 1000 keys 8.2 and 7.1 in eight, 4000 keys 19.7 and 8.6 in sixteen, 90001
// keys 34 in 16 to 64; 16 sequences of 1000 keys 9.6 whole, 11.6 in two).
constexpr int kFullGroups = 256;
constexpr int kLeastSplit = 1024;
constexpr int kLeastChunk = 256;
// Many of them are ragged and fill the device better in smaller pieces, of 1024 keys
// at least: 48 of up to 8192 keys take 102 us whole, 95.5 in four, 32 of 4000 keys
// 48.4 and 46.3.
constexpr int kRaggedGroups = 2048;
// Tiles of 32 rows leave as much as they read when they are split: 375 queries of two
// heads over 2000 keys take 16.8 us whole and 20.9 in two, 100 over 16000 take 80 us
// whole and 30 in four.
constexpr int kSplitGroups = 512;
constexpr int kLeastTileChunk = 1024;
// A wave takes a whole tile of 32 rows instead of a quarter of its keys where that
// still fills the device, two work-groups a CU (128 dims) or four (64), and the keys
// are few, so that the waves' join is much of the work: 32 sequences of 120 queries of
// two heads over 256 keys 21.6 us and 32.1 in quarters, over 1024 47.6 and 56.0 (16 of
// them, half of the device, 44.3 and 31.3; with 64 dims 39.1 and 31.3, 64 of them 51.8
// and 56.8). With 128 dims it also pays over any keys from two fills on: two causal
// prompts of 5000 tokens 234.5 and 239.9, 64 sequences of 120 over 2048 170 and 188.
constexpr int kOwnTiles = 2048;  // of 128 dims that fill the device
constexpr int kOwnKeys = 1024;
CacheAttentionPlan PlanCacheAttention(const CacheView& c, int group);
// Keys of each split of a sequence of `length` tokens: a whole number of the
// four waves' steps.
__host__ __device__ inline int ChunkOf(int length, int splits) {
  if (splits == 1)
    return length;
  const int even = (length + splits - 1) / splits;
  return (even > kLeastChunk ? even + 127 : kLeastChunk) & ~127;
}
void LaunchCacheAttention(const CacheAttentionParams& p, DType type, hipStream_t stream);

// ---------------------------------------------------------------- log probabilities
struct LogprobParams {
  const void* logits;  // [rows][vocab], rows `stride` elements apart
  const void* uncond;  // the same, or null
  std::int64_t stride, uncond_stride;
  const int* tokens;   // [rows], or null
  float guidance;
  int rows, vocab, mask_id, top;
  float* logprob;        // [rows], or null
  float* entropy;        // [rows], or null
  int* top_ids;          // [rows][top]
  float* top_logprobs;   // [rows][top]
  int splits;            // of each row (PlanLogprobs)
  float* states;         // [rows][splits][4 + 2 top] where there are several
};
constexpr int kMostAlternatives = 32;
constexpr int kLogprobGroups = 512;  // work-groups that a call is to have
constexpr int kMostLogprobSplits = 16;
int PlanLogprobs(int rows, int vocab);
void LaunchLogprobs(const LogprobParams& p, DType type, hipStream_t stream);

}  // namespace ovg

#endif  // OMNIVOICE_AMD_CACHE_HPP_
