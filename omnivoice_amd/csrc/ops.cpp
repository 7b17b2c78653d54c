// Device operators on caller-owned device pointers (include/omnivoice_mi355x.h,
// "Device operators"): each is one launcher of the generator's kernels
// behind the C ABI, for integration and for per-kernel parity tests.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "ops.hpp"

namespace {

using namespace ovg::ops;

// A device allocation that lives for one operator call.
template <typename T>
struct Scratch {
  T* data = nullptr;
  explicit Scratch(std::size_t count) {
    ovg::Check(hipMalloc(reinterpret_cast<void**>(&data),
                         std::max<std::size_t>(count, 1) * sizeof(T)),
               "hipMalloc");
  }
  ~Scratch() {
    if (data != nullptr)
      (void)hipFree(data);
  }
};

// The pool and sequences of a call, their sizes checked against what the
// kernels' 32-bit positions, rows and items hold.
ovg::CacheView ViewOf(const ovg_kv_cache* cache, const ovg_kv_sequences* sequences) {
  ovg::Require(cache && sequences, "null pointer");
  ovg::Require(cache->data && cache->scales, "null pool");
  ovg::Require(Aligned16(cache->data), "the pool must be 16-byte aligned");
  ovg::Require(cache->block_tokens == 16 || cache->block_tokens == 32 || cache->block_tokens == 64,
               "block_tokens must be 16, 32 or 64");
  ovg::Require(cache->head_dim == 64 || cache->head_dim == 128, "head_dim must be 64 or 128");
  ovg::Require(cache->kv_heads >= 1 && cache->kv_heads <= 1024, "kv_heads outside [1, 1024]");
  ovg::Require(cache->blocks >= 1 && FitsInt(cache->blocks), "blocks outside [1, 2^30]");
  ovg::Require(sequences->count >= 0 && sequences->count <= (1 << 20),
               "count outside [0, 2^20]");
  ovg::Require(sequences->rows >= 0 && sequences->rows <= (1 << 24), "rows outside [0, 2^24]");
  ovg::Require(sequences->table_width >= 1 &&
                   sequences->table_width <= (int64_t{1} << 30) / cache->block_tokens,
               "table_width outside [1, 2^30 / block_tokens]");
  ovg::Require(sequences->count == 0 ||
                   (sequences->tables && sequences->lengths && sequences->begins),
               "null pointer");
  ovg::CacheView c{};
  c.data = static_cast<unsigned char*>(cache->data);
  c.scales = cache->scales;
  c.tables = sequences->tables;
  c.lengths = sequences->lengths;
  c.begins = sequences->begins;
  c.blocks = static_cast<int>(cache->blocks);
  c.block_shift = cache->block_tokens == 16 ? 4 : cache->block_tokens == 32 ? 5 : 6;
  c.kv_heads = static_cast<int>(cache->kv_heads);
  c.dim = static_cast<int>(cache->head_dim);
  c.count = static_cast<int>(sequences->count);
  c.table_width = static_cast<int>(sequences->table_width);
  c.rows = sequences->count == 0 ? 0 : static_cast<int>(sequences->rows);
  return c;
}

// Query heads of a kv head, for the attention and for its workspace's size.
int GroupOf(const ovg_kv_cache* cache, int64_t heads) {
  ovg::Require(heads >= cache->kv_heads && heads % cache->kv_heads == 0 &&
                   heads / cache->kv_heads <= 64,
               "heads must be 1 to 64 times kv_heads");
  return static_cast<int>(heads / cache->kv_heads);
}

// The splits' outputs, then their maxima and sums.
int64_t AttentionBytes(const ovg::CacheView& c, const ovg::CacheAttentionPlan& plan) {
  return static_cast<int64_t>(plan.slots) * (c.dim + 2) * static_cast<int64_t>(sizeof(float));
}

// The splits' sums and lists.
int64_t LogprobBytes(int64_t rows, int64_t top, int splits) {
  return splits == 1 ? 0 : rows * splits * (4 + 2 * top) * static_cast<int64_t>(sizeof(float));
}

}  // namespace

extern "C" {

int ovg_op_score(const float* logits, int32_t* prediction, float* confidence,
                 int64_t frames, int64_t codebooks, int64_t vocab,
                 uint32_t mask_id, float guidance, void* stream, char* error,
                 size_t error_len) {
  return Guard("score: ", error, error_len, [&] {
    ovg::Require(logits && prediction && confidence, "null pointer");
    ovg::Require(frames >= 1 && FitsInt(frames) && codebooks >= 1 &&
                     codebooks <= 64 && vocab >= 1 && vocab <= 1088,
                 "shape outside the kernel's range");
    auto s = static_cast<hipStream_t>(stream);
    Scratch<ovg::ScoreItem> item(1);
    const ovg::ScoreItem host{0, static_cast<int>(frames), 0, 0};
    ovg::Check(hipMemcpyAsync(item.data, &host, sizeof(host),
                              hipMemcpyHostToDevice, s),
               "upload");
    ovg::ScoreParams p{};
    p.logits = logits;
    p.items = item.data;
    p.item_count = 1;
    p.max_frames = static_cast<int>(frames);
    p.codebooks = static_cast<int>(codebooks);
    p.vocab = static_cast<int>(vocab);
    p.width = p.codebooks * p.vocab;
    p.mask_id = mask_id;
    p.guidance = guidance;
    p.prediction = prediction;
    p.confidence = confidence;
    ovg::LaunchScore(p, s);
    ovg::Check(hipStreamSynchronize(s), "score");
  });
}

int ovg_op_select(const int32_t* prediction, const float* confidence,
                  const float* noise, int32_t* codes, int32_t* unmasked_at,
                  int64_t codebooks, int64_t frames, int64_t count,
                  int32_t step, float layer_penalty, float temperature,
                  uint32_t mask_id, void* stream, char* error,
                  size_t error_len) {
  return Guard("select: ", error, error_len, [&] {
    ovg::Require(prediction && confidence && codes && unmasked_at,
                 "null pointer");
    ovg::Require(temperature <= 0.0F || noise != nullptr,
                 "noise required when the temperature is positive");
    ovg::Require(codebooks >= 1 && frames >= 1 &&
                     codebooks * frames <=
                         ovg::kSelectThreads * ovg::kSelectPerThread,
                 "codebooks * frames outside [1, 16384]");
    ovg::Require(count >= 0, "negative count");
    auto s = static_cast<hipStream_t>(stream);
    Scratch<ovg::SelectItem> item(1);
    const ovg::SelectItem host{static_cast<int>(frames), 0, 0, 0};
    ovg::Check(hipMemcpyAsync(item.data, &host, sizeof(host),
                              hipMemcpyHostToDevice, s),
               "upload");
    ovg::SelectParams p{};
    p.prediction = prediction;
    p.confidence = confidence;
    p.noise = noise;
    p.codes = codes;
    p.unmasked_at = unmasked_at;
    p.ids = nullptr;
    p.items = item.data;
    p.item_count = 1;
    p.codebooks = static_cast<int>(codebooks);
    p.layer_penalty = layer_penalty;
    p.temperature = temperature;
    p.mask_id = mask_id;
    p.plan = nullptr;
    p.epoch = nullptr;
    p.single = {step, static_cast<int>(std::min<int64_t>(count, 1 << 30)), 0, 0};
    ovg::LaunchSelect(p, static_cast<int>(codebooks * frames), s);
    ovg::Check(hipStreamSynchronize(s), "select");
  });
}

int ovg_op_linear(const void* x, const void* w, float* y, int64_t rows,
                  int64_t in, int64_t out, int accumulate, void* stream,
                  char* error, size_t error_len) {
  return Guard("linear: ", error, error_len, [&] {
    ovg::Require(x && w && y, "null pointer");
    ovg::Require(rows >= 1 && in >= 64 && out >= 1 && FitsInt(rows) &&
                     FitsInt(in) && FitsInt(out),
                 "empty or oversized shape");
    auto s = static_cast<hipStream_t>(stream);
    const auto epi =
        accumulate ? ovg::Epilogue::kAccumulate : ovg::Epilogue::kStore;
    const ovg::GemmPlan plan = ovg::PlanGemm(
        static_cast<int>(rows), static_cast<int>(out), static_cast<int>(in), epi, true);
    Scratch<float> partials(plan.partial_floats);
    ovg::GemmParams p{};
    p.x = static_cast<const ovg::half_t*>(x);
    p.w = static_cast<const ovg::half_t*>(w);
    p.lda = static_cast<int>(in);
    p.ldb = static_cast<int>(in);
    p.m = static_cast<int>(rows);
    p.n = static_cast<int>(out);
    p.k = static_cast<int>(in);
    p.splits = plan.splits;
    p.partials = partials.data;
    p.y = y;
    p.ldc = static_cast<int>(out);
    ovg::LaunchGemm(p, plan, epi, s);
    ovg::Check(hipStreamSynchronize(s), "linear");
  });
}

int ovg_op_linear_packed(const void* x, const void* w, float* y, int64_t rows,
                         int64_t in, int64_t out, int accumulate, int64_t tile_rows,
                         int64_t tile_cols, void* stream, char* error, size_t error_len) {
  return Guard("linear: ", error, error_len, [&] {
    ovg::Require(x && w && y, "null pointer");
    ovg::Require(rows >= 1 && in >= 64 && out >= 1 && FitsInt(rows) &&
                     FitsInt(in) && FitsInt(out),
                 "empty or oversized shape");
    const bool rows_ok = tile_rows == 32 || tile_rows == 64 || tile_rows == 96 || tile_rows == 128;
    const bool narrow = (tile_cols == 128 || tile_cols == 64 || tile_cols == 32) && rows_ok;
    const bool wide = tile_cols == 256 && (tile_rows == 128 || tile_rows == 256);
    ovg::Require((tile_rows == 0 && tile_cols == 0) || narrow || wide,
                 "tile must be 0 x 0 (planned), 32/64/96/128 x 128, 64 or 32, 128 x 256 or "
                 "256 x 256");
    auto s = static_cast<hipStream_t>(stream);
    const auto epi =
        accumulate ? ovg::Epilogue::kAccumulate : ovg::Epilogue::kStore;
    Scratch<ovg::half_t> packed(ovg::PackedWeightHalves(static_cast<int>(out),
                                                        static_cast<int>(in)));
    ovg::PackWeights(static_cast<const ovg::half_t*>(w), nullptr, static_cast<int>(out),
                     static_cast<int>(in), ovg::PackMap::kIdentity, 0, packed.data, s);
    ovg::PackedPlan plan = ovg::PlanPacked(static_cast<int>(rows), static_cast<int>(out),
                                           static_cast<int>(in), epi);
    if (tile_rows != 0) {
      plan.n_main = 0;  // one launch of the forced tile
      plan.xb = static_cast<int>(tile_rows / 32);
      plan.wb = tile_cols == 256 ? 2 : 1;
      plan.nw = tile_cols == 64 ? 2 : tile_cols == 32 ? 1 : 4;
      plan.tiles = (static_cast<int>(rows) + static_cast<int>(tile_rows) - 1) /
                   static_cast<int>(tile_rows) *
                   ((static_cast<int>(out) + static_cast<int>(tile_cols) - 1) /
                    static_cast<int>(tile_cols));
    }
    ovg::GemmParams p{};
    p.x = static_cast<const ovg::half_t*>(x);
    p.w = packed.data;
    p.lda = static_cast<int>(in);
    p.ldb = static_cast<int>(in);
    p.m = static_cast<int>(rows);
    p.n = static_cast<int>(out);
    p.k = static_cast<int>(in);
    p.splits = plan.splits;
    p.y = y;
    p.ldc = static_cast<int>(out);
    ovg::LaunchPacked(p, plan, epi, s);
    ovg::Check(hipStreamSynchronize(s), "linear");
  });
}

int ovg_op_rmsnorm(const float* input, const float* weight, void* output,
                   int64_t rows, int64_t width, float epsilon, void* stream,
                   char* error, size_t error_len) {
  return Guard("rmsnorm: ", error, error_len, [&] {
    ovg::Require(input && weight && output, "null pointer");
    ovg::Require(rows >= 1 && FitsInt(rows), "bad rows");
    auto s = static_cast<hipStream_t>(stream);
    ovg::LaunchRmsNorm(input, nullptr, weight,
                       static_cast<ovg::half_t*>(output), static_cast<int>(rows),
                       static_cast<int>(width), epsilon, s);
    ovg::Check(hipStreamSynchronize(s), "rmsnorm");
  });
}

int ovg_op_attention(const void* qkv, void* output, int64_t rows,
                     int64_t heads, int64_t kv_heads,
                     const int64_t* sequences, int64_t count, void* stream,
                     char* error, size_t error_len) {
  return Guard("attention: ", error, error_len, [&] {
    ovg::Require(qkv && output && sequences, "null pointer");
    ovg::Require(rows >= 1 && FitsInt(rows) && heads >= 1 && kv_heads >= 1 &&
                     heads <= 64 && count >= 1,
                 "bad shape");
    const int ld_qkv = static_cast<int>((heads + 2 * kv_heads) * 128);
    std::vector<ovg::AttentionWork> work;
    int64_t end = 0;
    for (int64_t i = 0; i < count; ++i) {
      const int64_t first = sequences[2 * i], length = sequences[2 * i + 1];
      ovg::Require(first >= 0 && length >= 1 && first + length <= rows,
                   "sequence outside the rows");
      ovg::Require(first % ovg::kSequenceAlign == 0,
                   "sequence start must be a multiple of 16");
      end = std::max(end, first + (length + 31) / 32 * 32);
      for (int64_t q = 0; q < length; q += 32)
        work.push_back({static_cast<int>(first + q),
                        static_cast<int>(std::min<int64_t>(32, length - q)),
                        static_cast<int>(first), static_cast<int>(length)});
    }
    int exact_count = 0, exact_rounds = 0;
    ovg::PlanAttentionWork(work, &exact_count, &exact_rounds);
    auto s = static_cast<hipStream_t>(stream);
    // Keys are read in whole 32-row tiles: q and k go head-major into a
    // buffer padded past the last tile, V into V^T blocks.
    const int padded = static_cast<int>(std::max(end, rows));
    const int ldvt = (padded + 15) / 16 * 16;
    const int ldq = ldvt * 128;
    Scratch<ovg::half_t> qk(static_cast<std::size_t>(heads + kv_heads) * ldq);
    Scratch<ovg::half_t> vt(static_cast<std::size_t>(kv_heads) * 128 * ldvt);
    Scratch<ovg::AttentionWork> dwork(work.size());
    ovg::Check(hipMemsetAsync(qk.data, 0,
                              static_cast<std::size_t>(heads + kv_heads) * ldq * 2, s),
               "clear");
    ovg::Check(hipMemsetAsync(vt.data, 0,
                              static_cast<std::size_t>(kv_heads) * 128 * ldvt * 2, s),
               "clear");
    ovg::Check(hipMemcpyAsync(dwork.data, work.data(),
                              work.size() * sizeof(ovg::AttentionWork),
                              hipMemcpyHostToDevice, s),
               "upload");
    ovg::LaunchAttentionLayout(static_cast<const ovg::half_t*>(qkv), ld_qkv, qk.data, ldq,
                               vt.data, ldvt, static_cast<int>(rows),
                               static_cast<int>(heads), static_cast<int>(kv_heads), s);
    ovg::AttentionParams p{};
    p.qk = qk.data;
    p.vt = vt.data;
    p.out = static_cast<ovg::half_t*>(output);
    p.work = dwork.data;
    p.work_count = static_cast<int>(work.size());
    p.exact_count = exact_count;
    p.exact_rounds = exact_rounds;
    p.ld_qk = ldq;
    p.ldvt = ldvt;
    p.heads = static_cast<int>(heads);
    p.kv_heads = static_cast<int>(kv_heads);
    p.scale_log2 = 1.44269504088896341F / 11.313708498984761F;
    ovg::LaunchAttention(p, s);
    ovg::Check(hipStreamSynchronize(s), "attention");
  });
}

int ovg_op_cache_write(const ovg_kv_cache* cache, const ovg_kv_sequences* sequences,
                       const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                       int type, void* stream, char* error, size_t error_len) {
  return Guard("cache write: ", error, error_len, [&] {
    ovg::CacheWriteParams p{};
    p.cache = ViewOf(cache, sequences);
    const ovg::DType t = TypeOf(type, true);
    const int64_t width = cache->kv_heads * cache->head_dim;
    RequireStride(k_stride, width);
    RequireStride(v_stride, width);
    if (p.cache.rows == 0)
      return;
    ovg::Require(k && v, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    p.x[0] = k;
    p.x[1] = v;
    p.stride[0] = k_stride;
    p.stride[1] = v_stride;
    ovg::LaunchCacheWrite(p, t, s);
  });
}

int ovg_op_cache_read(const ovg_kv_cache* cache, const ovg_kv_sequences* sequences, void* k,
                      void* v, int64_t k_stride, int64_t v_stride, int type, void* stream,
                      char* error, size_t error_len) {
  return Guard("cache read: ", error, error_len, [&] {
    ovg::CacheReadParams p{};
    p.cache = ViewOf(cache, sequences);
    const ovg::DType t = TypeOf(type, true);
    const int64_t width = cache->kv_heads * cache->head_dim;
    RequireStride(k_stride, width);
    RequireStride(v_stride, width);
    if (p.cache.rows == 0)
      return;
    ovg::Require(k && v, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    p.x[0] = k;
    p.x[1] = v;
    p.stride[0] = k_stride;
    p.stride[1] = v_stride;
    ovg::LaunchCacheRead(p, t, s);
  });
}

int64_t ovg_op_cache_attention_workspace(const ovg_kv_cache* cache,
                                         const ovg_kv_sequences* sequences, int64_t heads) {
  try {
    const ovg::CacheView c = ViewOf(cache, sequences);
    return AttentionBytes(c, ovg::PlanCacheAttention(c, GroupOf(cache, heads)));
  } catch (const std::exception&) {
    return -1;  // as the call itself will say
  }
}

int ovg_op_cache_attention(const ovg_kv_cache* cache, const ovg_kv_sequences* sequences,
                           const void* q, void* out, int64_t q_stride, int64_t out_stride,
                           int64_t heads, float scale, int causal, int type, void* workspace,
                           int64_t workspace_bytes, void* stream, char* error,
                           size_t error_len) {
  return Guard("cache attention: ", error, error_len, [&] {
    ovg::CacheAttentionParams p{};
    p.cache = ViewOf(cache, sequences);
    const ovg::DType t = TypeOf(type, false);
    p.group = GroupOf(cache, heads);
    const float scale_log2 = std::fabs(scale) * 1.44269504088896341F;
    ovg::Require(scale_log2 - scale_log2 == 0.0F, "scale must be finite, also times log2(e)");
    RequireStride(q_stride, heads * cache->head_dim);
    RequireStride(out_stride, heads * cache->head_dim);
    if (p.cache.rows == 0)
      return;
    ovg::Require(q && out, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    p.group_inverse = ((1 << 16) + p.group - 1) / p.group;
    p.group_magic = ((1ull << 36) + p.group - 1) / p.group;
    const ovg::CacheAttentionPlan plan = ovg::PlanCacheAttention(p.cache, p.group);
    const int64_t bytes = AttentionBytes(p.cache, plan);
    ovg::Require(bytes == 0 || (workspace && workspace_bytes >= bytes && Aligned16(workspace)),
                 "workspace of " + std::to_string(bytes) + " bytes needed, 16-byte aligned");
    p.tile_shift = plan.tile_shift;
    p.splits = plan.splits;
    p.own_shift = plan.own_shift;
    p.partial_o = static_cast<float*>(workspace);
    p.partial_m = p.partial_o + plan.slots * p.cache.dim;
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.causal = causal != 0;
    p.scale_log2 = scale_log2;
    p.negate = scale < 0.0F;
    ovg::LaunchCacheAttention(p, t, s);
  });
}

int64_t ovg_op_token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t top) {
  if (rows < 0 || rows > (1 << 23) || vocab < 1 || !FitsInt(vocab) || top < 0 ||
      top > ovg::kMostAlternatives)
    return -1;
  return LogprobBytes(rows, top,
                      ovg::PlanLogprobs(static_cast<int>(rows), static_cast<int>(vocab)));
}

int ovg_op_token_logprobs(const void* logits, const void* uncond, int64_t rows, int64_t vocab,
                          int64_t stride, int64_t uncond_stride, float guidance,
                          int64_t mask_id, const int32_t* tokens, int64_t top, float* logprob,
                          float* entropy, int32_t* top_ids, float* top_logprobs, int type,
                          void* workspace, int64_t workspace_bytes, void* stream, char* error,
                          size_t error_len) {
  return Guard("token logprobs: ", error, error_len, [&] {
    const ovg::DType t = TypeOf(type, true);
    // A work-group of 256 a row, in a grid that counts 2^32 threads.
    ovg::Require(rows >= 0 && rows <= (1 << 23), "rows outside [0, 2^23]");
    ovg::Require(vocab >= 1 && FitsInt(vocab), "vocab outside [1, 2^30]");
    ovg::Require(top >= 0 && top <= ovg::kMostAlternatives, "top outside [0, 32]");
    ovg::Require(mask_id >= -1 && mask_id < (int64_t{1} << 31), "mask_id must be -1 or a token");
    ovg::Require(guidance == guidance && guidance - guidance == 0.0F, "guidance must be finite");
    RequireStride(stride, vocab);
    if (uncond != nullptr)
      RequireStride(uncond_stride, vocab);
    ovg::Require((tokens == nullptr) == (logprob == nullptr), "tokens and logprob go together");
    if (rows == 0)
      return;
    ovg::Require(logits != nullptr, "null pointer");
    ovg::Require(top == 0 || (top_ids && top_logprobs), "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    ovg::LogprobParams p{};
    p.splits = ovg::PlanLogprobs(static_cast<int>(rows), static_cast<int>(vocab));
    const int64_t bytes = LogprobBytes(rows, top, p.splits);
    ovg::Require(bytes == 0 || (workspace && workspace_bytes >= bytes && Aligned16(workspace)),
                 "workspace of " + std::to_string(bytes) + " bytes needed, 16-byte aligned");
    p.states = static_cast<float*>(workspace);
    p.logits = logits;
    p.uncond = uncond;
    p.stride = stride;
    p.uncond_stride = uncond_stride;
    p.tokens = tokens;
    p.guidance = guidance;
    p.rows = static_cast<int>(rows);
    p.vocab = static_cast<int>(vocab);
    p.mask_id = static_cast<int>(mask_id);
    p.top = static_cast<int>(top);
    p.logprob = logprob;
    p.entropy = entropy;
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    ovg::LaunchLogprobs(p, t, s);
  });
}

}  // extern "C"
