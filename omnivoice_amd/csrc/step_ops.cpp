// Entry points of a token's step around the cache (include/omnivoice_mi355x.h, "A
// token's step"): their checks, and the launchers' parameters.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ops.hpp"
#include "step.hpp"

namespace {

using namespace ovg::ops;

void RequireRows(int64_t rows, int64_t width) {
  ovg::Require(rows >= 0 && rows <= ovg::kMostRows, "rows outside [0, 2^22)");
  ovg::Require(width >= 1 && width <= ovg::kMostWidth, "width outside [1, 65536]");
}

bool Finite(float v) { return v - v == 0.0F; }

}  // namespace

extern "C" {

int ovg_op_add_rmsnorm(const void* x, int64_t x_stride, int x_type, const void* residual,
                       int64_t residual_stride, void* total, int64_t total_stride,
                       int residual_type, const float* weight, void* out, int64_t out_stride,
                       int out_type, float* scales, int64_t rows, int64_t width, float epsilon,
                       void* stream, char* error, size_t error_len) {
  return Guard("add rmsnorm: ", error, error_len, [&] {
    RequireRows(rows, width);
    const ovg::DType in = TypeOf(x_type, true);
    const ovg::DType to = out_type == OVG_E4M3 ? ovg::DType::kE4m3 : TypeOf(out_type, true);
    ovg::DType held = ovg::DType::kE4m3;  // none
    if (residual != nullptr || total != nullptr) {
      held = TypeOf(residual_type, true);
      ovg::Require(held == in || held == ovg::DType::kF32,
                   "the residual must be float32 or of x's type");
      RequireStride(residual_stride, width);
      RequireStride(total_stride, width);
      ovg::Require(residual && total, "residual and total go together");
    }
    ovg::Require((to == ovg::DType::kE4m3) == (scales != nullptr),
                 "scales go with an 8-bit output");
    ovg::Require(Finite(epsilon) && epsilon > 0.0F, "epsilon must be positive");
    RequireStride(x_stride, width);
    RequireStride(out_stride, width);
    if (rows == 0)
      return;
    ovg::Require(x && weight && out, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    ovg::RowParams p{};
    p.x = x;
    p.second = residual;
    p.total = total;
    p.weight = weight;
    p.out = out;
    p.scales = scales;
    p.x_stride = x_stride;
    p.second_stride = residual_stride;
    p.total_stride = total_stride;
    p.out_stride = out_stride;
    p.rows = static_cast<int>(rows);
    p.width = static_cast<int>(width);
    p.eps = epsilon;
    ovg::LaunchAddNorm(p, in, held, to, s);
  });
}

int ovg_op_quantize8(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                    int type, void* codes, int64_t codes_stride, float* scales, int64_t rows,
                    int64_t width, void* stream, char* error, size_t error_len) {
  return Guard("quantize8: ", error, error_len, [&] {
    RequireRows(rows, width);
    const ovg::DType in = TypeOf(type, true);
    RequireStride(x_stride, width);
    RequireStride(codes_stride, width);
    if (gate != nullptr)
      RequireStride(gate_stride, width);
    if (rows == 0)
      return;
    ovg::Require(x && codes && scales, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    ovg::RowParams p{};
    p.x = x;
    p.second = gate;
    p.out = codes;
    p.scales = scales;
    p.x_stride = x_stride;
    p.second_stride = gate_stride;
    p.out_stride = codes_stride;
    p.rows = static_cast<int>(rows);
    p.width = static_cast<int>(width);
    ovg::LaunchQuantize(p, in, s);
  });
}

int ovg_op_linear8(const void* x, int64_t x_stride, const float* x_scales, const void* w,
                   const float* w_scales, void* y, int64_t y_stride, int type, int64_t rows,
                   int64_t in, int64_t out, void* stream, char* error, size_t error_len) {
  return Guard("linear8: ", error, error_len, [&] {
    ovg::Require(rows >= 0 && rows <= ovg::kMostRows, "rows outside [0, 2^22)");
    ovg::Require(in >= 16 && in % 16 == 0 && in <= ovg::kMostWidth,
                 "in must be a multiple of 16 in [16, 65536]");
    ovg::Require(out >= 0 && out <= ovg::kMostRows, "out outside [0, 2^22)");
    const ovg::DType to = TypeOf(type, true);
    RequireStride(x_stride, in);
    ovg::Require(x_stride % 16 == 0, "x's rows must be a multiple of 16 codes apart");
    RequireStride(y_stride, out);
    if (rows == 0 || out == 0)
      return;
    ovg::Require(x && x_scales && w && w_scales && y, "null pointer");
    ovg::Require(Aligned16(x) && Aligned16(w), "codes must be 16-byte aligned");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    ovg::Linear8Params p{};
    p.x = static_cast<const unsigned char*>(x);
    p.x_scales = x_scales;
    p.w = static_cast<const unsigned char*>(w);
    p.w_scales = w_scales;
    p.y = y;
    p.x_stride = x_stride;
    p.y_stride = y_stride;
    p.rows = static_cast<int>(rows);
    p.in = static_cast<int>(in);
    p.out = static_cast<int>(out);
    ovg::LaunchLinear8(p, to, s);
  });
}

int ovg_rotary_frequencies(int64_t rotary, double theta, int scaling, double factor,
                           double original_positions, float* frequencies, float* magnitude) {
  if (rotary < 2 || rotary % 2 != 0 || rotary > ovg::kMostRotaryDim || !(theta > 1.0) ||
      !std::isfinite(theta) || frequencies == nullptr || magnitude == nullptr)
    return OVG_ERROR;
  if (scaling < OVG_ROTARY_PLAIN || scaling > OVG_ROTARY_PARTS)
    return OVG_ERROR;
  if (scaling != OVG_ROTARY_PLAIN && !(factor >= 1.0 && std::isfinite(factor)))
    return OVG_ERROR;
  if (scaling == OVG_ROTARY_PARTS &&
      !(original_positions >= 1.0 && std::isfinite(original_positions)))
    return OVG_ERROR;
  constexpr double kTurn = 6.283185307179586477;
  constexpr double kFast = 32.0, kSlow = 1.0;  // turns over the original positions
  const int64_t half = rotary / 2;
  if (scaling == OVG_ROTARY_BASE && rotary > 2)
    theta *= std::pow(factor, static_cast<double>(rotary) / static_cast<double>(rotary - 2));
  // The pair that makes so many turns, counted as a real number.
  const auto pair_of = [&](double turns) {
    return static_cast<double>(half) * std::log(original_positions / (turns * kTurn)) /
           std::log(theta);
  };
  double low = 0.0, high = 0.0;
  if (scaling == OVG_ROTARY_PARTS) {
    low = std::max(std::floor(pair_of(kFast)), 0.0);
    high = std::min(std::ceil(pair_of(kSlow)), static_cast<double>(rotary - 1));
  }
  for (int64_t i = 0; i < half; ++i) {
    double f = std::pow(theta, -static_cast<double>(i) / static_cast<double>(half));
    if (scaling == OVG_ROTARY_LINEAR)
      f /= factor;
    if (scaling == OVG_ROTARY_PARTS) {
      const double at = (static_cast<double>(i) - low) / std::max(high - low, 1e-3);
      // Also where no pair turns once, and `high` is below the first one.
      const double slow = static_cast<double>(i) >= high ? 1.0 : std::min(std::max(at, 0.0), 1.0);
      f = f / factor * slow + f * (1.0 - slow);
    }
    frequencies[i] = static_cast<float>(f);
  }
  *magnitude =
      scaling == OVG_ROTARY_PARTS ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0F;
  return OVG_OK;
}

int ovg_op_rotary(const void* q, void* q_out, int64_t q_stride, int64_t q_out_stride,
                  int64_t heads, const void* k, void* k_out, int64_t k_stride,
                  int64_t k_out_stride, int64_t kv_heads, int type, int64_t rows,
                  int64_t head_dim, int64_t rotary, const float* frequencies, float magnitude,
                  int interleaved, const int32_t* positions, const ovg_kv_sequences* sequences,
                  const float* q_norm, const float* k_norm, float epsilon, void* stream,
                  char* error, size_t error_len) {
  return Guard("rotary: ", error, error_len, [&] {
    ovg::Require(rows >= 0 && rows <= ovg::kMostRotaryRows, "rows outside [0, 2^24)");
    ovg::Require(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= ovg::kMostRotaryDim,
                 "head_dim must be even in [2, 512]");
    ovg::Require(rotary >= 2 && rotary % 2 == 0 && rotary <= head_dim,
                 "rotary must be even in [2, head_dim]");
    ovg::Require(heads >= 1 && heads <= 4096 && kv_heads >= 0 && kv_heads <= 4096,
                 "heads outside [1, 4096] or kv_heads outside [0, 4096]");
    const ovg::DType t = TypeOf(type, true);
    ovg::Require(Finite(magnitude), "magnitude must be finite");
    ovg::Require((q_norm == nullptr && k_norm == nullptr) || (Finite(epsilon) && epsilon > 0.0F),
                 "epsilon must be positive");
    RequireStride(q_stride, heads * head_dim);
    RequireStride(q_out_stride, heads * head_dim);
    if (kv_heads > 0) {
      RequireStride(k_stride, kv_heads * head_dim);
      RequireStride(k_out_stride, kv_heads * head_dim);
    }
    ovg::Require((positions == nullptr) != (sequences == nullptr),
                 "either positions or sequences");
    ovg::RotaryParams p{};
    if (sequences != nullptr) {
      ovg::Require(sequences->count >= 0 && sequences->count <= (1 << 20),
                   "count outside [0, 2^20]");
      ovg::Require(sequences->rows == rows, "the sequences' rows are others");
      ovg::Require(sequences->count == 0 || (sequences->lengths && sequences->begins),
                   "null pointer");
      p.sequences.lengths = sequences->lengths;
      p.sequences.begins = sequences->begins;
      p.sequences.count = static_cast<int>(sequences->count);
      p.sequences.rows = static_cast<int>(rows);
      if (sequences->count == 0)
        return;
    }
    if (rows == 0)
      return;
    ovg::Require(q && q_out && frequencies && (kv_heads == 0 || (k && k_out)), "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    p.x[0] = q;
    p.x[1] = k;
    p.out[0] = q_out;
    p.out[1] = k_out;
    p.x_stride[0] = q_stride;
    p.x_stride[1] = k_stride;
    p.out_stride[0] = q_out_stride;
    p.out_stride[1] = k_out_stride;
    p.norm[0] = q_norm;
    p.norm[1] = k_norm;
    p.heads[0] = static_cast<int>(heads);
    p.heads[1] = static_cast<int>(kv_heads);
    p.rows = static_cast<int>(rows);
    p.dim = static_cast<int>(head_dim);
    p.rotary = static_cast<int>(rotary);
    p.frequencies = frequencies;
    p.positions = positions;
    p.magnitude = magnitude;
    p.eps = epsilon;
    ovg::LaunchRotary(p, interleaved != 0, t, s);
  });
}

int64_t ovg_op_sample_workspace(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > ovg::kMostRows || vocab < 1 || !FitsInt(vocab))
    return -1;
  return ovg::SampleWorkBytes(rows, vocab);
}

int ovg_op_sample(const void* logits, const void* uncond, int64_t rows, int64_t vocab,
                  int64_t stride, int64_t uncond_stride, float guidance, int64_t mask_id,
                  const ovg_sampling* sampling, const float* random, int32_t* tokens, int type,
                  void* workspace, int64_t workspace_bytes, void* stream, char* error,
                  size_t error_len) {
  return Guard("sample: ", error, error_len, [&] {
    const ovg::DType t = TypeOf(type, true);
    ovg::Require(rows >= 0 && rows <= ovg::kMostRows, "rows outside [0, 2^22)");
    ovg::Require(vocab >= 1 && FitsInt(vocab), "vocab outside [1, 2^30]");
    ovg::Require(mask_id >= -1 && mask_id < (int64_t{1} << 31), "mask_id must be -1 or a token");
    ovg::Require(Finite(guidance), "guidance must be finite");
    RequireStride(stride, vocab);
    if (uncond != nullptr)
      RequireStride(uncond_stride, vocab);
    ovg::Require(sampling != nullptr, "null pointer");
    const auto number = [](const float* each, float all, const char* what) {
      ovg::Require(each != nullptr || all == all, std::string(what) + " must be a number");
    };
    number(sampling->temperatures, sampling->temperature, "temperature");
    number(sampling->top_ps, sampling->top_p, "top_p");
    number(sampling->min_ps, sampling->min_p, "min_p");
    const int64_t bytes = ovg::SampleWorkBytes(rows, vocab);
    ovg::Require(bytes >= 0, "rows times vocab too large");
    if (rows == 0)
      return;
    ovg::Require(logits && random && tokens, "null pointer");
    auto s = static_cast<hipStream_t>(stream);
    RequireCurrentDevice(s);
    ovg::Require(bytes == 0 || (workspace && workspace_bytes >= bytes && Aligned16(workspace)),
                 "workspace of " + std::to_string(bytes) + " bytes needed, 16-byte aligned");
    ovg::SampleParams p{};
    p.work = static_cast<unsigned*>(workspace);
    p.logits = logits;
    p.uncond = uncond;
    p.stride = stride;
    p.uncond_stride = uncond_stride;
    p.guidance = guidance;
    p.rows = static_cast<int>(rows);
    p.vocab = static_cast<int>(vocab);
    p.mask_id = static_cast<int>(mask_id);
    p.random = random;
    p.tokens = tokens;
    p.temperature = sampling->temperature;
    p.top_k = sampling->top_k;
    p.top_p = sampling->top_p;
    p.min_p = sampling->min_p;
    p.temperatures = sampling->temperatures;
    p.top_ks = sampling->top_ks;
    p.top_ps = sampling->top_ps;
    p.min_ps = sampling->min_ps;
    ovg::LaunchSample(p, t, s);
  });
}

}  // extern "C"
