// What the device operators' entry points share: the error message, the checks
// of arguments that come before every launch.
#ifndef OMNIVOICE_AMD_OPS_HPP_
#define OMNIVOICE_AMD_OPS_HPP_

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <string>

#include "../../include/omnivoice_mi355x.h"
#include "cache.hpp"
#include "kernels.hpp"

namespace ovg::ops {

inline void SetError(char* error, std::size_t len, const std::string& message) {
  if (error == nullptr || len == 0)
    return;
  const std::size_t n = std::min(len - 1, message.size());
  std::memcpy(error, message.data(), n);
  error[n] = '\0';
}

template <typename F>
int Guard(const char* prefix, char* error, std::size_t len, F&& body) {
  try {
    body();
    return OVG_OK;
  } catch (const std::exception& failure) {
    SetError(error, len, std::string(prefix) + failure.what());
    return OVG_ERROR;
  }
}

inline bool FitsInt(int64_t v) { return v >= 0 && v <= (int64_t{1} << 30); }

// A launch has to go to a device of its own: with another device current the
// kernel would run there, or fail in ways that depend on peer access.
inline void RequireCurrentDevice(hipStream_t stream) {
  if (stream == nullptr)
    return;  // the current device's own
  hipDevice_t of_stream = 0;
  int current = 0;
  ovg::Check(hipStreamGetDevice(stream, &of_stream), "hipStreamGetDevice");
  ovg::Check(hipGetDevice(&current), "hipGetDevice");
  ovg::Require(of_stream == current, "the stream is not the current device's");
}

inline bool Aligned16(const void* p) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0; }

inline ovg::DType TypeOf(int type, bool with_f32) {
  ovg::Require(type == OVG_F16 || type == OVG_BF16 || (with_f32 && type == OVG_F32),
               with_f32 ? "type must be fp16, bf16 or float32" : "type must be fp16 or bf16");
  return static_cast<ovg::DType>(type);
}

inline void RequireStride(int64_t stride, int64_t width) {
  ovg::Require(stride >= width && stride <= (int64_t{1} << 40), "row stride below the row's width");
}

}  // namespace ovg::ops

#endif  // OMNIVOICE_AMD_OPS_HPP_
