// Argument checks shared by the torch bindings (bindings.cpp, bindings_paged.cpp).
#pragma once
#include <limits>

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

namespace {
const auto BF = torch::kBFloat16;
const auto I32 = torch::kInt32;
const auto F32 = torch::kFloat32;
constexpr int HD = 256;

inline hipStream_t stream_of(const torch::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void chk(const torch::Tensor& t, torch::ScalarType dt, const char* name, bool dev) {
  if (dev) TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == dt, name, " has wrong dtype ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// Row view: (rows, width, row stride).
struct Rows {
  int n;
  long w;
  long ld;
};
inline Rows rows(const torch::Tensor& t, torch::ScalarType dt, const char* name, bool dev) {
  TORCH_CHECK((!dev || t.is_cuda()) && t.scalar_type() == dt, name, ": wrong device/dtype");
  if (t.dim() == 1) {
    TORCH_CHECK(t.stride(0) == 1, name, " not contiguous");
    return {1, (long)t.size(0), (long)t.size(0)};
  }
  TORCH_CHECK(t.dim() == 2 && t.stride(1) == 1, name, " must be [n, w] with unit inner stride");
  return {(int)t.size(0), (long)t.size(1), (long)t.stride(0)};
}

inline void chk16(const torch::Tensor& t, long ld, const char* name) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && ld % 8 == 0, name,
              " must be 16-byte aligned rows");
}

// The fp8 KV cache: E4M3FN codes, as torch.float8_e4m3fn or raw uint8 bytes.
inline void chk_kv8(const torch::Tensor& t, const char* name, bool dev) {
  if (dev) TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == torch::kFloat8_e4m3fn || t.scalar_type() == torch::kByte, name,
              " must be float8_e4m3fn (or uint8 codes), got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

inline void chk_pos(const torch::Tensor& pos, bool dev) {
  TORCH_CHECK((!dev || pos.is_cuda()) && pos.scalar_type() == I32 && pos.numel() >= 1,
              "pos must be an int32 GPU tensor with at least one element");
}

inline void raise_on(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " failed: ", hipGetErrorString(e));
}

// Scales of an fp8 cache.
inline void kv_scales(double k_scale, double v_scale) {
  // as fp32, the kernels' type: normal and finite, so that 1/scale is finite too
  const auto ok = [](double s) {
    const float f = (float)s;
    return f >= std::numeric_limits<float>::min() && f <= std::numeric_limits<float>::max();
  };
  TORCH_CHECK(ok(k_scale) && ok(v_scale),
              "k_scale and v_scale must be positive, finite and not subnormal as fp32");
}
}  // namespace
