// Device-side pieces that the operator kernels share. Device code: include
// from .hip files only.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "hip/core.h"
#include "collectives/reduce_fns.h"

namespace glooamd {
namespace hip {

// Makes `device` current for a launch and puts the caller's back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    GA_HIP_CHECK(hipGetDevice(&before_));
    if (device != before_) {
      GA_HIP_CHECK(hipSetDevice(device));
      changed_ = true;
    }
  }
  ~DeviceGuard() {
    if (changed_) {
      (void)hipSetDevice(before_);
    }
  }
  DeviceGuard(const DeviceGuard&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

__device__ inline float toFloat(float v) {
  return v;
}
__device__ inline float toFloat(__half v) {
  return __half2float(v);
}
__device__ inline float toFloat(__hip_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ inline T fromFloat(float v);
template <>
__device__ inline float fromFloat<float>(float v) {
  return v;
}
template <>
__device__ inline __half fromFloat<__half>(float v) {
  return __float2half(v);
}
template <>
__device__ inline __hip_bfloat16 fromFloat<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}

// Workgroups along x: a launch has fewer than 2^32 threads there.
inline unsigned groupsOf(int64_t groups, int threads) {
  GA_ENFORCE_LE(groups, UINT32_MAX / threads);
  return static_cast<unsigned>(groups);
}

// Stores past the caches where what a kernel writes would not stay in them
// anyhow: half of the 256 MB behind the dies' own ones. Below that the next
// kernel finds it there.
constexpr int64_t kStreamFrom = 128 << 20;

// 16 bytes of T, moved as one load or store.
template <typename T>
struct alignas(16) Vec16 {
  static constexpr int kSize = 16 / sizeof(T);
  T v[kSize];
};

template <typename F>
void dispatchFloat(DType d, const char* what, F&& f) {
  switch (d) {
    case DType::F32:
      return f(float{});
    case DType::F16:
      return f(__half{});
    case DType::BF16:
      return f(__hip_bfloat16{});
    default:
      GA_ENFORCE(false, what, ": float32, float16 or bfloat16 is needed");
  }
}

inline bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// --- e4m3 values with power-of-two scales -----------------------------------

// The e8m0 byte of a block whose largest absolute value has the fp32 bits
// `amax`: the least 2^e (e >= -127) with amax / 2^e <= 448. 448 is 1.75 *
// 2^8, so e is amax's exponent - 8, one more where its mantissa is above
// 1.75: adding the distance from 1.75 to 2 carries into the exponent just
// then. 127 (2^0) for a block of zeros, 255 (NaN) where one is inf or NaN:
// the bits of those are above every finite number's.
__device__ inline uint32_t fp8ScaleByte(uint32_t amax) {
  if (amax >= 0x7f800000u) {
    return 255u;
  }
  if (amax == 0) {
    return 127u;
  }
  const int e = static_cast<int>((amax + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(e < 0 ? 0 : e);
}

// 1 / scale, exact: 2^(127 - byte); NaN for 255.
__device__ inline float fp8InverseScale(uint32_t byte) {
  if (byte == 255u) {
    return __uint_as_float(0x7fc00000u);
  }
  // 2^-127 (byte 254) is below fp32's normal numbers
  return byte == 254u ? __uint_as_float(0x00400000u)
                      : __uint_as_float((254u - byte) << 23);
}

// Four e4m3 bytes, rounded to nearest even.
__device__ inline uint32_t fp8Pack4(float a, float b, float c, float d) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
  return static_cast<uint32_t>(p);
}

} // namespace hip
} // namespace glooamd
