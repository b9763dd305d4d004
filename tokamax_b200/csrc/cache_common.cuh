// What the kernels of the quantised key / value cache have in common: its layout (SplashKvCache), conversions, the
// checks of arguments.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "splash_common.cuh"

namespace sb {

constexpr float kE4m3Max = 448.0f;

// Bytes of a row's codes and of its scales.
__host__ __device__ constexpr int cache_row_bytes(int format, int width) { return format == SPLASH_CACHE_INT4 ? width / 2 : width; }
__host__ __device__ constexpr int cache_scale_bytes(int format, int width, int group) {
  return format == SPLASH_CACHE_INT4 ? 4 * (width / group) : 2;
}

__device__ __forceinline__ float bf16_bits_to_float(uint32_t bits) { return __uint_as_float(bits << 16); }

// Two bf16 or f16 values of a word.
__device__ __forceinline__ void unpack16(int dtype, uint32_t w, float& lo, float& hi) {
  if (dtype == SPLASH_BF16) {
    lo = bf16_bits_to_float(w);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(int dtype, float lo, float hi) {
  return dtype == SPLASH_BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}
// Eight values of one of the three element types to 16-byte aligned memory.
__device__ __forceinline__ void store8(void* base, int dtype, int64_t at, const float (&x)[8]) {
  if (dtype == SPLASH_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
      make_uint4(pack16(dtype, x[0], x[1]), pack16(dtype, x[2], x[3]), pack16(dtype, x[4], x[5]), pack16(dtype, x[6], x[7]));
}

// Two e4m3 codes (the low one first) as f16, which holds every one of them.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}

inline int log2_of(int power_of_two) {
  int n = 0;
  while ((1 << n) < power_of_two) ++n;
  return n;
}

int check_cache(const SplashKvCache& c);                              // SPLASH_OK or why not
int check_cache_tensor(const SplashTensor& t, bool f32_too);          // element type, strides, alignment

}  // namespace sb
