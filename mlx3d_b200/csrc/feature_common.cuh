// Shared pieces of the feature-field kernels (distill.cu, teacher.cu,
// decode.cu): element types and the teacher cache's record layout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>

#include "gs_common.cuh"

namespace gs {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The lowest finite value of a type: programs write it where a class is masked.
template <typename T>
__device__ __forceinline__ float lowest_of();
template <>
__device__ __forceinline__ float lowest_of<float>() { return -FLT_MAX; }
template <>
__device__ __forceinline__ float lowest_of<__half>() { return -65504.0f; }
template <>
__device__ __forceinline__ float lowest_of<__nv_bfloat16>() { return __uint_as_float(0xff7f0000u); }

// Pairs of float32 values in 64-bit registers: sm_100 multiplies and adds two at
// once.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(uint32_t lo, uint32_t hi) { return f2(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ void split(F2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Two neighbouring elements (p aligned to both) as floats, and back.
__device__ __forceinline__ F2 load_pair(const float* p) { return *reinterpret_cast<const F2*>(p); }
__device__ __forceinline__ F2 load_pair(const __half* p) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(p));
  return f2(v.x, v.y);
}
__device__ __forceinline__ F2 load_pair(const __nv_bfloat16* p) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  return f2(w << 16, w & 0xffff0000u);
}
__device__ __forceinline__ void store_pair(float* p, F2 v) { *reinterpret_cast<F2*>(p) = v; }
__device__ __forceinline__ void store_pair(__half* p, F2 v) {
  float lo, hi;
  split(v, lo, hi);
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(lo, hi);
}
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, F2 v) {
  float lo, hi;
  split(v, lo, hi);
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(lo, hi);
}

inline bool dtype_ok(int dtype) { return dtype == GS_F32 || dtype == GS_F16 || dtype == GS_BF16; }

// A teacher cache record: [offset f32][scale f32][index int16 x k][codes],
// padded to 16 bytes so that every record starts on a 16-byte boundary (k = 8
// with 8 bits is exactly one 32-byte sector).
__host__ __device__ __forceinline__ int record_bytes(int k, int bits) {
  return (8 + 2 * k + (k * bits + 7) / 8 + 15) / 16 * 16;
}
__device__ __forceinline__ int record_code(const uint8_t* codes, int e, int bits) {
  return bits == 8 ? codes[e] : (codes[e >> 1] >> ((e & 1) * 4)) & 15;
}
// One rounding: code * scale is exact inside the fma.
__device__ __forceinline__ float record_value(float offset, float scale, int code) {
  return __fmaf_rn(-(float)code, scale, offset);
}

}  // namespace gs
