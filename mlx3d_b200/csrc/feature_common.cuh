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

inline int elem_size(int dtype) { return dtype == GS_F32 ? 4 : 2; }
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
