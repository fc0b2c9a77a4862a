// Elements of float32, bfloat16 and float16 in memory; arithmetic is in float32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cfh {

enum { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };      // CFH_FLOAT32, CFH_BFLOAT16, CFH_FLOAT16

using bf16 = __bf16;
using f16 = _Float16;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return (float)x; }
__device__ __forceinline__ float to_float(f16 x) { return (float)x; }
// to the nearest, ties to even
template <typename T>
__device__ __forceinline__ T from_float(float x) { return (T)x; }

}  // namespace cfh
