// Element types of the row kernels (table rows, label logits): fp32, bf16 or fp16 in memory, fp32 in
// registers; a result is rounded to the memory type once, when it is stored.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace tts {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Calls f with a value of the element type `type` names (TTS_ROW_*), the caller has checked the range.
template <class F>
inline int with_row_type(int type, F f) {
  if (type == TTS_ROW_F32) return f(float());
  if (type == TTS_ROW_BF16) return f(__nv_bfloat16());
  return f(__half());
}

// An index or label as given (int32 or int64).
__device__ __forceinline__ long long load_index(const void* p, int is64, long long n) {
  return is64 ? __ldg(static_cast<const long long*>(p) + n) : (long long)__ldg(static_cast<const int*>(p) + n);
}

}  // namespace tts
