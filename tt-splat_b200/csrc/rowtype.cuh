// Element types of the row kernels (table rows, label logits): fp32, bf16 or fp16 in memory, fp32 in
// registers; a result is rounded to the memory type once, when it is stored.
#pragma once
#include <cuda_fp16.h>

#include <initializer_list>

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

// Two 16-bit elements of a word, the first in the low half.
template <class T>
__device__ __forceinline__ float2 unpack2(unsigned w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(unsigned w) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
template <class T>
__device__ __forceinline__ unsigned pack2(float a, float b);
template <>
__device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  unsigned w;
  memcpy(&w, &h, 4);
  return w;
}
template <>
__device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  unsigned w;
  memcpy(&w, &h, 4);
  return w;
}

// Memory units of VB bytes (16, 4 or 2) holding VB / sizeof(T) elements.
template <int VB>
struct UnitWord;
template <>
struct UnitWord<16> { using type = uint4; };
template <>
struct UnitWord<4> { using type = unsigned; };
template <>
struct UnitWord<2> { using type = unsigned short; };

template <class T, int VB>
struct Unit {
  static constexpr int E = VB / (int)sizeof(T);
  using W = typename UnitWord<VB>::type;
  W w;
  __device__ __forceinline__ Unit() {}
  __device__ __forceinline__ explicit Unit(W x) : w(x) {}
  __device__ __forceinline__ void get(float (&v)[E]) const {
    if constexpr (VB == 2) {
      T t;
      memcpy(&t, &w, 2);
      v[0] = to_f32(t);
    } else {
      unsigned x[VB / 4];
      memcpy(x, &w, VB);
#pragma unroll
      for (int i = 0; i < VB / 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          v[i] = __uint_as_float(x[i]);
        } else {
          const float2 f = unpack2<T>(x[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[E]) {
    if constexpr (VB == 2) {
      const T t = from_f32<T>(v[0]);
      memcpy(&w, &t, 2);
    } else {
      unsigned x[VB / 4];
#pragma unroll
      for (int i = 0; i < VB / 4; ++i) {
        if constexpr (sizeof(T) == 4)
          x[i] = __float_as_uint(v[i]);
        else
          x[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
      }
      memcpy(&w, x, VB);
    }
  }
};

// Calls f with a value of the element type `type` names (TTS_ROW_*), the caller has checked the range.
template <class F>
inline int with_row_type(int type, F f) {
  if (type == TTS_ROW_F32) return f(float());
  if (type == TTS_ROW_BF16) return f(__nv_bfloat16());
  return f(__half());
}

// Whether each pointer lies on a multiple of n bytes: a misaligned access ends the context, so that the entry
// points refuse it.
inline bool aligned_to(size_t n, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % n) return false;
  return true;
}
// Whether R rows of C elements, stride apart, share memory with bytes [q, q + n): results are written while other
// blocks still read the rows.
inline bool rows_overlap(const void* rows, long long R, long long C, long long stride, size_t elem, const void* q,
                         long long n) {
  if (!rows || !q || R <= 0 || C <= 0 || n <= 0) return false;
  const char *p = static_cast<const char*>(rows), *o = static_cast<const char*>(q);
  const long long far = (R - 1) * stride * (long long)elem, row = C * (long long)elem;
  return p + (far < 0 ? far : 0) < o + n && o < p + (far > 0 ? far : 0) + row;
}
inline size_t row_elem(int type) { return type == TTS_ROW_F32 ? 4 : 2; }

// An index or label as given (int32 or int64).
__device__ __forceinline__ long long load_index(const void* p, int is64, long long n) {
  return is64 ? __ldg(static_cast<const long long*>(p) + n) : (long long)__ldg(static_cast<const int*>(p) + n);
}

}  // namespace tts
