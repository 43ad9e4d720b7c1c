// Loads and stores of V consecutive elements as FP32, for kernels over float, bfloat16 and half: V elements at a multiple of
// their size together (up to 16 bytes at a time; two floats one by one).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace amsim {

// Code of a 16-bit type (0: there is none beside float), for parameters that may be float or have the activations' type.
template <typename T> __device__ __forceinline__ constexpr int type16();
template <> __device__ __forceinline__ constexpr int type16<float>() { return 0; }
template <> __device__ __forceinline__ constexpr int type16<__nv_bfloat16>() { return 1; }
template <> __device__ __forceinline__ constexpr int type16<__half>() { return 2; }

__device__ __forceinline__ float elem_to_float(float v) { return v; }
__device__ __forceinline__ float elem_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float elem_to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T elem_from_float(float v);
template <> __device__ __forceinline__ float elem_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 elem_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half elem_from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V>
__device__ __forceinline__ void load_vec(const void* base, long long at, float (&o)[V]) {
  const T* p = static_cast<const T*>(base) + at;
  if constexpr (V == 1) {
    o[0] = elem_to_float(*p);
  } else if constexpr (sizeof(T) == 4 && V < 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = p[i];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(p + 4 * i);
      o[4 * i] = v.x; o[4 * i + 1] = v.y; o[4 * i + 2] = v.z; o[4 * i + 3] = v.w;
    }
  } else {
    static_assert(V == 2 || V == 4 || V == 8, "4, 8 or 16 bytes");
    uint32_t w[V / 2];
    if constexpr (V == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (V == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      T pair[2];
      memcpy(pair, &w[i], 4);
      o[2 * i] = elem_to_float(pair[0]);
      o[2 * i + 1] = elem_to_float(pair[1]);
    }
  }
}

// The elements of 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void unpack16(const uint32_t (&w)[4], float (&o)[V]) {
  static_assert(V * sizeof(T) == 16, "16 bytes");
  T e[V];
  memcpy(e, w, 16);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = elem_to_float(e[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(void* base, long long at, const float (&o)[V]) {
  T* p = static_cast<T*>(base) + at;
  if constexpr (V == 1) {
    *p = elem_from_float<T>(o[0]);
  } else if constexpr (sizeof(T) == 4 && V < 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = o[i];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) *reinterpret_cast<float4*>(p + 4 * i) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const T pair[2] = {elem_from_float<T>(o[2 * i]), elem_from_float<T>(o[2 * i + 1])};
      memcpy(&w[i], pair, 4);
    }
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// A parameter's elements: float, or the 16-bit type of that code.
template <int V>
__device__ __forceinline__ void load_param(const void* base, long long at, bool f32, int t16, float (&o)[V]) {
  if (f32 || t16 == 0) load_vec<float, V>(base, at, o);
  else if (t16 == 1) load_vec<__nv_bfloat16, V>(base, at, o);
  else load_vec<__half, V>(base, at, o);
}
template <int V>
__device__ __forceinline__ void store_param(void* base, long long at, bool f32, int t16, const float (&o)[V]) {
  if (f32 || t16 == 0) store_vec<float, V>(base, at, o);
  else if (t16 == 1) store_vec<__nv_bfloat16, V>(base, at, o);
  else store_vec<__half, V>(base, at, o);
}

}  // namespace amsim
