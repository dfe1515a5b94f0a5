// Rows of router logits in one warp: a lane holds V neighbouring values, in fp32 whatever their type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace b200moe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V neighbouring values at p, of which `live` exist; vec: whole and aligned.  Values that do not exist are -inf.
template <class T, int V>
__device__ __forceinline__ void load_values(const T* p, int live, bool vec, float (&z)[V]) {
  constexpr int B = V * static_cast<int>(sizeof(T));
  if (vec && live == V) {
    T raw[V];
    if constexpr (B >= 16) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    } else if constexpr (B == 4) {
      *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
    } else {
      raw[0] = p[0];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = to_f32(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = i < live ? to_f32(p[i]) : -INFINITY;
  }
}
template <class T, int V>
__device__ __forceinline__ void store_values(T* p, int live, bool vec, const float (&z)[V]) {
  constexpr int B = V * static_cast<int>(sizeof(T));
  if (vec && live == V) {
    T raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = from_f32<T>(z[i]);
    if constexpr (B >= 16) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
    } else if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
    } else if constexpr (B == 4) {
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(raw);
    } else {
      p[0] = raw[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < live) p[i] = from_f32<T>(z[i]);
  }
}

template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

template <class F>
static void by_logits(int type, F f) {
  if (type == B200MOE_LOGITS_BF16) f(__nv_bfloat16());
  else if (type == B200MOE_LOGITS_F16) f(__half());
  else f(float());
}
template <class F>
static void by_values(int v, F f) {
  if (v <= 1) f(std::integral_constant<int, 1>());
  else if (v <= 2) f(std::integral_constant<int, 2>());
  else if (v <= 4) f(std::integral_constant<int, 4>());
  else if (v <= 8) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}
static bool known_logits(int type) {
  return type == B200MOE_LOGITS_BF16 || type == B200MOE_LOGITS_F32 || type == B200MOE_LOGITS_F16;
}
static int type_bytes(int type) { return type == B200MOE_LOGITS_F32 ? 4 : 2; }

}  // namespace b200moe
