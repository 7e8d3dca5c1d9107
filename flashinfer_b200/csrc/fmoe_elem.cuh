// fmoe_elem.cuh -- loads and stores of 1 or 16-byte groups of bf16, fp16 and fp32 elements as
// fp32 values, shared by the token-sorting, quantisation and norm kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace fmoe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }

// The raw bits of V elements, as they sit in registers between load and use.
template <typename T, int V>
struct alignas(V * sizeof(T) == 16 ? 16 : alignof(T)) Pack {
  T e[V];
};

// Loads through L2 (ld.global.cg): under programmatic dependent launch the data may have been
// written by a grid that was still running when this one started, so neither the non-coherent
// path nor a line that this SM's L1 kept from before may serve it.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V * sizeof(T) == 16) {
    const uint4 w = __ldcg(reinterpret_cast<const uint4*>(p));
    memcpy(&r, &w, 16);
  } else {
    static_assert(V == 1, "16-byte groups or single elements");
    if constexpr (sizeof(T) == 4) {
      const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(p));
      memcpy(&r, &w, 4);
    } else {
      const uint16_t w = __ldcg(reinterpret_cast<const uint16_t*>(p));
      memcpy(&r, &w, 2);
    }
  }
  return r;
}

// Two neighbouring 16-bit elements as one word, first element low.
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16*, float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &p, 4);
  return w;
}
__device__ __forceinline__ uint32_t pack2(__half*, float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &p, 4);
  return w;
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16*, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(__half*, uint32_t w) {
  __half2 p;
  memcpy(&p, &w, 4);
  return __half22float2(p);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack(const float (&v)[V]) {
  Pack<T, V> r;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2(static_cast<T*>(nullptr), v[2 * i], v[2 * i + 1]);
    memcpy(&r, w, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) from_f32(v[i], &r.e[i]);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  const Pack<T, V> r = pack<T, V>(v);
  if constexpr (V * sizeof(T) == 16) {
    uint4 w;
    memcpy(&w, &r, 16);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
    *p = r.e[0];
  }
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& r, float (&v)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t w[V / 2];
    memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = unpack2(static_cast<T*>(nullptr), w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(r.e[i]);
  }
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace fmoe
