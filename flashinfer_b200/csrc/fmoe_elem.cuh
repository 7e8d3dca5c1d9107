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

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) from_f32(v[i], &r.e[i]);
  if constexpr (V * sizeof(T) == 16) {
    uint32_t w[4];
    memcpy(w, &r, 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *p = r.e[0];
  }
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& r, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(r.e[i]);
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace fmoe
