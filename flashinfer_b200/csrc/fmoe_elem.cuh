// fmoe_elem.cuh -- loads and stores of 1 or 16-byte groups of bf16, fp16 and fp32 elements as
// fp32 values, shared by the token-sorting, quantisation and norm kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fmoe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }

// The raw bits of one element, or of a 16-byte group as four words: kept as words between load and
// use, since copies of 16-bit element arrays compile to byte shuffles.
template <typename T, int V>
struct Pack {
  static_assert(V == 1, "16-byte groups or single elements");
  T e;
};
struct alignas(16) Words {
  uint32_t w[4];
};
template <>
struct Pack<float, 4> : Words {};
template <>
struct Pack<__nv_bfloat16, 8> : Words {};
template <>
struct Pack<__half, 8> : Words {};

// Two neighbouring 16-bit elements as one word, first element low.
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16*, float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(__half*, float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16*, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(__half*, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Loads through L2 (ld.global.cg): under programmatic dependent launch the data may have been
// written by a grid that was still running when this one started, so neither the non-coherent
// path nor a line that this SM's L1 kept from before may serve it.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V > 1) {
    const uint4 w = __ldcg(reinterpret_cast<const uint4*>(p));
    r.w[0] = w.x;
    r.w[1] = w.y;
    r.w[2] = w.z;
    r.w[3] = w.w;
  } else if constexpr (sizeof(T) == 4) {
    r.e = __ldcg(p);
  } else {
    const uint16_t w = __ldcg(reinterpret_cast<const uint16_t*>(p));
    r.e = *reinterpret_cast<const T*>(&w);
  }
  return r;
}

// 16 bytes of a row that is read once: not kept in L1, fetched into L2 by 256-byte lines. Adding up
// eight rows per token (4096 x 2048 bf16) took 30.6 us with ld.global.cg and takes 26.1 us with it
// (the backward pass and the quantisation, which also store as much, are no faster).
__device__ __forceinline__ uint4 load_row16(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& r, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(r.e);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(static_cast<T*>(nullptr), r.w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    from_f32(v[0], p);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(static_cast<T*>(nullptr), v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Elements of a 16-byte granule.
template <typename T>
constexpr int kV = 16 / static_cast<int>(sizeof(T));

// A granule's values in fp32, as pairs for the packed instructions.
template <typename T>
struct Gran {
  static constexpr int N = kV<T> / 2;
  float2 p[N];
};

template <typename T>
__device__ __forceinline__ void zero(Gran<T>& v) {
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) v.p[i] = make_float2(0.0f, 0.0f);
}
// a * b, a * s, a * b + c, a * s + c, element by element
template <typename T>
__device__ __forceinline__ Gran<T> mul(const Gran<T>& a, const Gran<T>& b) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) r.p[i] = __fmul2_rn(a.p[i], b.p[i]);
  return r;
}
template <typename T>
__device__ __forceinline__ Gran<T> mul(const Gran<T>& a, float s) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) r.p[i] = __fmul2_rn(a.p[i], make_float2(s, s));
  return r;
}
template <typename T>
__device__ __forceinline__ Gran<T> fma(const Gran<T>& a, const Gran<T>& b, const Gran<T>& c) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) r.p[i] = __ffma2_rn(a.p[i], b.p[i], c.p[i]);
  return r;
}
template <typename T>
__device__ __forceinline__ Gran<T> fma(const Gran<T>& a, float s, const Gran<T>& c) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i)
    r.p[i] = __ffma2_rn(a.p[i], make_float2(s, s), c.p[i]);
  return r;
}
// acc += a * b, in two interleaved sums
template <typename T>
__device__ __forceinline__ void dot(float2& acc, const Gran<T>& a, const Gran<T>& b) {
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) acc = __ffma2_rn(a.p[i], b.p[i], acc);
}

template <typename T>
__device__ __forceinline__ Gran<T> gran_of(const uint4& q) {
  Gran<T> r;
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) {
    if constexpr (sizeof(T) == 4)
      r.p[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      r.p[i] = unpack2(static_cast<T*>(nullptr), w[i]);
  }
  return r;
}

// The granule rounded to T.
template <typename T>
__device__ __forceinline__ uint4 words_of(const Gran<T>& g) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(g.p[0].x), __float_as_uint(g.p[0].y),
                      __float_as_uint(g.p[1].x), __float_as_uint(g.p[1].y));
  } else {
    T* type = nullptr;
    return make_uint4(pack2(type, g.p[0].x, g.p[0].y), pack2(type, g.p[1].x, g.p[1].y),
                      pack2(type, g.p[2].x, g.p[2].y), pack2(type, g.p[3].x, g.p[3].y));
  }
}

// Stores the bytes [lo, hi) of q to the granule at p (element size E).
template <int E>
__device__ __forceinline__ void store_part(uint8_t* p, const uint4& q, int lo, int hi) {
  if (lo <= 0 && hi >= 16) {
    *reinterpret_cast<uint4*>(p) = q;
    return;
  }
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 16; i += E) {
    if (i < lo || i >= hi) continue;
    if constexpr (E == 4)
      *reinterpret_cast<uint32_t*>(p + i) = w[i / 4];
    else if constexpr (E == 2)
      *reinterpret_cast<uint16_t*>(p + i) = static_cast<uint16_t>(w[i / 4] >> (8 * (i % 4)));
    else
      p[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace fmoe
