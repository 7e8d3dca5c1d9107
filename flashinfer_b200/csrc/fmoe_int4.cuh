// fmoe_int4.cuh -- what the kernels of 4-bit weights share: the value format, expert bases and the
// rows of no expert.
#pragma once

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"

namespace fmoe {

struct I4Args {
  const void* x;              // [M, K]
  const uint8_t* w;           // [E, N, K / 2], value 2i in the low half of byte i
  const void* scale;          // [E, N, groups], of x's type or fp32
  const uint8_t* zero;        // [E, N, groups] (the low four bits count), or null: 8
  const float* bias;          // [N] or null
  const int32_t* expert_base; // [E + 1] or null: one matrix
  void* out;                  // [M, N], of x's type
  float* part;                // split products: [S][M][N] partial sums
  int64_t M;
  int N, K, E;
  int group, groups;
  int scale_f32;
  int zero_tail;
};

// fmoe_int4_mm.cu: the product on the tensor cores (plan.bn > 0).
cudaError_t launch_int4_mm(const Int4Product& p, const I4Args& a, const Int4Plan& plan, int sms,
                           cudaStream_t s);

// Rows of expert e of a product of M rows: bases clamped to [0, M], one that is smaller than an earlier
// one counting as that one. By a whole warp. Without bases all rows are expert 0's.
__device__ __forceinline__ void expert_rows(const int32_t* base, int e, int64_t M, int64_t* r0,
                                            int64_t* r1) {
  if (!base) {
    *r0 = 0;
    *r1 = M;
    return;
  }
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = 0;
  for (int i = lane; i <= e + 1; i += 32) {
    int b = __ldcg(base + i);
    b = b < 0 ? 0 : b > M ? static_cast<int>(M) : b;
    if (i <= e) lo = max(lo, b);
    hi = max(hi, b);
  }
  *r0 = __reduce_max_sync(0xffffffffu, lo);
  *r1 = __reduce_max_sync(0xffffffffu, hi);
}

// Zeroes rows [from, to) of an output of 16-bit elements, by thread `tid` of `threads`.
__device__ __forceinline__ void zero_rows16(void* out, int N, int64_t from, int64_t to, int64_t tid,
                                            int64_t threads) {
  const int64_t bytes = (to - from) * N * 2;
  if (bytes <= 0) return;
  uint8_t* p = static_cast<uint8_t*>(out) + from * N * 2;
  int64_t head = (16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15u)) & 15;
  if (head > bytes) head = bytes;
  const int64_t wide = (bytes - head) / 16;
  for (int64_t i = tid; i < wide; i += threads)
    reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0u, 0u, 0u, 0u);
  const int64_t rest = bytes - head - wide * 16;  // like head an even number below 16
  if (tid < head / 2) reinterpret_cast<uint16_t*>(p)[tid] = 0;
  if (tid < rest / 2) reinterpret_cast<uint16_t*>(p + head + wide * 16)[tid] = 0;
}

// The rows that no expert has, zeroed by the whole grid (block `block` of `blocks`, every warp).
__device__ __forceinline__ void zero_foreign_rows(const I4Args& a, int64_t block, int64_t blocks) {
  if (!a.zero_tail || !a.expert_base) return;
  int64_t first, none, end;
  expert_rows(a.expert_base, 0, a.M, &first, &none);
  expert_rows(a.expert_base, a.E - 1, a.M, &none, &end);
  const int64_t tid = block * blockDim.x + threadIdx.x, threads = blocks * blockDim.x;
  zero_rows16(a.out, a.N, 0, first, tid, threads);
  zero_rows16(a.out, a.N, end, a.M, tid, threads);
}

// 4-bit values as 16-bit floats. The bits of 128 (bf16) or 1024 (fp16) with a value in the low mantissa
// bits are that number plus the value; taking away the same number plus the zero point is exact.
__device__ __forceinline__ uint32_t nibble_base(__nv_bfloat16*) { return 0x43004300u; }
__device__ __forceinline__ uint32_t nibble_base(__half*) { return 0x64006400u; }
__device__ __forceinline__ uint32_t sub2(__nv_bfloat16*, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t sub2(__half*, uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}


// (a & mask) | base in one instruction. Written with operators, and both constants known, it takes two: an
// instruction has room for one constant (104 instead of 72 bit operations for 64 values).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(base));
  return r;
}

__device__ __forceinline__ uint32_t mul2(__nv_bfloat16*, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                      *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t mul2(__half*, uint32_t a, uint32_t b) {
  const __half2 r = __hmul2_rn(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t fma2(__nv_bfloat16*, uint32_t a, uint32_t b, uint32_t c) {
  const __nv_bfloat162 r =
      __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b),
              *reinterpret_cast<const __nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t fma2(__half*, uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight values of one group as 16-bit weights, in order. hi, lo: the scale (twice) and, with F32S, what its
// rounding left.
template <typename T, bool F32S>
__device__ __forceinline__ uint4 weights8(uint32_t q, uint32_t zp, uint32_t hi, uint32_t lo) {
  T* type = nullptr;
  // byte i holds values 2i and 2i + 1: from q its low half to a word's low 16 bits, from q >> 4 its high
  // half to the high 16 bits
  const uint32_t q4 = q >> 4, base = nibble_base(type);
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = sub2(type, and_or(__byte_perm(q, q4, i | (i + 4) << 8), 0x000f000fu, base), zp);
    if constexpr (F32S)
      v[i] = fma2(type, hi, v[i], mul2(type, lo, v[i]));
    else
      v[i] = mul2(type, hi, v[i]);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

}  // namespace fmoe
