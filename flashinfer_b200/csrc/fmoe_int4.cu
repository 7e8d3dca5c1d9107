// fmoe_int4.cu -- products of 16-bit activations with 4-bit weights, for one matrix or one per expert,
// few tokens; the quantisation of weights to that format and back.
//
//   w[n, k] = scale[n, g] * (q[n, k] - zero[n, g]),  g = k / group,  q, zero in 0 .. 15
//   y[t, n] = sum_k x[t, k] w[n, k] (+ bias[n])
//
// q - zero is exact in the activations' 16 bits; a group's sum of x * (q - zero) runs in fp32, is multiplied
// with its scale in fp32 and added up in fp32: no weight is rounded, and the result once.
#include <type_traits>

#include "fmoe_int4.cuh"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

// ------------------------------------------------------------------ few tokens
// A stream of the weights, 16 rows (times RT) per block: the block's eight warps take 128-value pieces of
// K in turn, so that a step of the block reads 512 consecutive bytes of each row. Lane (g, t), g = lane / 4,
// t = lane % 4, loads the 16 bytes of values 32 t .. 32 t + 31 of rows g and g + 8, D pieces ahead, and
// turns them into the fragments of mma.m16n8k16 in its own registers: which values of k a lane has is free
// as long as the tokens' fragment has the same ones. No shared memory before the end, when the warps' sums
// are added in order.
//
// The weights are the 16 rows of the MMA and the tokens its 8 columns (times NT). The tensor cores' larger
// instruction would need the widened weights in shared memory first; for a handful of tokens the loads and
// the widening (11 instructions for 8 values) are all there is, and the MMAs are idle most of the time.
//
// SPREAD (group 32 or 64): an MMA sums over all four lanes of a quad, which must then be in one group: the
// quad's 4 x 4 words are transposed by shuffles, after which step c of lane t has values 32 c + 8 t ...
constexpr int kFewWarps = 8;

__device__ __forceinline__ void mma_16816(__nv_bfloat16*, float (&c)[4], const uint32_t (&a)[4],
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(__half*, float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Word j of lane t of a quad goes to word t of lane j.
__device__ __forceinline__ void transpose_quad(uint4& q) {
  const int t = threadIdx.x & 3;
  uint32_t a = t & 1 ? q.x : q.y, b = t & 1 ? q.z : q.w;
  a = __shfl_xor_sync(0xffffffffu, a, 1);
  b = __shfl_xor_sync(0xffffffffu, b, 1);
  if (t & 1) {
    q.x = a;
    q.z = b;
  } else {
    q.y = a;
    q.w = b;
  }
  a = t & 2 ? q.x : q.z;
  b = t & 2 ? q.y : q.w;
  a = __shfl_xor_sync(0xffffffffu, a, 2);
  b = __shfl_xor_sync(0xffffffffu, b, 2);
  if (t & 2) {
    q.x = a;
    q.y = b;
  } else {
    q.z = a;
    q.w = b;
  }
}

// Eight values less the zero point (zp: the base plus it, twice) as pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <typename T>
__device__ __forceinline__ void widen8(uint32_t q, uint32_t zp, uint32_t (&v)[4]) {
  T* type = nullptr;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = sub2(type, and_or(q >> (4 * i), 0x000f000fu, nibble_base(type)), zp);
}

template <typename T, int RT, int NT, int D, bool SPREAD>
__global__ void __launch_bounds__(kFewWarps * 32, 2) k_int4_few(const I4Args a, const uint32_t group_magic) {
  constexpr int ROWS = 16 * RT, COLS = 8 * NT;
  __shared__ float red[kFewWarps][COLS][ROWS + 1];
  T* type = nullptr;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int e = blockIdx.y;
  const int n0 = blockIdx.x * ROWS;
  pdl_begin_in_order();
  zero_foreign_rows(a, static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x,
                    static_cast<int64_t>(gridDim.x) * gridDim.y);
  int64_t r0, r1;
  expert_rows(a.expert_base, e, a.M, &r0, &r1);
  if (r0 >= r1) return;

  const int blocks = (a.K + 127) / 128;
  const int ssize = a.scale_f32 ? 4 : 2;
  // of the block's first row, and how far this lane's rows are from it (rows behind the last are the last,
  // and are not stored)
  const int64_t row0 = static_cast<int64_t>(e) * a.N + n0;
  const uint8_t* wp = a.w + row0 * (a.K / 2);
  const uint8_t* sp = static_cast<const uint8_t*>(a.scale) + row0 * a.groups * ssize;
  const uint8_t* zp = a.zero ? a.zero + row0 * a.groups : nullptr;
  int away[2 * RT];
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) away[i] = min(8 * i + g, a.N - 1 - n0);
  const auto scale = [&](int i, int grp) {  // as its bits
    const int at = away[i] * a.groups + grp;
    return a.scale_f32 ? reinterpret_cast<const uint32_t*>(sp)[at]
                       : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(sp)[at]);
  };
  const auto zero = [&](int i, int grp) -> uint32_t { return zp ? zp[away[i] * a.groups + grp] : 8u; };
  const auto number = [&](uint32_t bits) {
    if (a.scale_f32) return __uint_as_float(bits);
    if constexpr (std::is_same<T, __half>::value)
      return __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
    else
      return __uint_as_float(bits << 16);
  };

  for (int64_t m0 = r0; m0 < r1; m0 += COLS) {
    // the tokens of this lane's column, from its first value in a block on (SPREAD: in a step)
    const T* xp[NT];
    bool has[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t row = m0 + 8 * j + g;
      has[j] = row < r1;
      xp[j] = static_cast<const T*>(a.x) + (has[j] ? row : r0) * a.K + (SPREAD ? 8 : 32) * t;
    }
    struct Ahead {
      uint4 w[2 * RT];
      uint32_t s[SPREAD ? 1 : 2 * RT], z[SPREAD ? 1 : 2 * RT];
    };
    Ahead q[D];
    const auto fetch = [&](int b, Ahead& to) {
      if (b >= blocks) return;
      // K is a multiple of 32: a lane's 16 bytes are in the row, or the tokens there are zeros
      if (b * 128 + 32 * t < a.K) {
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i)
          to.w[i] = load_row16(
              reinterpret_cast<const uint4*>(wp + (away[i] * (a.K / 2) + b * 64 + 16 * t)));
      }
      if constexpr (!SPREAD) {
        const int grp = static_cast<int>((static_cast<uint32_t>(b) * group_magic) >> 20);
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) {
          to.s[i] = scale(i, grp);
          to.z[i] = zero(i, grp);
        }
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) {
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) q[d].w[i] = make_uint4(0u, 0u, 0u, 0u);
      fetch(warp + d * kFewWarps, q[d]);
    }
    float acc[RT][NT][4] = {};
    for (int b0 = warp; b0 < blocks; b0 += D * kFewWarps) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int b = b0 + d * kFewWarps;
        if (b >= blocks) break;
        uint4 v[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = b * 128 + (SPREAD ? 32 * c : 32 * t);
            v[j][c] = make_uint4(0u, 0u, 0u, 0u);
            if (has[j] && k < a.K)
              v[j][c] = *reinterpret_cast<const uint4*>(xp[j] + b * 128 + (SPREAD ? 32 : 8) * c);
          }
        if constexpr (SPREAD) {
#pragma unroll
          for (int i = 0; i < 2 * RT; ++i) transpose_quad(q[d].w[i]);
        }
        float part[RT][NT][4] = {};  // of the group at hand
        float sc[2 * RT];
        uint32_t zb[2 * RT];
        const auto open = [&](int grp) {
#pragma unroll
          for (int i = 0; i < 2 * RT; ++i) {
            // a step behind the row's end adds nothing, whatever the last scale
            const bool in = !SPREAD || grp < a.groups;
            sc[i] = in ? number(SPREAD ? scale(i, grp) : q[d].s[SPREAD ? 0 : i]) : 0.0f;
            const uint32_t z = in ? SPREAD ? zero(i, grp) : q[d].z[SPREAD ? 0 : i] : 8u;
            zb[i] = nibble_base(type) + (z & 15u) * 0x00010001u;  // the base has the low four bits free
          }
        };
        const auto close = [&]() {
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                acc[r][j][i] = fmaf(sc[2 * r + (i >> 1)], part[r][j][i], acc[r][j][i]);
                part[r][j][i] = 0.0f;
              }
        };
        if constexpr (!SPREAD) open(0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if constexpr (SPREAD) {  // a step is 32 values of one group
            if (a.group == 32)
              open(4 * b + c);
            else if ((c & 1) == 0)
              open(2 * b + c / 2);
          }
          uint32_t bf[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            bf[j][0] = __byte_perm(v[j][c].x, v[j][c].z, 0x5410);
            bf[j][1] = __byte_perm(v[j][c].x, v[j][c].z, 0x7632);
            bf[j][2] = __byte_perm(v[j][c].y, v[j][c].w, 0x5410);
            bf[j][3] = __byte_perm(v[j][c].y, v[j][c].w, 0x7632);
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint4 &wl = q[d].w[2 * r], &wh = q[d].w[2 * r + 1];
            uint32_t lo[4], hi[4];
            widen8<T>(c == 0 ? wl.x : c == 1 ? wl.y : c == 2 ? wl.z : wl.w, zb[2 * r], lo);
            widen8<T>(c == 0 ? wh.x : c == 1 ? wh.y : c == 2 ? wh.z : wh.w, zb[2 * r + 1], hi);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma_16816(type, part[r][j], {lo[0], hi[0], lo[1], hi[1]}, bf[j][0], bf[j][1]);
              mma_16816(type, part[r][j], {lo[2], hi[2], lo[3], hi[3]}, bf[j][2], bf[j][3]);
            }
          }
          if (SPREAD ? a.group == 32 || (c & 1) == 1 : c == 3) close();
        }
        fetch(b + D * kFewWarps, q[d]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[warp][8 * j + 2 * t + (i & 1)][16 * r + 8 * (i >> 1) + g] = acc[r][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * COLS; i += kFewWarps * 32) {
      const int c = i / ROWS, r = i - c * ROWS;
      if (m0 + c < r1 && n0 + r < a.N) {
        float sum = a.bias ? a.bias[n0 + r] : 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) sum += red[w][c][r];
        from_f32(sum, static_cast<T*>(a.out) + (m0 + c) * a.N + n0 + r);
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ quantisation
// Eight consecutive values of a row per lane. A group of up to 256 values is in the registers of up to 32
// neighbouring lanes between its maximum and the rounding; a longer one (WIDE) is a warp's and read twice.
//   symmetric: scale = max|w| / 7,             q = round(w / scale) + 8 in 1 .. 15
//   else:      scale = (high - low) / 15,      zero = round(-low / scale), q = round(w / scale) + zero,
//              low = min(w, 0), high = max(w, 0)
// rounded to the weights' type before the division by it, and no smaller than the type's least scale.
// Rounding is to the nearest integer, ties to even; the divisions are IEEE's.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += kV<T>) {
    float w[kV<T>];
    unpack(load_pack<T, kV<T>>(p + i), w);
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) v[i + j] = w[j];
  }
}

struct GroupRange {
  uint32_t amax;  // bits of the largest absolute value: NaN above infinity above all
  float low, high;
};

__device__ __forceinline__ void widen(GroupRange& r, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r.amax = max(r.amax, __float_as_uint(v[i]) & 0x7fffffffu);
    r.low = fminf(r.low, v[i]);
    r.high = fmaxf(r.high, v[i]);
  }
}

template <typename T>
__device__ __forceinline__ float group_scale(const GroupRange& r, bool symmetric) {
  const float amax = __uint_as_float(r.amax);
  float step = symmetric ? __fdiv_rn(amax, 7.0f) : __fdiv_rn(__fsub_rn(r.high, r.low), 15.0f);
  const float least = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-100f;
  step = fmaxf(step, least);
  if (r.amax >= 0x7f800000u) step = __fadd_rn(amax, amax);  // infinite or NaN
  T s;
  from_f32(step, &s);
  return to_f32(s);
}

template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], float scale, float zero, float least) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf(rintf(__fdiv_rn(v[i], scale)) + zero, least), 15.0f);
    w |= static_cast<uint32_t>(q) << (4 * i);
  }
  return w;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(256)
    k_quantize_int4(const T* w, int64_t rows, int K, int group, int groups, int symmetric,
                    uint8_t* packed, T* scale, uint8_t* zero) {
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  // pieces of a row: 256 values, or a group
  const int pieces = WIDE ? groups : (K + 255) / 256;
  const int64_t row = warp / pieces;
  if (row >= rows) return;
  const int piece = static_cast<int>(warp - row * pieces);
  const int k0 = piece * (WIDE ? group : 256);
  const int k1 = min(K, k0 + (WIDE ? group : 256));
  const T* wr = w + row * K;
  uint8_t* out = packed + row * (K / 2);
  GroupRange r{0u, 0.0f, 0.0f};
  float v[8];
  if (WIDE) {
    for (int k = k0 + 8 * lane; k < k1; k += 256) {
      load8(wr + k, v);
      widen(r, v);
    }
  } else if (k0 + 8 * lane < k1) {
    load8(wr + k0 + 8 * lane, v);
    widen(r, v);
  }
  // a group's lanes: group / 8 of them, a power of two and aligned (WIDE: all)
  const int width = WIDE || group > 256 ? 32 : group / 8;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t m = __shfl_xor_sync(0xffffffffu, r.amax, o);
    const float l = __shfl_xor_sync(0xffffffffu, r.low, o), h = __shfl_xor_sync(0xffffffffu, r.high, o);
    if (o < width) {
      r.amax = max(r.amax, m);
      r.low = fminf(r.low, l);
      r.high = fmaxf(r.high, h);
    }
  }
  const float s = group_scale<T>(r, symmetric);
  const float z = symmetric ? 8.0f : fminf(fmaxf(rintf(__fdiv_rn(-r.low, s)), 0.0f), 15.0f);
  const float least = symmetric ? 1.0f : 0.0f;
  const int k = k0 + 8 * lane;
  if (k < k1 && (WIDE ? lane == 0 : k % group == 0)) {
    const int64_t at = row * groups + k / group;
    from_f32(s, scale + at);
    if (zero) zero[at] = static_cast<uint8_t>(z);
  }
  if (WIDE) {
    for (int j = k; j < k1; j += 256) {
      load8(wr + j, v);
      *reinterpret_cast<uint32_t*>(out + j / 2) = quantise8<T>(v, s, z, least);
    }
  } else if (k < k1) {
    *reinterpret_cast<uint32_t*>(out + k / 2) = quantise8<T>(v, s, z, least);
  }
}

// 32 values per thread, all of one group: 16 bytes in, scale * (q - zero) in fp32, rounded once.
template <typename T, typename S>
__global__ void __launch_bounds__(256)
    k_dequantize_int4(const uint8_t* packed, const S* scale, const uint8_t* zero, int64_t rows, int K,
                      int group, int groups, T* out) {
  pdl_begin_in_order();
  const int per = K / 32;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = i / per;
  if (row >= rows) return;
  const int k = static_cast<int>(i - row * per) * 32;
  const uint4 q = load_row16(reinterpret_cast<const uint4*>(packed + row * (K / 2) + k / 2));
  const int64_t at = row * groups + k / group;
  const float s = to_f32(scale[at]);
  const float z = zero ? static_cast<float>(zero[at] & 15u) : 8.0f;
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  T* o = out + row * K + k;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int h = 0; h < 8; h += kV<T>) {
      float v[kV<T>];
#pragma unroll
      for (int l = 0; l < kV<T>; ++l)
        v[l] = (static_cast<float>((w[j] >> (4 * (h + l))) & 15u) - z) * s;
      store_pack(o + 8 * j + h, v);
    }
  }
}

// ------------------------------------------------------------------ launches
template <typename T>
cudaError_t quantise(const Int4Weights& p, cudaStream_t s) {
  const bool wide = p.group > 256;
  const int64_t pieces = p.rows * (wide ? p.groups : (p.K + 255) / 256);
  const dim3 grid(static_cast<unsigned>((pieces + 7) / 8));
  const T* w = static_cast<const T*>(p.w);
  T* scale = static_cast<T*>(p.scale);
  if (wide)
    return launch_pdl(k_quantize_int4<T, true>, grid, dim3(256), 0, s, w, p.rows, p.K, p.group, p.groups,
                      p.symmetric, p.packed, scale, p.zero);
  return launch_pdl(k_quantize_int4<T, false>, grid, dim3(256), 0, s, w, p.rows, p.K, p.group, p.groups,
                    p.symmetric, p.packed, scale, p.zero);
}

template <typename T, typename S>
cudaError_t dequantise(const Int4Weights& p, cudaStream_t s) {
  const int64_t threads = p.rows * (p.K / 32);
  return launch_pdl(k_dequantize_int4<T, S>, dim3(static_cast<unsigned>((threads + 255) / 256)),
                    dim3(256), 0, s, p.packed, static_cast<const S*>(p.scale), p.zero, p.rows, p.K,
                    p.group, p.groups, static_cast<T*>(p.w));
}

template <typename T>
cudaError_t dequantise(const Int4Weights& p, cudaStream_t s) {
  switch (p.scale_dtype) {
    case FMOE_DTYPE_F32:
      return dequantise<T, float>(p, s);
    case FMOE_DTYPE_BF16:
      return dequantise<T, __nv_bfloat16>(p, s);
    default:
      return dequantise<T, __half>(p, s);
  }
}

template <typename T, int RT, int NT, int D>
cudaError_t few(const I4Args& a, cudaStream_t s) {
  const dim3 grid((a.N + 16 * RT - 1) / (16 * RT), a.E);
  // a block of 128 values b, at most 1023, is in group (b * magic) >> 20 = b / (group / 128): the error of the
  // product is below 2^-10
  const int per = a.group / 128;
  const uint32_t magic = per == 0 || per > 1024 ? 0u : (1u << 20) / per + 1;
  if (a.group < 128)
    return launch_pdl(k_int4_few<T, RT, NT, D, true>, grid, dim3(kFewWarps * 32), 0, s, a, magic);
  return launch_pdl(k_int4_few<T, RT, NT, D, false>, grid, dim3(kFewWarps * 32), 0, s, a, magic);
}

template <typename T>
cudaError_t few(const I4Args& a, int64_t per, int sms, cudaStream_t s) {
  // 32 rows per block share the tokens' loads, as long as there are blocks enough
  const int64_t used = a.M < a.E ? a.M : a.E;
  const bool tall = (a.N + 31) / 32 * used >= 4 * sms;
  if (per <= 8) return tall ? few<T, 2, 1, 2>(a, s) : few<T, 1, 1, 4>(a, s);
  return few<T, 1, 2, 2>(a, s);
}

}  // namespace

cudaError_t launch_quantize_int4(const Int4Weights& p, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return quantise<float>(p, s);
    case FMOE_DTYPE_BF16:
      return quantise<__nv_bfloat16>(p, s);
    default:
      return quantise<__half>(p, s);
  }
}

cudaError_t launch_dequantize_int4(const Int4Weights& p, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return dequantise<float>(p, s);
    case FMOE_DTYPE_BF16:
      return dequantise<__nv_bfloat16>(p, s);
    default:
      return dequantise<__half>(p, s);
  }
}

// An expert is taken to have up to twice its even share of the rows, which the device alone knows.
Int4Plan int4_plan(int64_t M, int N, int K, int E, bool grouped) {
  const int64_t used = M < E ? M : E;
  int64_t per = used > 0 ? (M + used - 1) / used : 0;
  if (per <= (grouped ? 8 : 16)) return Int4Plan{0, 1};
  if (grouped) per = 2 * per < M ? 2 * per : M;
  Int4Plan p{per <= 64 ? 64 : per <= 128 ? 128 : 256, 1};
  // a tile of 256 tokens has 256 weight rows and takes two SMs
  const int rows = p.bn == 256 ? 256 : 128, slots = p.bn == 256 ? 74 : 148;
  const int64_t tiles = (per + p.bn - 1) / p.bn * used * ((N + rows - 1) / rows);
  // K in parts while there are fewer tiles than run at a time (148 SMs), each of four blocks of 64 or more
  const int64_t most = (K + 63) / 64 / 4;
  while (p.S < 8 && (p.S + 1) * tiles <= slots && p.S < most) ++p.S;
  return p;
}

cudaError_t launch_int4_product(const Int4Product& p, int sms, cudaStream_t s) {
  I4Args a{};
  a.x = p.x;
  a.w = p.w;
  a.scale = p.scale;
  a.zero = p.zero;
  a.bias = p.bias;
  a.expert_base = p.expert_base;
  a.out = p.out;
  a.M = p.M;
  a.N = p.N;
  a.K = p.K;
  a.E = p.E;
  a.group = p.group;
  a.groups = (p.K + p.group - 1) / p.group;
  a.scale_f32 = p.scale_dtype == FMOE_DTYPE_F32;
  a.zero_tail = p.zero_tail;
  a.part = p.part;
  Int4Plan plan = int4_plan(p.M, p.N, p.K, p.E, p.expert_base != nullptr);
  if (p.tile_tokens != 0) plan = Int4Plan{p.tile_tokens, p.split};
  if (p.wait_ns != 0 && plan.bn == 0) plan.bn = 64;  // the kernel for few has no waits
  if (plan.bn != 0) return launch_int4_mm(p, a, plan, sms, s);
  const int64_t used = p.M < p.E ? p.M : p.E;
  const int64_t per = (p.M + used - 1) / used;
  return p.dtype == FMOE_DTYPE_BF16 ? few<__nv_bfloat16>(a, per, sms, s) : few<__half>(a, per, sms, s);
}

}  // namespace fmoe
