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
// A stream of the weights, 16 rows (times RT) per block: the block's W warps take 128-value pieces of K in
// turn, so that a step of the block reads 64 W consecutive bytes of each row. Lane (g, t), g = lane / 4,
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

template <typename T, int RT, int NT, int D, int W, bool SPREAD>
__global__ void __launch_bounds__(W * 32, 16 / W) k_int4_few(const I4Args a, const uint32_t group_magic) {
  constexpr int ROWS = 16 * RT, COLS = 8 * NT;
  __shared__ float red[W][COLS][ROWS + 1];
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
      fetch(warp + d * W, q[d]);
    }
    float acc[RT][NT][4] = {};
    for (int b0 = warp; b0 < blocks; b0 += D * W) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int b = b0 + d * W;
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
        fetch(b + D * W, q[d]);
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
    for (int i = threadIdx.x; i < ROWS * COLS; i += W * 32) {
      const int c = i / ROWS, r = i - c * ROWS;
      if (m0 + c < r1 && n0 + r < a.N) {
        float sum = a.bias ? a.bias[n0 + r] : 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += red[w][c][r];
        from_f32(sum, static_cast<T*>(a.out) + (m0 + c) * a.N + n0 + r);
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ quantisation
// Eight consecutive values of a row per lane. A group of up to 256 values is in the registers of up to 32
// neighbouring lanes between its maximum and the rounding.
//   symmetric: scale = max|w| / 7,             q = round(w / scale) + 8 in 1 .. 15
//   else:      scale = (high - low) / 15,      zero = round(-low / scale), q = round(w / scale) + zero,
//              low = min(w, 0), high = max(w, 0)
// rounded to the weights' type before the division by it, and no smaller than the type's least scale.
// Rounding is of the IEEE quotients to the nearest integer, ties to even.
struct GroupRange {
  uint32_t amax;  // bits of the largest absolute value: NaN above infinity above all
  float low, high;
};

__device__ __forceinline__ void widen(GroupRange& r, const float (&v)[8], int symmetric) {
#pragma unroll
  for (int i = 0; i < 8; ++i) r.amax = max(r.amax, __float_as_uint(v[i]) & 0x7fffffffu);
  if (symmetric) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r.low = fminf(r.low, v[i]);
    r.high = fmaxf(r.high, v[i]);
  }
}

// The two values of a word, 16-bit floats, by their larger and smaller; a NaN stays in the larger.
__device__ __forceinline__ uint32_t max2(__nv_bfloat16*, uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(__half*, uint32_t a, uint32_t b) {
  const __half2 m =
      __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t min2(__nv_bfloat16*, uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t min2(__half*, uint32_t a, uint32_t b) {
  const __half2 m = __hmin2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

template <typename T>
__device__ __forceinline__ float group_scale(const GroupRange& r, bool symmetric) {
  const float amax = __uint_as_float(r.amax);
  float step = symmetric ? __fdiv_rn(amax, 7.0f) : __fdiv_rn(__fsub_rn(r.high, r.low), 15.0f);
  // finite values further apart than fp32 reaches: from their halves
  if (!std::is_same<T, __half>::value && step == INFINITY)
    step = __fdiv_rn(__fsub_rn(0.5f * r.high, 0.5f * r.low), 7.5f);
  const float least = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-100f;
  step = fmaxf(step, least);
  if (r.amax >= 0x7f800000u) step = __fadd_rn(amax, amax);  // infinite or NaN
  T s;
  from_f32(step, &s);
  return to_f32(s);
}

// Eight values as q. 16-bit weights are not divided: v = w * inv is within two units of the quotient and
// w - v * scale is exact, so the corrected v is the quotient where that is halfway between integers, and any
// other quotient of 11-bit numbers is 2^-20 (relative) or more away from halfway. Adding 1.5 * 2^23 rounds to
// the even integer, which is then the low byte of the sum. The zero point is added to four such bytes at a
// time; of the results, 0 .. 16 (see zero and low, which are rounded alike), only 16 has to be brought back. Not so
// where the scale itself was rounded among fp16's subnormal numbers: those are done value by value, like
// fp32 weights.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], float scale, float inv, int zero, int least) {
  uint32_t w = 0;
  if (sizeof(T) == 4 || (std::is_same<T, __half>::value && scale < 0x1p-14f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = rintf(__fdiv_rn(v[i], scale));
      w |= static_cast<uint32_t>(max(least, min(15, static_cast<int>(r) + zero))) << (4 * i);
    }
    return w;
  }
  const float2 s2 = make_float2(-scale, -scale), i2 = make_float2(inv, inv);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 p = make_float2(v[i], v[i + 1]);
    float2 r = __fmul2_rn(p, i2);
    r = __ffma2_rn(__ffma2_rn(r, s2, p), i2, r);
    r = __fadd2_rn(r, make_float2(12582912.0f, 12582912.0f));
    b[i] = __float_as_uint(r.x);
    b[i + 1] = __float_as_uint(r.y);
  }
  const uint32_t z4 = static_cast<uint32_t>(zero) * 0x01010101u;
  uint32_t h[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __byte_perm(b[4 * i], b[4 * i + 1], 0x0040);
    const uint32_t x = __byte_perm(lo, __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    uint32_t q = ((x & 0x7f7f7f7fu) + z4) ^ (x & 0x80808080u);  // no byte carries into the next
    q = (q - ((q >> 4) & 0x01010101u)) & 0x0f0f0f0fu;
    h[i] = q | q >> 4;  // bytes 0 and 2 have two values each
  }
  return __byte_perm(h[0], h[1], 0x6420);
}

// Eight values as they are in memory.
template <typename T>
struct Raw8 {
  Pack<T, kV<T>> p[8 / kV<T>];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 8 / kV<T>; ++i) r.p[i] = load_pack<T, kV<T>>(p + i * kV<T>);
  return r;
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8 / kV<T>; ++i) {
    float w[kV<T>];
    unpack(r.p[i], w);
#pragma unroll
    for (int j = 0; j < kV<T>; ++j) v[i * kV<T> + j] = w[j];
  }
}

template <typename T>
__device__ __forceinline__ GroupRange range8(const Raw8<T>& raw, int symmetric) {
  GroupRange r{0u, 0.0f, 0.0f};
  if constexpr (sizeof(T) == 4) {
    float v[8];
    values8(raw, v);
    widen(r, v, symmetric);
  } else {
    T* type = nullptr;
    const uint32_t* w = raw.p[0].w;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max2(type, m, w[i] & 0x7fff7fffu);
    float2 f = unpack2(type, m);
    r.amax = max(__float_as_uint(f.x), __float_as_uint(f.y)) & 0x7fffffffu;
    if (!symmetric) {
      uint32_t lo = w[0], hi = w[0];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        lo = min2(type, lo, w[i]);
        hi = max2(type, hi, w[i]);
      }
      f = unpack2(type, lo);
      r.low = fminf(0.0f, fminf(f.x, f.y));
      f = unpack2(type, hi);
      r.high = fmaxf(0.0f, fmaxf(f.x, f.y));
    }
  }
  return r;
}

// Joins the ranges of `width` neighbouring lanes (a power of two, the same in every thread).
__device__ __forceinline__ void join_lanes(GroupRange& r, int width, int symmetric) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o >= width) continue;
    r.amax = max(r.amax, __shfl_xor_sync(0xffffffffu, r.amax, o));
    if (!symmetric) {
      r.low = fminf(r.low, __shfl_xor_sync(0xffffffffu, r.low, o));
      r.high = fmaxf(r.high, __shfl_xor_sync(0xffffffffu, r.high, o));
    }
  }
}

template <typename T>
struct GroupCode {
  float s, inv;
  int z, least;
  __device__ __forceinline__ GroupCode(const GroupRange& r, int symmetric) {
    s = group_scale<T>(r, symmetric);
    inv = 1.0f / s;
    z = symmetric ? 8 : static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(-r.low, s)), 0.0f), 15.0f));
    least = symmetric ? 1 : 0;
  }
};

// Groups of up to 256 values: a warp takes 256 values at a time, two such pieces side by side and the next two
// on their way; blockIdx.y and gridDim.y share out a row's pieces. A warp per piece, its row found by a 64-bit
// division and each value divided, took 51 us for 4096 x 7168.
template <typename T>
__global__ void __launch_bounds__(256)
    k_quantize_int4(const T* w, int64_t rows, int K, int group, int groups, int symmetric,
                    uint8_t* packed, T* scale, uint8_t* zero) {
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* wr = w + row * K + 8 * lane;
  uint32_t* out = reinterpret_cast<uint32_t*>(packed + row * (K / 2)) + lane;
  const int width = group / 8;              // lanes of a group
  const int per = 256 / group;              // groups of a piece
  const int mine = lane / width;
  const bool first = (lane & (width - 1)) == 0;
  const int step = gridDim.y;
  const auto in = [&](int piece) { return piece * 256 + 8 * lane < K; };
  Raw8<T> next[2];
  int piece = blockIdx.y;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (in(piece + i * step)) next[i] = load_raw8(wr + (piece + i * step) * 256);
  for (; piece * 256 < K; piece += 2 * step) {
    Raw8<T> now[2];
    GroupRange r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[i] = GroupRange{0u, 0.0f, 0.0f};
      now[i] = next[i];
      if (in(piece + i * step)) r[i] = range8(now[i], symmetric);
      if (in(piece + (2 + i) * step)) next[i] = load_raw8(wr + (piece + (2 + i) * step) * 256);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) join_lanes(r[i], width, symmetric);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = piece + i * step;
      if (!in(at)) continue;
      const GroupCode<T> c(r[i], symmetric);
      float v[8];
      values8(now[i], v);
      out[at * 32] = quantise8<T>(v, c.s, c.inv, c.z, c.least);
      if (first) {
        const int64_t g = row * groups + at * per + mine;
        from_f32(c.s, scale + g);
        if (zero) zero[g] = static_cast<uint8_t>(c.z);
      }
    }
  }
}

// Longer groups: a warp's at a time, read twice.
template <typename T>
__global__ void __launch_bounds__(256)
    k_quantize_int4_wide(const T* w, int64_t rows, int K, int group, int groups, int symmetric,
                         uint8_t* packed, T* scale, uint8_t* zero) {
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* wr = w + row * K;
  uint8_t* out = packed + row * (K / 2);
  for (int g = blockIdx.y; g < groups; g += gridDim.y) {
    const int k0 = g * group, k = k0 + 8 * lane, k1 = K - k0 < group ? K : k0 + group;
    GroupRange r{0u, 0.0f, 0.0f};
    float v[8];
#pragma unroll 4
    for (int j = k; j < k1; j += 256) {
      values8(load_raw8(wr + j), v);
      widen(r, v, symmetric);
    }
    join_lanes(r, 32, symmetric);
    const GroupCode<T> c(r, symmetric);
    if (lane == 0) {
      from_f32(c.s, scale + row * groups + g);
      if (zero) zero[row * groups + g] = static_cast<uint8_t>(c.z);
    }
#pragma unroll 4
    for (int j = k; j < k1; j += 256) {
      values8(load_raw8(wr + j), v);
      *reinterpret_cast<uint32_t*>(out + j / 2) = quantise8<T>(v, c.s, c.inv, c.z, c.least);
    }
  }
}

// Eight values per lane at a time, four of them on their way: scale * (q - zero) in fp32, rounded once. A warp
// takes every gridDim.y-th 1024 values of a row.
template <typename T, typename S>
__global__ void __launch_bounds__(256)
    k_dequantize_int4(const uint8_t* packed, const S* scale, const uint8_t* zero, int64_t rows, int K,
                      int groups, uint32_t magic, T* out) {
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const uint32_t* p = reinterpret_cast<const uint32_t*>(packed + row * (K / 2));
  const S* sr = scale + row * groups;
  const uint8_t* zr = zero ? zero + row * groups : nullptr;
  T* o = out + row * K;
  const int n = K / 8;
  for (int u0 = blockIdx.y * 128 + lane; u0 < n; u0 += gridDim.y * 128) {
    uint32_t q[4], z[4];
    S s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + 32 * i;
      if (u < n) {
        q[i] = __ldcg(p + u);
        const uint32_t g = __umulhi(static_cast<uint32_t>(u), magic);
        s[i] = sr[g];
        z[i] = zr ? zr[g] & 15u : 8u;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + 32 * i;
      if (u >= n) break;
      if constexpr (std::is_same<T, S>::value && sizeof(T) == 2) {
        // the product has at most 15 bits: rounded in 16 bits it is what fp32 would round to
        T* type = nullptr;
        const uint32_t hi = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&s[i])) * 0x00010001u;
        *reinterpret_cast<uint4*>(o + 8 * u) =
            weights8<T, false>(q[i], nibble_base(type) + z[i] * 0x00010001u, hi, 0u);
        continue;
      }
      // 2^23 + q less 2^23 + zero: exact
      const float base = 8388608.0f + static_cast<float>(z[i]), scale = to_f32(s[i]);
#pragma unroll
      for (int h = 0; h < 8; h += kV<T>) {
        float v[kV<T>];
#pragma unroll
        for (int l = 0; l < kV<T>; ++l)
          v[l] = (__uint_as_float(((q[i] >> (4 * (h + l))) & 15u) | 0x4b000000u) - base) * scale;
        store_pack(o + 8 * u + h, v);
      }
    }
  }
}

// ------------------------------------------------------------------ launches
// Blocks of eight rows, and how many blocks share a row: until there are 32 warps per SM.
dim3 row_grid(int64_t rows, int pieces, int sms) {
  const int64_t blocks = (rows + 7) / 8;
  int64_t share = (4 * sms + blocks - 1) / blocks;
  if (share > pieces) share = pieces;
  return dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(share));
}

template <typename T>
cudaError_t quantise(const Int4Weights& p, int sms, cudaStream_t s) {
  const T* w = static_cast<const T*>(p.w);
  T* scale = static_cast<T*>(p.scale);
  if (p.group > 256)
    return launch_pdl(k_quantize_int4_wide<T>, row_grid(p.rows, p.groups, sms), dim3(256), 0, s, w, p.rows,
                      p.K, p.group, p.groups, p.symmetric, p.packed, scale, p.zero);
  return launch_pdl(k_quantize_int4<T>, row_grid(p.rows, (p.K + 255) / 256, sms), dim3(256), 0, s, w,
                    p.rows, p.K, p.group, p.groups, p.symmetric, p.packed, scale, p.zero);
}

template <typename T, typename S>
cudaError_t dequantise(const Int4Weights& p, int sms, cudaStream_t s) {
  // u * magic >> 32 is u / (group / 8): u is below 2^14, which makes the product's error less than 2^-18, and a
  // longer group than that is all there is
  const uint32_t g8 = static_cast<uint32_t>(p.group / 8);
  const uint32_t magic = g8 > 16384 ? 0u : static_cast<uint32_t>((1ull << 32) / g8 + 1);
  return launch_pdl(k_dequantize_int4<T, S>, row_grid(p.rows, (p.K + 1023) / 1024, sms), dim3(256), 0, s,
                    static_cast<const uint8_t*>(p.packed), static_cast<const S*>(p.scale),
                    static_cast<const uint8_t*>(p.zero), p.rows, p.K, p.groups, magic, static_cast<T*>(p.w));
}

template <typename T>
cudaError_t dequantise(const Int4Weights& p, int sms, cudaStream_t s) {
  switch (p.scale_dtype) {
    case FMOE_DTYPE_F32:
      return dequantise<T, float>(p, sms, s);
    case FMOE_DTYPE_BF16:
      return dequantise<T, __nv_bfloat16>(p, sms, s);
    default:
      return dequantise<T, __half>(p, sms, s);
  }
}

template <typename T, int RT, int NT, int D, int W>
cudaError_t few(const I4Args& a, cudaStream_t s) {
  const dim3 grid((a.N + 16 * RT - 1) / (16 * RT), a.E);
  // a block of 128 values b, at most 1023, is in group (b * magic) >> 20 = b / (group / 128): the error of the
  // product is below 2^-10
  const int per = a.group / 128;
  const uint32_t magic = per == 0 || per > 1024 ? 0u : (1u << 20) / per + 1;
  if (a.group < 128)
    return launch_pdl(k_int4_few<T, RT, NT, D, W, true>, grid, dim3(W * 32), 0, s, a, magic);
  return launch_pdl(k_int4_few<T, RT, NT, D, W, false>, grid, dim3(W * 32), 0, s, a, magic);
}

template <typename T, int RT, int NT, int D>
cudaError_t few(const I4Args& a, int64_t used, int sms, cudaStream_t s) {
  // Short rows leave eight warps a step or two each, and the block's barrier at its end as long as its work.
  // Four warps and twice the blocks per SM, where there are blocks enough: 128 rows over 32 experts of 7168 x
  // 2048 take 95 us instead of 125, one of 7168 x 2048 5.2 instead of 6.2. But with 256 blocks four warps
  // leave SMs idle (1 x 4096 x 4096: 8.2 instead of 5.7), and with long rows eight are as good or better (32
  // rows over 16 experts of 4096 x 7168: 68 against 70, 128 rows: 130 against 150).
  const int64_t blocks = (a.N + 16ll * RT - 1) / (16 * RT) * used;
  if (a.K <= 4096 && blocks >= 2 * sms) return few<T, RT, NT, D, 4>(a, s);
  return few<T, RT, NT, D, 8>(a, s);
}

template <typename T>
cudaError_t few(const I4Args& a, int64_t used, int64_t per, int sms, cudaStream_t s) {
  // 32 rows per block share the tokens' loads, as long as there are blocks enough
  const bool tall = (a.N + 31) / 32 * used >= 4 * sms;
  if (per <= 8) return tall ? few<T, 2, 1, 2>(a, used, sms, s) : few<T, 1, 1, 4>(a, used, sms, s);
  return few<T, 1, 2, 2>(a, used, sms, s);
}

}  // namespace

cudaError_t launch_quantize_int4(const Int4Weights& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return quantise<float>(p, sms, s);
    case FMOE_DTYPE_BF16:
      return quantise<__nv_bfloat16>(p, sms, s);
    default:
      return quantise<__half>(p, sms, s);
  }
}

cudaError_t launch_dequantize_int4(const Int4Weights& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return dequantise<float>(p, sms, s);
    case FMOE_DTYPE_BF16:
      return dequantise<__nv_bfloat16>(p, sms, s);
    default:
      return dequantise<__half>(p, sms, s);
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
  return p.dtype == FMOE_DTYPE_BF16 ? few<__nv_bfloat16>(a, used, per, sms, s)
                                    : few<__half>(a, used, per, sms, s);
}

}  // namespace fmoe
