// fmoe_layernorm.cu -- layer norm of the residual stream in front of a block, forward and backward.
//
//   hidden = residual + branch                      (branch may be absent)
//   mean, var = over the row's H columns,  r = 1 / sqrt(var + eps),  n = (hidden - mean) * r
//   normed = n * weight + bias
// and with dh, dy the gradients of hidden and normed, u = dy * weight:
//   d branch = d residual = dh + r * (u - mean(u) - n * mean(u * n))
//   d weight = sum over rows of dy * n,  d bias = sum over rows of dy
//
// A row is read once and stays in registers, up to 32 values per thread, so the variance is taken of the
// deviations from the mean and not from a difference of squares. Short rows are a warp's, longer ones a
// block's. Everything is fp32 between the load and the one rounding on the way out. Bound by HBM; the
// figures stand at the kernels.
#include <atomic>
#include <type_traits>

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

struct LnArgs {
  const void *f, *x, *w, *b;  // branch or null, residual, weight or null, bias or null
  int w_f32, b_f32;
  float eps;
  int64_t T;
  int H;
  // forward
  void *h, *y;                // each may be null
  uint8_t* q;                 // or e4m3 with scales [H / 128, T]
  float *q_scale, *stats;     // stats [T, 2]: mean, r (or null)
  // backward
  const void *dh, *dy;        // null: zero
  void* dx;                   // or null
  float* part;                // [2][blocks][H]: d weight, d bias; 16-byte aligned
  int want_w, want_b;
};

// A unit of a row: V elements (a 16-byte granule, or 1 where rows are not on 16-byte boundaries) as fp32, in
// pairs for the packed instructions or singly.
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float mad(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 mad(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float total(float a) { return a; }
__device__ __forceinline__ float total(float2 a) { return a.x + a.y; }
__device__ __forceinline__ void set(float& a, float s) { a = s; }
__device__ __forceinline__ void set(float2& a, float s) { a = make_float2(s, s); }

template <typename T, int V>
struct Unit {
  using P = typename std::conditional<V == 1, float, float2>::type;
  static constexpr int N = V > 1 ? V / 2 : 1;
  P p[N];
};
template <typename P>
__device__ __forceinline__ P all(float s) {
  P a;
  set(a, s);
  return a;
}
template <typename T, int V>
__device__ __forceinline__ Unit<T, V> unit_of(const Pack<T, V>& r) {
  Unit<T, V> u;
  float v[V];
  unpack(r, v);
  if constexpr (V == 1) {
    u.p[0] = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < Unit<T, V>::N; ++i) u.p[i] = make_float2(v[2 * i], v[2 * i + 1]);
  }
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void store_unit(T* p, const Unit<T, V>& u) {
  if constexpr (V == 1) {
    from_f32(u.p[0], p);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(u.p[0].x, u.p[0].y, u.p[1].x, u.p[1].y);
  } else {
    T* type = nullptr;
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(type, u.p[0].x, u.p[0].y), pack2(type, u.p[1].x, u.p[1].y),
                                              pack2(type, u.p[2].x, u.p[2].y), pack2(type, u.p[3].x, u.p[3].y));
  }
}

// V consecutive parameters as fp32.
template <typename T, int V>
__device__ __forceinline__ Unit<T, V> param(const void* p, int f32, int i) {
  if (!f32) return unit_of(load_pack<T, V>(static_cast<const T*>(p) + i));
  const float* s = static_cast<const float*>(p) + i;
  Unit<T, V> u;
  if constexpr (V == 1) {
    u.p[0] = __ldcg(s);
  } else {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 w = __ldcg(reinterpret_cast<const float4*>(s + 4 * j));
      u.p[2 * j] = make_float2(w.x, w.y);
      u.p[2 * j + 1] = make_float2(w.z, w.w);
    }
  }
  return u;
}

// Rows off the 16-byte boundaries (ODD): the units are memory's granules. A row's first column is element `off`
// of its first unit, the same in every tensor, and in every row of a block: their distance is a multiple of
// 16 bytes, so that a thread's columns and the block's parameters in shared memory stay what they are. Unit i has
// columns c .. c + V - 1, c = i * V - off; those below 0 and from H on are another row's: read, and never
// written. With hidden in the residual's place that row's block may be writing them meanwhile, so what was read is
// of no use: keep() puts zeros in their place before any sum over the row.
template <int V>
__device__ __forceinline__ bool whole(int c, int H) {
  return c >= 0 && c + V <= H;
}
template <typename T, int V>
__device__ __forceinline__ void keep(Unit<T, V>& u, int c, int H) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < Unit<T, V>::N; ++j) {
      if (c + 2 * j < 0 || c + 2 * j >= H) u.p[j].x = 0.0f;
      if (c + 2 * j + 1 < 0 || c + 2 * j + 1 >= H) u.p[j].y = 0.0f;
    }
  }
}
// The first `some` elements of a unit behind which the tensor ends.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_some(const T* p, int some) {
  Pack<T, V> r = {};
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j >= some) break;
      if constexpr (sizeof(T) == 4)
        r.w[j] = __ldcg(reinterpret_cast<const uint32_t*>(p) + j);
      else
        r.w[j / 2] |= static_cast<uint32_t>(__ldcg(reinterpret_cast<const uint16_t*>(p) + j)) << (16 * (j & 1));
    }
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_cols(T* p, const Unit<T, V>& u, int c, int H) {
  if (whole<V>(c, H)) return store_unit(p, u);
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c + j >= 0 && c + j < H) from_f32(j & 1 ? u.p[j / 2].y : u.p[j / 2].x, p + j);
  }
}
// A unit's parameters, zeros in other rows' columns.
template <typename T, int V>
__device__ __forceinline__ Unit<T, V> param_cols(const void* p, int f32, int c, int H) {
  Unit<T, V> u;
  if constexpr (V > 1) {
    if (f32) {
#pragma unroll
      for (int j = 0; j < Unit<T, V>::N; ++j)
        u.p[j] = make_float2(__ldcg(static_cast<const float*>(p) + min(max(c + 2 * j, 0), H - 1)),
                             __ldcg(static_cast<const float*>(p) + min(max(c + 2 * j + 1, 0), H - 1)));
    } else {
      T v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = load_pack<T, 1>(static_cast<const T*>(p) + min(max(c + j, 0), H - 1)).e;
#pragma unroll
      for (int j = 0; j < Unit<T, V>::N; ++j) u.p[j] = make_float2(to_f32(v[2 * j]), to_f32(v[2 * j + 1]));
    }
    if (!whole<V>(c, H)) keep(u, c, H);
  }
  return u;
}

// The most that a row's units hold, wherever its first column is.
constexpr int odd_floats(int H, int V) { return (H + 2 * V - 2) / V * V; }

// Parameters in shared memory as fp32: unit i's values in V / 4 planes of float4, so that a warp's
// 16-byte reads are next to each other (V = 1: plain).
template <typename T, int V>
__device__ __forceinline__ void put_param(float* s, int n, int i, const Unit<T, V>& u) {
  if constexpr (V == 1) {
    s[i] = u.p[0];
  } else {
#pragma unroll
    for (int p = 0; p < V / 4; ++p)
      reinterpret_cast<float4*>(s)[p * n + i] =
          make_float4(u.p[2 * p].x, u.p[2 * p].y, u.p[2 * p + 1].x, u.p[2 * p + 1].y);
  }
}
template <typename T, int V>
__device__ __forceinline__ Unit<T, V> get_param(const float* s, int n, int i) {
  Unit<T, V> u;
  if constexpr (V == 1) {
    u.p[0] = s[i];
  } else {
#pragma unroll
    for (int p = 0; p < V / 4; ++p) {
      const float4 w = reinterpret_cast<const float4*>(s)[p * n + i];
      u.p[2 * p] = make_float2(w.x, w.y);
      u.p[2 * p + 1] = make_float2(w.z, w.w);
    }
  }
  return u;
}

// Blocks per SM that the forward kernel's registers are to leave room for: 128 per thread with 32 values, else
// 80. Fewer threads with more values each are better than the reverse, since a warp's sums and barrier cost
// as much as the arithmetic of 16 values: 3000 x 7168 took 49 us with 512 threads per row.
constexpr int ln_blocks(int G, int values) {
  const int threads = G == 32 ? 256 : G;
  const int most = (values > 16 ? 512 : 768) / threads;
  return most < 1 ? 1 : most;
}

// ------------------------------------------------------------------ forward
// G threads share a row, U units each, G apart: a warp per row (G = 32, eight warps per block), or a block.
// Both are known to the compiler, so that a thread's units are at fixed distances: with the block size left
// open the kernel took 29 instructions per element, most of them addresses, and 8192 x 7168 172 us. SP: the
// parameters are kept in shared memory for the block's rows, else read where they are used (few rows per
// block).
template <typename T, int V, int U, int G, bool SP, bool ODD>
__global__ void __launch_bounds__(G == 32 ? 256 : G, ln_blocks(G, U * V))
    k_layer_norm(const LnArgs a) {
  constexpr bool WARP = G == 32, AHEAD = V > 1;
  constexpr int WARPS = WARP ? 1 : G / 32;  // that share a row
  using Un = Unit<T, V>;
  using P = typename Un::P;
  extern __shared__ float4 ln_smem[];
  float* sw = reinterpret_cast<float*>(ln_smem);
  float* sb = sw + (ODD ? odd_floats(a.H, V) : a.H);
  __shared__ float4 part[2][32];  // a warp's sum, squared deviations and what its mean's rounding left
  __shared__ float2 count[32];
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = WARP ? lane : static_cast<int>(threadIdx.x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 8 : 1);
  int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  const int off = ODD ? static_cast<int>(row * a.H & (V - 1)) : 0;
  const int n = ODD ? (off + a.H + V - 1) / V : a.H / V;
  const int64_t at = row * a.H + g * V - off, by = step * a.H;
  const T* x = static_cast<const T*>(a.x) + at;
  const T* f = a.f ? static_cast<const T*>(a.f) + at : nullptr;
  T* h = a.h ? static_cast<T*>(a.h) + at : nullptr;
  T* yo = a.y ? static_cast<T*>(a.y) + at : nullptr;

  Pack<T, V> nx[U], nf[U];
  // Unit u of a row is loaded as a whole unless it passes the tensor's end, `left` elements behind the row's
  // first; if it does, by elements and only when it is used, since a branch around loads on their way would
  // wait for them (4096 x 4095 took 71 us with it).
  const auto behind = [&](int64_t r) -> int {
    const int64_t left = (a.T - r) * a.H;
    return left < (1 << 30) ? static_cast<int>(left) : 1 << 30;
  };
  const auto here = [&](int u, int left) {
    return u * G + g < n && (!ODD || (u * G + g + 1) * V - off <= left);
  };
  const auto finish = [&](Pack<T, V>& to, const T* p, int u, int left) {
    if (ODD && !here(u, left)) to = load_some<T, V>(p + u * G * V, left - ((u * G + g) * V - off));
  };
  const auto fetch = [&](int64_t r) {
    if (r >= a.T) return;
    const int left = ODD ? behind(r) : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (here(u, left)) nx[u] = load_pack<T, V>(x + u * G * V);
    x += by;
    if (f) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (here(u, left)) nf[u] = load_pack<T, V>(f + u * G * V);
      f += by;
    }
  };
  if constexpr (AHEAD) fetch(row);

  const auto read = [&](const void* p, int f32, int i) {
    return ODD ? param_cols<T, V>(p, f32, i * V - off, a.H) : param<T, V>(p, f32, i * V);
  };
  if constexpr (SP) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      if (a.w) put_param(sw, n, i, read(a.w, a.w_f32, i));
      if (a.b) put_param(sb, n, i, read(a.b, a.b_f32, i));
    }
  }
  // elements of a row that this warp has
  int mine = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (u * G + (WARP ? 0 : warp * 32)) * V - off;
    mine += max(0, min(c + 32 * V, a.H) - max(c, 0));
  }
  const float own = static_cast<float>(mine > 0 ? mine : 1), cols = static_cast<float>(a.H);
  const float own_inv = mine > 0 ? 1.0f / own : 0.0f;
  if (!WARP && lane == 0) count[warp] = make_float2(static_cast<float>(mine), own_inv);
  if (SP || !WARP) __syncthreads();
  const float inv_h = 1.0f / cols;

  for (int flip = 0; row < a.T; row += step, flip ^= 1) {
    if constexpr (!AHEAD) fetch(row);
    const int now = ODD ? behind(row) : 0;
    Un v[U];
    P two = all<P>(0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * G + g < n) {
        finish(nx[u], x - by, u, now);
        v[u] = unit_of(nx[u]);
        if (a.f) {
          finish(nf[u], f - by, u, now);
          const Un w = unit_of(nf[u]);
#pragma unroll
          for (int j = 0; j < Un::N; ++j) v[u].p[j] = add(v[u].p[j], w.p[j]);
        }
        if (ODD && !whole<V>((u * G + g) * V - off, a.H)) keep(v[u], (u * G + g) * V - off, a.H);
      }
    }
    if constexpr (AHEAD) fetch(row + step);
    if (h) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u * G + g < n) {
          if constexpr (ODD)
            store_cols(h + u * G * V, v[u], (u * G + g) * V - off, a.H);
          else
            store_unit(h + u * G * V, v[u]);
        }
      h += by;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * G + g < n) {
#pragma unroll
        for (int j = 0; j < Un::N; ++j) two = add(two, v[u].p[j]);
      }
    }
    // the warp's own mean and squared deviations first, then all warps' joined: one barrier a row
    const float sum = warp_sum_f32(total(two));
    // the mean is divided, not multiplied with a rounded 1 / H: equal values whose sum is exact are their mean. A
    // warp's own is rounded before it is used, here and below: `left` is what that rounding left.
    float mean = WARP ? __fdiv_rn(sum, own) : __fmul_rn(sum, own_inv);
    two = all<P>(0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * G + g < n) {
        Un d;
#pragma unroll
        for (int j = 0; j < Un::N; ++j) d.p[j] = add(v[u].p[j], all<P>(-mean));
        if (ODD && !whole<V>((u * G + g) * V - off, a.H)) keep(d, (u * G + g) * V - off, a.H);
#pragma unroll
        for (int j = 0; j < Un::N; ++j) two = mad(d.p[j], d.p[j], two);
      }
    }
    float dev = warp_sum_f32(total(two));
    // A mean beyond 2^12 deviations: the rounding of its sum is no longer small beside them (rows of 3000 fp32
    // values around 10^5 deviations: normed off by 0.015; now by 0.004, half a step of the mean). What is left of
    // it is the mean of the deviations from it, whose square is taken off theirs. A row of equal values has that value
    // as its mean.
    const auto far = [](float m, float var) { return var < m * m * 0x1p-24f; };
    float left = 0.0f;
    if (far(mean, dev * own_inv)) {
      P rest = all<P>(0.0f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u * G + g < n) {
          Un d;
#pragma unroll
          for (int j = 0; j < Un::N; ++j) d.p[j] = add(v[u].p[j], all<P>(-mean));
          if (ODD && !whole<V>((u * G + g) * V - off, a.H)) keep(d, (u * G + g) * V - off, a.H);
#pragma unroll
          for (int j = 0; j < Un::N; ++j) rest = add(rest, d.p[j]);
        }
      }
      const float all_rest = warp_sum_f32(total(rest));
      left = all_rest * own_inv;
      dev = fmaxf(dev - all_rest * left, 0.0f);
      if (WARP) mean += left;
    }
    if constexpr (!WARP) {
      if (lane == 0) part[flip][warp] = make_float4(sum, dev, left, 0.0f);
      __syncthreads();
      // a lane per warp (all of them unrolled took too many registers)
      const float4 p = lane < WARPS ? part[flip][lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      mean = __fdiv_rn(warp_sum_f32(p.x), cols);
      const float2 c = lane < WARPS ? count[lane] : make_float2(0.0f, 0.0f);
      // without columns there is no mean of its own: 0 * (0 - mean)^2 would be NaN where the square is infinite
      const float away = c.x > 0.0f ? __fsub_rn(__fmul_rn(p.x, c.y), mean) + p.z : 0.0f;
      dev = warp_sum_f32(fmaf(away * away, c.x, p.y));
      // beside the sum above: 4096 x 2047 takes 49 us, behind a branch 50, the row's correction as a whole behind
      // one and another barrier 57 (47 without any)
      left = warp_sum_f32(away * c.x) * inv_h;
      if (far(mean, dev * inv_h)) {
        dev = fmaxf(dev - left * left * cols, 0.0f);
        mean += left;
      }
    }
    const float r = rsqrtf(fmaf(dev, inv_h, a.eps));
    if (a.stats && g == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, r);
    if (!yo && !a.q) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      const bool in = i < n;
      Un y;
      if (in) {
#pragma unroll
        for (int j = 0; j < Un::N; ++j) y.p[j] = mul(add(v[u].p[j], all<P>(-mean)), all<P>(r));
        if (a.w) {
          const Un w = SP ? get_param<T, V>(sw, n, i) : read(a.w, a.w_f32, i);
#pragma unroll
          for (int j = 0; j < Un::N; ++j) y.p[j] = mul(y.p[j], w.p[j]);
        }
        if (a.b) {
          const Un b = SP ? get_param<T, V>(sb, n, i) : read(a.b, a.b_f32, i);
#pragma unroll
          for (int j = 0; j < Un::N; ++j) y.p[j] = add(y.p[j], b.p[j]);
        }
        if (ODD && yo)
          store_cols(yo + u * G * V, y, i * V - off, a.H);
        else if (yo)
          store_unit(yo + u * G * V, y);
      }
      if constexpr (V > 1 && !ODD) {
        if (a.q) {
          // 128 columns are the units of 128 / V neighbouring lanes, which are inside the row or
          // outside together (H is a multiple of 128)
          float m = 0.0f;
          if (in) {
#pragma unroll
            for (int j = 0; j < Un::N; ++j) m = fmaxf(m, fmaxf(fabsf(y.p[j].x), fabsf(y.p[j].y)));
          }
#pragma unroll
          for (int o = 64 / V; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (in) {
            const float scale = __fdiv_rn(fmaxf(m, 1e-30f), 448.0f);
            uint32_t w[V / 4];
#pragma unroll
            for (int j = 0; j < V / 4; ++j) {
              const float2 lo = y.p[2 * j], hi = y.p[2 * j + 1];
              w[j] = static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(lo.x, scale), __fdiv_rn(lo.y, scale))) |
                     static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(hi.x, scale), __fdiv_rn(hi.y, scale)))
                         << 16;
            }
            uint8_t* q = a.q + row * a.H + i * V;
            if constexpr (V == 8)
              *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
            else
              *reinterpret_cast<uint32_t*>(q) = w[0];
            if (i % (128 / V) == 0) a.q_scale[static_cast<int64_t>(i / (128 / V)) * a.T + row] = scale;
          }
        }
      }
    }
    if (yo) yo += by;
  }
}

// ------------------------------------------------------------------ backward
// As above, a row's inputs loaded one row ahead where a thread has no more than 16 values. The sums over rows are in registers, or (WIDE, more than 16 values per thread) in shared memory, each
// thread's own.
template <typename T, int V, int U, int G, bool WIDE, bool ODD>
__global__ void __launch_bounds__(G == 32 ? 256 : G, 1) k_layer_norm_back(const LnArgs a) {
  constexpr bool WARP = G == 32, AHEAD = V > 1 && !WIDE;
  constexpr int WARPS = WARP ? 1 : G / 32;
  using Un = Unit<T, V>;
  using P = typename Un::P;
  constexpr int N = Un::N;
  extern __shared__ float4 ln_smem[];
  float* sw = reinterpret_cast<float*>(ln_smem);   // weight [H]
  P* acc = reinterpret_cast<P*>(sw + ((ODD ? odd_floats(a.H, V) : a.H) + 3) / 4 * 4);  // WIDE: [2][U * N][G]
  float* rows = sw;                                // WARP, at the end: [8][2][H]
  __shared__ float2 part[2][32];
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = WARP ? lane : static_cast<int>(threadIdx.x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 8 : 1);
  int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  const int off = ODD ? static_cast<int>(row * a.H & (V - 1)) : 0;
  const int n = ODD ? (off + a.H + V - 1) / V : a.H / V;
  const int64_t at = row * a.H + g * V - off, by = step * a.H;
  const bool dy_in = a.dy != nullptr, f_in = dy_in && a.f != nullptr;
  const T* x = static_cast<const T*>(a.x) + at;
  const T* f = f_in ? static_cast<const T*>(a.f) + at : nullptr;
  const T* dy = dy_in ? static_cast<const T*>(a.dy) + at : nullptr;
  const T* dh = a.dh ? static_cast<const T*>(a.dh) + at : nullptr;
  T* dx = a.dx ? static_cast<T*>(a.dx) + at : nullptr;
  const float inv_h = 1.0f / static_cast<float>(a.H);

  struct Row {
    Pack<T, V> x[U], f[U], dy[U];
    float2 stat;
  } next;
  // Unit u of a row is loaded as a whole unless it passes the tensor's end, `left` elements behind the row's
  // first; if it does, by elements and only when it is used, since a branch around loads on their way would
  // wait for them (4096 x 4095 took 71 us with it).
  const auto behind = [&](int64_t r) -> int {
    const int64_t left = (a.T - r) * a.H;
    return left < (1 << 30) ? static_cast<int>(left) : 1 << 30;
  };
  const auto here = [&](int u, int left) {
    return u * G + g < n && (!ODD || (u * G + g + 1) * V - off <= left);
  };
  const auto finish = [&](Pack<T, V>& to, const T* p, int u, int left) {
    if (ODD && !here(u, left)) to = load_some<T, V>(p + u * G * V, left - ((u * G + g) * V - off));
  };
  const auto fetch = [&](int64_t r) {
    if (r >= a.T) return;
    const int left = ODD ? behind(r) : 0;
    next.stat = __ldcg(reinterpret_cast<const float2*>(a.stats) + r);
    if (dy_in) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (here(u, left)) next.x[u] = load_pack<T, V>(x + u * G * V);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (here(u, left)) next.dy[u] = load_pack<T, V>(dy + u * G * V);
      x += by;
      dy += by;
    }
    if (f) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (here(u, left)) next.f[u] = load_pack<T, V>(f + u * G * V);
      f += by;
    }
  };
  if constexpr (AHEAD) fetch(row);

  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    Un one;
#pragma unroll
    for (int j = 0; j < N; ++j) one.p[j] = all<P>(1.0f);
    if (a.w) one = ODD ? param_cols<T, V>(a.w, a.w_f32, i * V - off, a.H) : param<T, V>(a.w, a.w_f32, i * V);
    put_param(sw, n, i, one);
  }
  Un aw[WIDE ? 1 : U], ab[WIDE ? 1 : U];
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < 2 * U * N * G; i += G) acc[i] = all<P>(0.0f);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < N; ++j) aw[u].p[j] = ab[u].p[j] = all<P>(0.0f);
  }
  __syncthreads();

  for (int flip = 0; row < a.T; row += step, flip ^= 1) {
    if constexpr (!AHEAD) fetch(row);
    const float mean = next.stat.x, r = next.stat.y;
    const int now = ODD ? behind(row) : 0;
    Un v[U], d[U];  // n, and dy and then u
    Pack<T, V> ph[U];
    P t1 = all<P>(0.0f), t2 = t1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (dh && here(u, now)) ph[u] = load_pack<T, V>(dh + u * G * V);
      if (dy_in && u * G + g < n) {
        finish(next.x[u], x - by, u, now);
        finish(next.dy[u], dy - by, u, now);
        v[u] = unit_of(next.x[u]);
        if (f_in) {
          finish(next.f[u], f - by, u, now);
          const Un t = unit_of(next.f[u]);
#pragma unroll
          for (int j = 0; j < N; ++j) v[u].p[j] = add(v[u].p[j], t.p[j]);
        }
        d[u] = unit_of(next.dy[u]);
        // other rows' columns are zeros: 0 * n with an infinite n of theirs would not be
        if (ODD && !whole<V>((u * G + g) * V - off, a.H)) {
          keep(v[u], (u * G + g) * V - off, a.H);
          keep(d[u], (u * G + g) * V - off, a.H);
        }
      }
    }
    if (dh) dh += by;
    if constexpr (AHEAD) fetch(row + step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (dy_in && u * G + g < n) {
        const Un w = get_param<T, V>(sw, n, u * G + g);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          v[u].p[j] = mul(add(v[u].p[j], all<P>(-mean)), all<P>(r));
          if constexpr (WIDE) {
            P* m = acc + (u * N + j) * G + g;
            m[0] = mad(d[u].p[j], v[u].p[j], m[0]);
            m[U * N * G] = add(d[u].p[j], m[U * N * G]);
          } else {
            aw[u].p[j] = mad(d[u].p[j], v[u].p[j], aw[u].p[j]);
            ab[u].p[j] = add(d[u].p[j], ab[u].p[j]);
          }
          d[u].p[j] = mul(d[u].p[j], w.p[j]);
          t1 = add(t1, d[u].p[j]);
          t2 = mad(d[u].p[j], v[u].p[j], t2);
        }
      }
    }
    if (!dx) continue;
    float s1 = warp_sum_f32(total(t1));
    float s2 = warp_sum_f32(total(t2));
    if constexpr (!WARP) {
      if (lane == 0) part[flip][warp] = make_float2(s1, s2);
      __syncthreads();
      const float2 p = lane < WARPS ? part[flip][lane] : make_float2(0.0f, 0.0f);
      s1 = warp_sum_f32(p.x);
      s2 = warp_sum_f32(p.y);
    }
    s1 *= inv_h;
    s2 *= inv_h;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * G + g < n) {
        Un o;
        if (dy_in) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const P m = mad(v[u].p[j], all<P>(-s2), add(d[u].p[j], all<P>(-s1)));
            o.p[j] = mul(m, all<P>(r));
          }
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) o.p[j] = all<P>(0.0f);
        }
        if (dh) {
          finish(ph[u], dh - by, u, now);
          const Un t = unit_of(ph[u]);
#pragma unroll
          for (int j = 0; j < N; ++j) o.p[j] = add(o.p[j], t.p[j]);
        }
        if constexpr (ODD)
          store_cols(dx + u * G * V, o, (u * G + g) * V - off, a.H);
        else
          store_unit(dx + u * G * V, o);
      }
    }
    dx += by;
  }

  if (!a.want_w && !a.want_b) return;
  float* pw = a.part + static_cast<int64_t>(blockIdx.x) * a.H;
  float* pb = pw + static_cast<int64_t>(gridDim.x) * a.H;
  const auto put = [&](float* to, int i, int j, const P& p) {  // pair j of unit i
    if constexpr (ODD) {
      const int c = i * V - off + 2 * j;
      if (c >= 0 && c < a.H) to[c] = p.x;
      if (c + 1 >= 0 && c + 1 < a.H) to[c + 1] = p.y;
    } else {
      *reinterpret_cast<P*>(to + i * V + 2 * j) = p;
    }
  };
  if constexpr (WARP) {
    __syncthreads();  // the weights are no longer read
    float* own = rows + warp * 2 * a.H;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      if (i < n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          put(own, i, j, aw[u].p[j]);
          put(own + a.H, i, j, ab[u].p[j]);
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.H; c += blockDim.x) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += rows[i * 2 * a.H + c];
      if (c < a.H)
        pw[c] = s;
      else
        pb[c - a.H] = s;
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      if (i < n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          put(pw, i, j, WIDE ? acc[(u * N + j) * G + g] : aw[WIDE ? 0 : u].p[j]);
          put(pb, i, j, WIDE ? acc[(U * N + u * N + j) * G + g] : ab[WIDE ? 0 : u].p[j]);
        }
      }
    }
  }
}

// The blocks' shares of d weight (blockIdx.y 0) and d bias (1), added in a fixed order: 32 columns per block,
// V of them per thread, 8 V threads per column, so that with V = 4 the usual 148 shares are one batch of
// loads per thread.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    k_layer_norm_sums(const float* part, int blocks, int H, void* dw, void* db, int w_f32, int b_f32) {
  pdl_begin_in_order();
  constexpr int ROWS = 8 * V;  // threads per column
  __shared__ float buf[ROWS][33];
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int f32 = blockIdx.y ? b_f32 : w_f32;
  const int x = threadIdx.x % (32 / V) * V, y = threadIdx.x / (32 / V);
  const int c = blockIdx.x * 32 + x;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * blocks * H;
  float sum[V] = {};
  if (c < H) {  // H is a multiple of V
    for (int b0 = y; b0 < blocks; b0 += ROWS * 5) {
      float v[5][V];
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const float* s = p + static_cast<int64_t>(b0 + ROWS * i) * H + c;
        const bool in = b0 + ROWS * i < blocks;
        if constexpr (V == 4) {
          const float4 w = in ? __ldcg(reinterpret_cast<const float4*>(s)) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[i][0] = w.x;
          v[i][1] = w.y;
          v[i][2] = w.z;
          v[i][3] = w.w;
        } else {
          v[i][0] = in ? __ldcg(s) : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 5; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += v[i][k];
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) buf[y][x + k] = sum[k];
  __syncthreads();
  if (threadIdx.x < 32 && blockIdx.x * 32 + threadIdx.x < H) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) s += buf[i][threadIdx.x];
    const int col = blockIdx.x * 32 + threadIdx.x;
    if (f32)
      static_cast<float*>(out)[col] = s;
    else
      from_f32(s, static_cast<T*>(out) + col);
  }
}

// ------------------------------------------------------------------ launches
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// two fp32 parameters of the longest row; the weight and two sums, and what ODD's units have beyond a row
constexpr int kLnMaxSmem = 3 * 16384 * 4 + 1024;

template <typename K>
cudaError_t allow_smem(K kernel, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLnMaxSmem);
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  return e;
}

LnArgs args_of(const LayerNorm& p) {
  LnArgs a{};
  a.f = p.f;
  a.x = p.x;
  a.w = p.w;
  a.b = p.b;
  a.w_f32 = p.w_dtype == FMOE_DTYPE_F32;
  a.b_f32 = p.b_dtype == FMOE_DTYPE_F32;
  a.eps = p.eps;
  a.T = p.T;
  a.H = p.H;
  a.h = p.h;
  a.y = p.y;
  a.q = static_cast<uint8_t*>(p.q);
  a.q_scale = p.q_scale;
  a.stats = p.stats;
  a.dh = p.dh;
  a.dy = p.dy;
  a.dx = p.dx;
  a.part = p.part;
  a.want_w = p.dw != nullptr;
  a.want_b = p.db != nullptr;
  return a;
}

// Blocks that share many rows: with ODD as many that the rows of each are multiples of 16 bytes apart.
template <int V, bool ODD>
int64_t aligned_blocks(int64_t most, int H) {
  if (!ODD) return most;
  int period = V;
  while (period > 1 && H % 2 == 0) {
    period /= 2;
    H /= 2;
  }
  return most / period * period;
}

template <typename T, int V, int U, int G, bool SP, bool ODD>
cudaError_t run_forward(const LnArgs& a, int64_t blocks, cudaStream_t s) {
  static std::atomic<bool> done[64];
  const size_t smem = SP ? static_cast<size_t>(ODD ? odd_floats(a.H, V) : a.H) * 8 : 0;
  if (smem > 44 * 1024) {  // of the 48 KB without opting in, some are static
    const cudaError_t e = allow_smem(k_layer_norm<T, V, U, G, SP, ODD>, done);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(k_layer_norm<T, V, U, G, SP, ODD>, dim3(static_cast<unsigned>(blocks)),
                    dim3(G == 32 ? 256 : G), smem, s, a);
}

template <typename T, int V, int U, int G, bool ODD>
cudaError_t forward(const LayerNorm& p, int sms, cudaStream_t s) {
  const LnArgs a = args_of(p);
  const int64_t blocks = G == 32 ? (p.T + 7) / 8 : p.T;
  // what runs at a time; with shared parameters for more rows than that
  const int64_t most = static_cast<int64_t>(sms) * ln_blocks(G, U * V);
  if (blocks <= most) return run_forward<T, V, U, G, false, ODD>(a, blocks, s);
  return run_forward<T, V, U, G, true, ODD>(a, aligned_blocks<V, ODD>(most, p.H), s);
}

template <typename T, int V, int U, int G, bool WIDE, bool ODD>
cudaError_t backward(const LayerNorm& p, int sms, cudaStream_t s) {
  static std::atomic<bool> done[64];
  const LnArgs a = args_of(p);
  size_t smem = (static_cast<size_t>(ODD ? odd_floats(p.H, V) : p.H) + 3) / 4 * 16;
  if (WIDE) smem += sizeof(typename Unit<T, V>::P) * 2 * U * Unit<T, V>::N * G;
  if (G == 32) smem = static_cast<size_t>(8) * 2 * p.H * 4;
  if (smem > 44 * 1024) {  // of the 48 KB without opting in, some are static
    const cudaError_t e = allow_smem(k_layer_norm_back<T, V, U, G, WIDE, ODD>, done);
    if (e != cudaSuccess) return e;
  }
  int64_t blocks = G == 32 ? (p.T + 7) / 8 : p.T;
  const int64_t most = static_cast<int64_t>(sms) * (G >= 512 ? 1 : 2);
  static_assert(kMaxLnBlocks >= 2 * 148, "shares of all blocks");
  if (blocks > most) blocks = aligned_blocks<V, ODD>(most, p.H);
  if (blocks > kMaxLnBlocks) blocks = kMaxLnBlocks / V * V;
  cudaError_t e = launch_pdl(k_layer_norm_back<T, V, U, G, WIDE, ODD>, dim3(static_cast<unsigned>(blocks)),
                             dim3(G == 32 ? 256 : G), smem, s, a);
  if (e != cudaSuccess || (!p.dw && !p.db)) return e;
  const auto sums = p.H % 4 == 0 ? k_layer_norm_sums<T, 4> : k_layer_norm_sums<T, 1>;
  return launch_pdl(sums, dim3((p.H + 31) / 32, 2), dim3(256), 0, s, static_cast<const float*>(p.part),
                    static_cast<int>(blocks), p.H, p.dw, p.db, a.w_f32, a.b_f32);
}

// The smallest variant that holds a row of n units.
template <typename T, int V, bool ODD>
cudaError_t sized(const LayerNorm& p, int sms, cudaStream_t s) {
  const int n = ODD ? (p.H + 2 * V - 2) / V : p.H / V;  // whatever the first column's place in its unit
  constexpr int A = V == 8 ? 1 : 2;  // of fp32, twice the units are as many values per thread
  if constexpr (V > 1) {
    if (p.back) {
      if (!ODD && n <= 32 * A) return backward<T, V, A, 32, false, false>(p, sms, s);
      if (!ODD && n <= 64 * A) return backward<T, V, 2 * A, 32, false, false>(p, sms, s);
      if (!ODD && n <= 256 * A) return backward<T, V, A, 256, false, false>(p, sms, s);
      if (n <= 512 * A) return backward<T, V, 2 * A, 256, false, ODD>(p, sms, s);
      if (n <= 1024 * A) return backward<T, V, 2 * A, 512, false, ODD>(p, sms, s);
      return backward<T, V, 2 * A, 1024, true, ODD>(p, sms, s);
    }
    if (!ODD && n <= 32 * A) return forward<T, V, A, 32, false>(p, sms, s);
    if (!ODD && n <= 64 * A) return forward<T, V, 2 * A, 32, false>(p, sms, s);
    if (!ODD && n <= 128 * A) return forward<T, V, 4 * A, 32, false>(p, sms, s);
    if (!ODD && n <= 256 * A) return forward<T, V, 2 * A, 128, false>(p, sms, s);
    if (n <= 512 * A) return forward<T, V, 4 * A, 128, ODD>(p, sms, s);
    if (n <= 768 * A) return forward<T, V, 3 * A, 256, ODD>(p, sms, s);
    if (n <= 1024 * A) return forward<T, V, 4 * A, 256, ODD>(p, sms, s);
    return forward<T, V, 4 * A, 512, ODD>(p, sms, s);
  } else {
    if (p.back) {
      if (n <= 128) return backward<T, 1, 4, 32, false, ODD>(p, sms, s);
      if (n <= 1024) return backward<T, 1, 4, 256, false, ODD>(p, sms, s);
      if (n <= 2048) return backward<T, 1, 8, 256, false, ODD>(p, sms, s);
      if (n <= 4096) return backward<T, 1, 8, 512, false, ODD>(p, sms, s);
      if (n <= 8192) return backward<T, 1, 16, 512, false, ODD>(p, sms, s);
      return backward<T, 1, 16, 1024, true, ODD>(p, sms, s);
    }
    if (p.q) return cudaErrorInvalidValue;  // the caller checks the alignment
    if (n <= 128) return forward<T, 1, 4, 32, ODD>(p, sms, s);
    if (n <= 1024) return forward<T, 1, 8, 128, ODD>(p, sms, s);
    if (n <= 2048) return forward<T, 1, 16, 128, ODD>(p, sms, s);
    if (n <= 4096) return forward<T, 1, 16, 256, ODD>(p, sms, s);
    if (n <= 8192) return forward<T, 1, 32, 256, ODD>(p, sms, s);
    return forward<T, 1, 32, 512, ODD>(p, sms, s);
  }
}

template <typename T>
cudaError_t typed(const LayerNorm& p, int sms, cudaStream_t s) {
  constexpr int V = kV<T>;
  bool wide = true;
  for (const void* q : {p.f, p.x, p.w, p.b, p.dh, p.dy, static_cast<const void*>(p.h),
                        static_cast<const void*>(p.y), static_cast<const void*>(p.dx)})
    wide = wide && on16(q);
  if (wide && p.H % V == 0) return sized<T, V, false>(p, sms, s);
  // Off the boundary, long rows go by memory's 16 bytes and shorter ones by elements: 3001 rows of 7001 bf16
  // columns take 47 us instead of 205 (with gradients 140 instead of 515; 3000 of 7168: 34 and 92), but 500 of
  // 1407 took 16 instead of 11, for the parameters that each row then gathers by elements. The largest
  // variants hold 16384 columns.
  if (wide && !p.q && p.H > 2048 && p.H + 2 * V - 2 <= 16384) return sized<T, V, true>(p, sms, s);
  return sized<T, 1, false>(p, sms, s);
}

}  // namespace

cudaError_t launch_layer_norm(const LayerNorm& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return typed<float>(p, sms, s);
    case FMOE_DTYPE_BF16:
      return typed<__nv_bfloat16>(p, sms, s);
    default:
      return typed<__half>(p, sms, s);
  }
}

}  // namespace fmoe
