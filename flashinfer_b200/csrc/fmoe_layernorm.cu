// fmoe_layernorm.cu -- layer norm of the residual stream in front of a block, forward and backward.
//
//   hidden = residual + branch                      (branch may be absent)
//   mean, var = over the row's H columns,  r = 1 / sqrt(var + eps),  n = (hidden - mean) * r
//   normed = n * weight + bias
// and with dh, dy the gradients of hidden and normed, u = dy * weight:
//   d branch = d residual = dh + r * (u - mean(u) - n * mean(u * n))
//   d weight = sum over rows of dy * n,  d bias = sum over rows of dy
//
// A row is read once and stays in registers, 32 values per thread (16 in the backward pass), so the
// variance is taken of the deviations from the mean and not from a difference of squares. Rows of up to
// 1024 (512) columns are a warp's, longer ones a block's. Everything is fp32 between the load and the
// one rounding on the way out. Bound by HBM; the figures stand at the kernels.
#include <atomic>

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
  float* part;                // [2][blocks][H]: d weight, d bias
  int want_w, want_b;
};

// V consecutive parameters as fp32.
template <typename T, int V>
__device__ __forceinline__ void param(const void* p, int f32, int i, float (&v)[V]) {
  if (f32) {
    const float* s = static_cast<const float*>(p) + i;
    if constexpr (V >= 4) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 w = __ldcg(reinterpret_cast<const float4*>(s + j));
        v[j] = w.x;
        v[j + 1] = w.y;
        v[j + 2] = w.z;
        v[j + 3] = w.w;
      }
    } else {
      v[0] = __ldcg(s);
    }
  } else {
    unpack(load_pack<T, V>(static_cast<const T*>(p) + i), v);
  }
}

// Parameters in shared memory as fp32: unit i's values in V / 4 planes of float4, so that a warp's
// 16-byte reads are next to each other (V = 1: plain).
template <int V>
__device__ __forceinline__ void put_param(float* s, int n, int i, const float (&v)[V]) {
  if constexpr (V == 1) {
    s[i] = v[0];
  } else {
#pragma unroll
    for (int p = 0; p < V / 4; ++p)
      reinterpret_cast<float4*>(s)[p * n + i] =
          make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
  }
}
template <int V>
__device__ __forceinline__ void get_param(const float* s, int n, int i, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = s[i];
  } else {
#pragma unroll
    for (int p = 0; p < V / 4; ++p) {
      const float4 w = reinterpret_cast<const float4*>(s)[p * n + i];
      v[4 * p] = w.x;
      v[4 * p + 1] = w.y;
      v[4 * p + 2] = w.z;
      v[4 * p + 3] = w.w;
    }
  }
}

// ------------------------------------------------------------------ forward
// T: element type. V: elements per unit (a 16-byte granule, or 1 where rows are not on 16-byte
// boundaries). A thread has U = 32 / V units, G threads apart. WARP: a row per warp (G = 32), eight
// warps per block; else a row per block of G threads. SP: the parameters are kept in shared memory for
// the block's rows, else read where they are used (few rows per block).
template <typename T, int V, bool WARP, bool SP>
__global__ void __launch_bounds__(WARP ? 256 : 512) k_layer_norm(const LnArgs a) {
  constexpr int U = 32 / V;
  // 16-bit rows: the next row's loads are under way while this one is worked on
  constexpr bool AHEAD = V == 8;
  extern __shared__ float4 ln_smem[];
  float* sw = reinterpret_cast<float*>(ln_smem);
  float* sb = sw + a.H;
  __shared__ float2 part[2][16];
  __shared__ float count[16], inv_count[16];
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int g = WARP ? lane : static_cast<int>(threadIdx.x);
  const int n = a.H / V;
  const T* x = static_cast<const T*>(a.x);
  const T* f = static_cast<const T*>(a.f);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 8 : 1);
  int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;

  Pack<T, V> nx[AHEAD ? U : 1], nf[AHEAD ? U : 1];
  const auto fetch = [&](int64_t r, int u) {
    const int i = u * G + g;
    if (r < a.T && i < n) {
      const int64_t at = r * a.H + static_cast<int64_t>(i) * V;
      nx[AHEAD ? u : 0] = load_pack<T, V>(x + at);
      if (f) nf[AHEAD ? u : 0] = load_pack<T, V>(f + at);
    }
  };
  if constexpr (AHEAD) {
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(row, u);
  }

  if (SP) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      float v[V];
      if (a.w) {
        param<T, V>(a.w, a.w_f32, i * V, v);
        put_param<V>(sw, n, i, v);
      }
      if (a.b) {
        param<T, V>(a.b, a.b_f32, i * V, v);
        put_param<V>(sb, n, i, v);
      }
    }
  }
  // elements of this row that this warp has
  int mine = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int first = u * G + (WARP ? 0 : warp * 32);
    mine += max(0, min(32, n - first)) * V;
  }
  const float own = static_cast<float>(mine > 0 ? mine : 1), cols = static_cast<float>(a.H);
  if (!WARP && lane == 0) {
    count[warp] = static_cast<float>(mine);
    inv_count[warp] = mine > 0 ? 1.0f / own : 0.0f;
  }
  if (SP || !WARP) __syncthreads();
  const float inv_h = 1.0f / static_cast<float>(a.H);

  for (int flip = 0; row < a.T; row += step, flip ^= 1) {
    float v[U][V];
    float sum = 0.0f;
    T* hr = static_cast<T*>(a.h) + row * a.H;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      if constexpr (!AHEAD) fetch(row, u);
      if (i < n) {
        unpack(nx[AHEAD ? u : 0], v[u]);
        if (f) {
          float w[V];
          unpack(nf[AHEAD ? u : 0], w);
#pragma unroll
          for (int j = 0; j < V; ++j) v[u][j] += w[j];
        }
        if (a.h) store_pack(hr + static_cast<int64_t>(i) * V, v[u]);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[u][j];
      }
    }
    if constexpr (AHEAD) {
#pragma unroll
      for (int u = 0; u < U; ++u) fetch(row + step, u);
    }
    // the warp's own mean and squared deviations first, then all warps' joined: one barrier a row
    sum = warp_sum_f32(sum);
    // divided, not multiplied with a rounded 1 / H: equal values whose sum is exact are their mean
    float mean = __fdiv_rn(sum, own);
    float dev = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * G + g < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[u][j] - mean;
          dev = fmaf(d, d, dev);
        }
      }
    }
    dev = warp_sum_f32(dev);
    if (!WARP) {
      if (lane == 0) part[flip][warp] = make_float2(sum, dev);
      __syncthreads();
      const int warps = G >> 5;
      float total = 0.0f;
      for (int i = 0; i < warps; ++i) total += part[flip][i].x;
      mean = __fdiv_rn(total, cols);
      dev = 0.0f;
      for (int i = 0; i < warps; ++i) {
        const float2 p = part[flip][i];
        const float d = p.x * inv_count[i] - mean;
        dev += fmaf(d * d, count[i], p.y);
      }
    }
    const float r = rsqrtf(fmaf(dev, inv_h, a.eps));
    if (a.stats && g == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, r);
    if (!a.y && !a.q) continue;
    T* yr = static_cast<T*>(a.y) + row * a.H;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      const bool in = i < n;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = in ? (v[u][j] - mean) * r : 0.0f;
      if (in && a.w) {
        float w[V];
        if constexpr (SP)
          get_param<V>(sw, n, i, w);
        else
          param<T, V>(a.w, a.w_f32, i * V, w);
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] *= w[j];
      }
      if (in && a.b) {
        float w[V];
        if constexpr (SP)
          get_param<V>(sb, n, i, w);
        else
          param<T, V>(a.b, a.b_f32, i * V, w);
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] += w[j];
      }
      if (a.y) {
        if (in) store_pack(yr + static_cast<int64_t>(i) * V, y);
      } else if constexpr (V > 1) {
        // 128 columns are the units of 128 / V neighbouring lanes, which are inside the row or
        // outside together (H is a multiple of 128)
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, fabsf(y[j]));
#pragma unroll
        for (int o = 64 / V; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (in) {
          const float scale = __fdiv_rn(fmaxf(m, 1e-30f), 448.0f);
          uint32_t w[V / 4];
#pragma unroll
          for (int j = 0; j < V; j += 4)
            w[j / 4] = static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(y[j], scale),
                                                         __fdiv_rn(y[j + 1], scale))) |
                       static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(y[j + 2], scale),
                                                         __fdiv_rn(y[j + 3], scale)))
                           << 16;
          uint8_t* q = a.q + row * a.H + static_cast<int64_t>(i) * V;
          if constexpr (V == 8)
            *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
          else
            *reinterpret_cast<uint32_t*>(q) = w[0];
          if (i % (128 / V) == 0) a.q_scale[static_cast<int64_t>(i / (128 / V)) * a.T + row] = scale;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ backward
// NV values per thread. WIDE (rows of more than 8192 columns): 32 values per thread, and the sums over
// rows, each thread's own, in shared memory since the registers do not hold them.
template <typename T, int V, int NV, bool WARP, bool WIDE>
__global__ void __launch_bounds__(WARP ? 256 : 512) k_layer_norm_back(const LnArgs a) {
  constexpr int U = NV / V;
  constexpr bool AHEAD = V == 8 && !WIDE;
  extern __shared__ float4 ln_smem[];
  float* acc = reinterpret_cast<float*>(ln_smem);  // WIDE: [2][NV][G]; WARP, at the end: [8][2][H]
  __shared__ float2 part[2][16];
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int g = WARP ? lane : static_cast<int>(threadIdx.x);
  const int n = a.H / V;
  const T *x = static_cast<const T*>(a.x), *f = static_cast<const T*>(a.f);
  const T *dh = static_cast<const T*>(a.dh), *dy = static_cast<const T*>(a.dy);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 8 : 1);
  int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  const float inv_h = 1.0f / static_cast<float>(a.H);

  constexpr int R = AHEAD ? U : 1;
  Pack<T, V> nx[R], nf[R], ny[R], nh[U];
  float2 nstat = make_float2(0.0f, 0.0f);
  const auto fetch_stat = [&](int64_t r) {
    if (r < a.T) nstat = __ldcg(reinterpret_cast<const float2*>(a.stats) + r);
  };
  const auto fetch = [&](int64_t r, int u) {
    const int i = u * G + g, b = AHEAD ? u : 0;
    if (r < a.T && i < n) {
      const int64_t at = r * a.H + static_cast<int64_t>(i) * V;
      if (dy) {
        nx[b] = load_pack<T, V>(x + at);
        if (f) nf[b] = load_pack<T, V>(f + at);
        ny[b] = load_pack<T, V>(dy + at);
      }
      if (dh) nh[u] = load_pack<T, V>(dh + at);
    }
  };
  if constexpr (AHEAD) {
    fetch_stat(row);
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(row, u);
  }

  float w[WIDE ? 1 : U][V], aw[WIDE ? 1 : U][V], ab[WIDE ? 1 : U][V];
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < 2 * NV * G; i += G) acc[i] = 0.0f;
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[u][j] = 1.0f;
        aw[u][j] = ab[u][j] = 0.0f;
      }
      if (a.w && u * G + g < n) param<T, V>(a.w, a.w_f32, (u * G + g) * V, w[u]);
    }
  }

  for (int flip = 0; row < a.T; row += step, flip ^= 1) {
    if constexpr (!AHEAD) fetch_stat(row);
    const float mean = nstat.x, r = nstat.y;
    float v[U][V], d[U][V];  // n, and dy and then u
    Pack<T, V> ph[U];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g, b = AHEAD ? u : 0;
      if constexpr (!AHEAD) fetch(row, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[u][j] = d[u][j] = 0.0f;
      if (i < n) {
        if (dy) {
          unpack(nx[b], v[u]);
          if (f) {
            float t[V];
            unpack(nf[b], t);
#pragma unroll
            for (int j = 0; j < V; ++j) v[u][j] += t[j];
          }
          unpack(ny[b], d[u]);
          float wt[V];
          if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < V; ++j) wt[j] = 1.0f;
            if (a.w) param<T, V>(a.w, a.w_f32, i * V, wt);
          }
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[u][j] = (v[u][j] - mean) * r;
            if constexpr (WIDE) {
              float* mine = acc + (u * V + j) * G + g;
              *mine = fmaf(d[u][j], v[u][j], *mine);
              mine[NV * G] += d[u][j];
              d[u][j] *= wt[j];
            } else {
              aw[u][j] = fmaf(d[u][j], v[u][j], aw[u][j]);
              ab[u][j] += d[u][j];
              d[u][j] *= w[u][j];
            }
            s1 += d[u][j];
            s2 = fmaf(d[u][j], v[u][j], s2);
          }
        }
        if (dh) ph[u] = nh[u];
      }
    }
    if constexpr (AHEAD) {
      fetch_stat(row + step);
#pragma unroll
      for (int u = 0; u < U; ++u) fetch(row + step, u);
    }
    if (!a.dx) continue;
    s1 = warp_sum_f32(s1);
    s2 = warp_sum_f32(s2);
    if (!WARP) {
      if (lane == 0) part[flip][warp] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.0f;
      for (int i = 0; i < (G >> 5); ++i) {
        const float2 p = part[flip][i];
        s1 += p.x;
        s2 += p.y;
      }
    }
    s1 *= inv_h;
    s2 *= inv_h;
    T* out = static_cast<T*>(a.dx) + row * a.H;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      if (i < n) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = r * (d[u][j] - fmaf(v[u][j], s2, s1));
        if (!dy) {  // r may be infinite
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = 0.0f;
        }
        if (dh) {
          float t[V];
          unpack(ph[u], t);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += t[j];
        }
        store_pack(out + static_cast<int64_t>(i) * V, o);
      }
    }
  }

  if (!a.want_w && !a.want_b) return;
  float* pw = a.part + static_cast<int64_t>(blockIdx.x) * a.H;
  float* pb = pw + static_cast<int64_t>(gridDim.x) * a.H;
  if constexpr (WARP) {
    float* mine = acc + warp * 2 * a.H;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * G + g;
      if (i < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          mine[i * V + j] = aw[u][j];
          mine[a.H + i * V + j] = ab[u][j];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.H; c += blockDim.x) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += acc[i * 2 * a.H + c];
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
        for (int j = 0; j < V; ++j) {
          if constexpr (WIDE) {
            pw[i * V + j] = acc[(u * V + j) * G + g];
            pb[i * V + j] = acc[(NV + u * V + j) * G + g];
          } else {
            pw[i * V + j] = aw[u][j];
            pb[i * V + j] = ab[u][j];
          }
        }
      }
    }
  }
}

// The blocks' shares of d weight (blockIdx.y 0) and d bias (1), added in a fixed order: 32 columns per
// block, eight threads per column.
template <typename T>
__global__ void __launch_bounds__(256)
    k_layer_norm_sums(const float* part, int blocks, int H, void* dw, void* db, int w_f32, int b_f32) {
  pdl_begin_in_order();
  __shared__ float buf[8][33];
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int f32 = blockIdx.y ? b_f32 : w_f32;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * blocks * H;
  float sum = 0.0f;
  if (c < H) {
    for (int b0 = threadIdx.y; b0 < blocks; b0 += 64) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = b0 + 8 * i < blocks ? __ldcg(p + static_cast<int64_t>(b0 + 8 * i) * H + c) : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
  }
  buf[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < H) {
    for (int i = 1; i < 8; ++i) sum += buf[i][threadIdx.x];
    if (f32)
      static_cast<float*>(out)[c] = sum;
    else
      from_f32(sum, static_cast<T*>(out) + c);
  }
}

// ------------------------------------------------------------------ launches
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kLnMaxSmem = 2 * 16384 * 4;  // two fp32 parameters, or the sums, of the longest row

// Threads of a block that hold a row of n units, `units` per thread.
int threads_for(int n, int units) { return ((n + units - 1) / units + 31) / 32 * 32; }

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

template <typename T, int V, bool WARP, bool SP>
cudaError_t run_forward(const LnArgs& a, int threads, int64_t blocks, cudaStream_t s) {
  static std::atomic<bool> done[64];
  const size_t smem = SP ? static_cast<size_t>(a.H) * 8 : 0;
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_smem(k_layer_norm<T, V, WARP, SP>, done);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(k_layer_norm<T, V, WARP, SP>, dim3(static_cast<unsigned>(blocks)), dim3(threads),
                    smem, s, a);
}

template <typename T, int V>
cudaError_t forward(const LayerNorm& p, int sms, cudaStream_t s) {
  if (V == 1 && p.q) return cudaErrorInvalidValue;  // the caller checks the alignment
  const LnArgs a = args_of(p);
  const int n = p.H / V;
  if (p.H <= 1024) {
    const int64_t rows = (p.T + 7) / 8, most = static_cast<int64_t>(sms) * 3;
    if (rows <= most) return run_forward<T, V, true, false>(a, 256, rows, s);
    return run_forward<T, V, true, true>(a, 256, most, s);
  }
  const int threads = threads_for(n, 32 / V);
  const int64_t most = static_cast<int64_t>(sms) * (threads <= 256 ? 3 : threads <= 320 ? 2 : 1);
  if (p.T <= most) return run_forward<T, V, false, false>(a, threads, p.T, s);
  return run_forward<T, V, false, true>(a, threads, most, s);
}

template <typename T, int V, int NV, bool WARP, bool WIDE>
cudaError_t run_backward(const LayerNorm& p, int threads, int64_t most, cudaStream_t s) {
  static std::atomic<bool> done[64];
  const LnArgs a = args_of(p);
  const size_t smem = WIDE ? static_cast<size_t>(2) * NV * threads * 4
                      : WARP ? static_cast<size_t>(8) * 2 * p.H * 4 : 0;
  if (smem > 48 * 1024) {
    const cudaError_t e = allow_smem(k_layer_norm_back<T, V, NV, WARP, WIDE>, done);
    if (e != cudaSuccess) return e;
  }
  int64_t blocks = WARP ? (p.T + 7) / 8 : p.T;
  if (blocks > most) blocks = most;
  if (blocks > kMaxLnBlocks) blocks = kMaxLnBlocks;
  cudaError_t e = launch_pdl(k_layer_norm_back<T, V, NV, WARP, WIDE>,
                             dim3(static_cast<unsigned>(blocks)), dim3(threads), smem, s, a);
  if (e != cudaSuccess || (!p.dw && !p.db)) return e;
  return launch_pdl(k_layer_norm_sums<T>, dim3((p.H + 31) / 32, 2), dim3(32, 8), 0, s,
                    static_cast<const float*>(p.part), static_cast<int>(blocks), p.H, p.dw, p.db,
                    a.w_f32, a.b_f32);
}

template <typename T, int V>
cudaError_t backward(const LayerNorm& p, int sms, cudaStream_t s) {
  const int n = p.H / V;
  if (p.H <= 512) return run_backward<T, V, 16, true, false>(p, 256, 2 * sms, s);
  if (p.H <= 8192) {
    const int threads = threads_for(n, 16 / V);
    return run_backward<T, V, 16, false, false>(p, threads, sms * (threads > 256 ? 1 : 512 / threads),
                                                s);
  }
  return run_backward<T, V, 32, false, true>(p, threads_for(n, 32 / V), sms, s);
}

template <typename T>
cudaError_t typed(const LayerNorm& p, int sms, cudaStream_t s) {
  bool wide = p.H % kV<T> == 0;
  for (const void* q : {p.f, p.x, p.w, p.b, p.dh, p.dy, static_cast<const void*>(p.h),
                        static_cast<const void*>(p.y), static_cast<const void*>(p.dx)})
    wide = wide && on16(q);
  if (p.back) return wide ? backward<T, kV<T>>(p, sms, s) : backward<T, 1>(p, sms, s);
  return wide ? forward<T, kV<T>>(p, sms, s) : forward<T, 1>(p, sms, s);
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
