// fmoe_norm.cu -- the norms before and after a block, fused with the block's gate and the residual
// scale, and their gradients.
//
// Per row (token), with f the block's output and x the residual stream:
//   n = f * r1 * wp, r1 = rsqrt(mean(f^2) + eps)     (post norm; without it n = f)
//   h = s * x + g * n                                (the new residual stream)
//   y = h * r2 * wq, r2 = rsqrt(mean(h^2) + eps)     (pre norm of the next block)
// y leaves in the input type, or as e4m3 with one fp32 scale per 128 columns in the layout of the
// fused expert layer's input (scale = max(amax, 1e-30) / 448, [H / 128, T]). h is kept in fp32
// between the two norms and rounded once, on its way out.
//
// Gradients, from da (of h), dy (of y) and the saved r1, r2: with u = dy * wq, t = da + r2 * u
// and c = r2^3 / H * sum(u * h),
//   dh = t - c * h,  dx = s * dh,  dwq = sum over rows of dy * h * r2
//   df = r1 * (g * wp * dh) - f * r1^2 / H * S1,  S1 = sum(g n dh) = sum(g n t) - c * sum(g n h)
//   dwp = sum over rows of dh * g * f * r1,  dg = dh * n (summed over what the gate broadcasts to)
// so one pass over the row collects all three sums before anything is written. r1 enters the sums,
// and the cube of r2 is multiplied up from the sum's side, because without eps r1, r2 and f are of
// opposite size: f * wp * h and r^3 alone leave fp32 for rows of 1e-13.
// All sums and statistics are fp32; the sums over rows run in a fixed order (rows of a block
// ascending, then blocks ascending).
#include <atomic>

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

struct NormGeom {
  int64_t T;
  int H, nvec;
  int gate;          // FMOE_GATE_*
  int wp_f32, wq_f32, g_f32;  // parameters held in fp32 (else in the activations' type)
  float s, eps;
};

struct NormIn {
  const void* f;     // null: no block output (pre norm of x alone)
  const void* x;
  const void* wp;    // null: no post norm
  const void* g;
  const void* wq;    // null: no pre norm
};

struct NormOut {
  void* h;           // null: not written
  void* y;
  uint8_t* q;
  float* q_scale;
  float* stats;      // [T, 2] r1, r2, or null
};

struct NormGrad {
  const void* da;    // null: zero
  const void* dy;    // null: zero
  const float* stats;
  void* df;          // nulls: not wanted
  void* dx;
  void* dg_row;      // gate per token or per element
  float* part;       // [3][blocks][H]: dwp, dwq, dg per channel
  int want_wp, want_wq, want_gc;
};

// V values of a parameter row, of the activations' type or fp32.
template <typename T, int V>
__device__ __forceinline__ void load_param(const void* p, int f32, int64_t i, float (&v)[V]) {
  if (f32) {
    const float* s = static_cast<const float*>(p) + i;
    if constexpr (V >= 4) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 w = *reinterpret_cast<const float4*>(s + j);
        v[j] = w.x;
        v[j + 1] = w.y;
        v[j + 2] = w.z;
        v[j + 3] = w.w;
      }
    } else {
      v[0] = *s;
    }
  } else {
    const T* s = static_cast<const T*>(p) + i;
    Pack<T, V> r;
    if constexpr (V > 1) {
      const uint4 w = *reinterpret_cast<const uint4*>(s);
      r.w[0] = w.x;
      r.w[1] = w.y;
      r.w[2] = w.z;
      r.w[3] = w.w;
    } else {
      r.e = *s;
    }
    unpack(r, v);
  }
}

template <typename T>
__device__ __forceinline__ float load_scalar(const void* p, int f32, int64_t i) {
  return f32 ? __ldcg(static_cast<const float*>(p) + i)
             : to_f32(load_pack<T, 1>(static_cast<const T*>(p) + i).e);
}

// The gate of V columns starting at col of row t (token gates are passed in).
template <typename T, int V>
__device__ __forceinline__ void load_gate(const NormGeom& a, const void* g, float g_tok, int64_t t,
                                          int64_t col, float (&v)[V]) {
  if (a.gate == FMOE_GATE_CHANNEL) {
    load_param<T, V>(g, a.g_f32, col, v);
  } else if (a.gate == FMOE_GATE_FULL) {
    load_param<T, V>(g, a.g_f32, t * a.H + col, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = g_tok;
  }
}

// V (4 or 8) values over their block's scale as e4m3.
template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&y)[V], float scale) {
  uint32_t w[V / 4];
#pragma unroll
  for (int j = 0; j < V; j += 4)
    w[j / 4] = static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(y[j], scale), __fdiv_rn(y[j + 1], scale))) |
               static_cast<uint32_t>(pack_e4m3x2(__fdiv_rn(y[j + 2], scale),
                                                 __fdiv_rn(y[j + 3], scale)))
                   << 16;
  if constexpr (V == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}

// Sums of N values over the block, the same in every thread. buf: [32][N], one per call site in
// turn; a barrier stands between two uses of the same one.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* buf) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_f32(v[i]);
  if (nwarp == 1) return;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[warp * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_f32(lane < nwarp ? buf[lane * N + i] : 0.0f);
}

// ------------------------------------------------------------------ direct kernels
// Rows whose tensors do not start on 16-byte boundaries (V = 1: single elements), or that are too
// long for the ring of the kernels below (V: a 16-byte group): VPT groups per thread, one row per
// block at a time, parameters read from global memory. Only V > 1 can leave as e4m3.
template <typename T, int V, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT)
    k_block_norm(const NormGeom a, const NormIn in, const NormOut out) {
  pdl_begin_in_order();
  __shared__ float buf[2][32];
  const int64_t t = blockIdx.x;
  const int64_t row = t * a.H;
  Pack<T, V> pf[VPT], px[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < a.nvec) {
      if (in.f) pf[i] = load_pack<T, V>(static_cast<const T*>(in.f) + row + v * V);
      px[i] = load_pack<T, V>(static_cast<const T*>(in.x) + row + v * V);
    }
  }
  float r1 = 1.0f;
  if (in.wp) {
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < a.nvec) {
        float f[V];
        unpack(pf[i], f);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] = fmaf(f[j], f[j], sum[0]);
      }
    }
    block_sum<1>(sum, buf[0]);
    r1 = rsqrtf(sum[0] / a.H + a.eps);
  }
  const float g_tok = a.gate == FMOE_GATE_TOKEN ? load_scalar<T>(in.g, a.g_f32, t) : 1.0f;
  float h[VPT][V];
  float sum[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < a.nvec) {
      const int64_t col = static_cast<int64_t>(v) * V;
      unpack(px[i], h[i]);
      if (in.f) {
        float f[V], g[V];
        unpack(pf[i], f);
        load_gate<T, V>(a, in.g, g_tok, t, col, g);
        if (in.wp) {
          float w[V];
          load_param<T, V>(in.wp, a.wp_f32, col, w);
#pragma unroll
          for (int j = 0; j < V; ++j) f[j] *= r1 * w[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = fmaf(g[j], f[j], a.s * h[i][j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] *= a.s;
      }
      if (out.h) store_pack<T, V>(static_cast<T*>(out.h) + row + col, h[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] = fmaf(h[i][j], h[i][j], sum[0]);
    }
  }
  if (!in.wq) {
    if (out.stats && threadIdx.x == 0) out.stats[2 * t] = r1;
    return;
  }
  block_sum<1>(sum, buf[1]);
  const float r2 = rsqrtf(sum[0] / a.H + a.eps);
  if (out.stats && threadIdx.x == 0) {
    out.stats[2 * t] = r1;
    out.stats[2 * t + 1] = r2;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    // whole warps keep going for the e4m3 maximum: 128 columns are 128 / V neighbouring lanes
    const bool live = v < a.nvec;
    const int64_t col = static_cast<int64_t>(live ? v : 0) * V;
    float w[V];
    load_param<T, V>(in.wq, a.wq_f32, col, w);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = live ? h[i][j] * r2 * w[j] : 0.0f;
    if constexpr (V > 1) {
      if (out.q) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(w[j]));
#pragma unroll
        for (int o = kBlock / V / 2; o > 0; o >>= 1)
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float scale = __fdiv_rn(fmaxf(amax, 1e-30f), 448.0f);
        if (live) {
          store_e4m3<V>(out.q + row + col, w, scale);
          if (col % kBlock == 0) out.q_scale[(col / kBlock) * a.T + t] = scale;
        }
        continue;
      }
    }
    if (live) store_pack<T, V>(static_cast<T*>(out.y) + row + col, w);
  }
}

// Rows blockIdx.x, + gridDim.x, ...: the row's gradients, and this block's share of the sums over
// rows in registers, written to part at the end.
template <typename T, int V, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT)
    k_block_norm_back(const NormGeom a, const NormIn in, const NormGrad d) {
  pdl_begin_in_order();
  __shared__ float buf[2][32 * 3];
  float awp[VPT][V], awq[VPT][V], agc[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) awp[i][j] = awq[i][j] = agc[i][j] = 0.0f;
  const bool tok = a.gate == FMOE_GATE_TOKEN;
  int flip = 0;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, flip ^= 1) {
    const int64_t row = t * a.H;
    Pack<T, V> pf[VPT], px[VPT], pa[VPT], py[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < a.nvec) {
        if (in.f) pf[i] = load_pack<T, V>(static_cast<const T*>(in.f) + row + v * V);
        px[i] = load_pack<T, V>(static_cast<const T*>(in.x) + row + v * V);
        if (d.da) pa[i] = load_pack<T, V>(static_cast<const T*>(d.da) + row + v * V);
        if (d.dy) py[i] = load_pack<T, V>(static_cast<const T*>(d.dy) + row + v * V);
      }
    }
    const float r1 = in.wp ? __ldcg(d.stats + 2 * t) : 1.0f;
    const float r2 = d.dy ? __ldcg(d.stats + 2 * t + 1) : 0.0f;
    const float g_tok = tok ? load_scalar<T>(in.g, a.g_f32, t) : 1.0f;
    // f, g, wp, h and t of a group of columns
    auto column = [&](int i, int64_t col, float (&f)[V], float (&g)[V], float (&w)[V],
                      float (&h)[V], float (&tt)[V]) {
      unpack(px[i], h);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[j] = 0.0f;
        g[j] = w[j] = 1.0f;
        tt[j] = 0.0f;
      }
      if (in.f) {
        unpack(pf[i], f);
        load_gate<T, V>(a, in.g, g_tok, t, col, g);
        if (in.wp) load_param<T, V>(in.wp, a.wp_f32, col, w);
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = fmaf(g[j], f[j] * r1 * w[j], a.s * h[j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] *= a.s;
      }
      if (d.da) unpack(pa[i], tt);
      if (d.dy) {
        float wq[V], dy[V];
        load_param<T, V>(in.wq, a.wq_f32, col, wq);
        unpack(py[i], dy);
#pragma unroll
        for (int j = 0; j < V; ++j) tt[j] = fmaf(r2 * dy[j], wq[j], tt[j]);
      }
    };
    float sum[3] = {0.0f, 0.0f, 0.0f};  // u h; (g) n t; (g) n h
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < a.nvec) {
        const int64_t col = static_cast<int64_t>(v) * V;
        float f[V], g[V], w[V], h[V], tt[V];
        column(i, col, f, g, w, h, tt);
        if (d.dy) {
          float wq[V], dy[V];
          load_param<T, V>(in.wq, a.wq_f32, col, wq);
          unpack(py[i], dy);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            sum[0] = fmaf(dy[j] * wq[j], h[j], sum[0]);
            awq[i][j] = fmaf(dy[j] * r2, h[j], awq[i][j]);
          }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float m = f[j] * r1 * (tok ? w[j] : g[j] * w[j]);
          sum[1] = fmaf(m, tt[j], sum[1]);
          sum[2] = fmaf(m, h[j], sum[2]);
        }
      }
    }
    block_sum<3>(sum, buf[flip]);
    const float c = r2 * (r2 * (r2 * (sum[0] / a.H)));
    const float gm = sum[1] - c * sum[2];
    if (tok && d.dg_row && threadIdx.x == 0) {
      if (a.g_f32)
        static_cast<float*>(d.dg_row)[t] = gm;
      else
        from_f32(gm, static_cast<T*>(d.dg_row) + t);
    }
    const float k1 = in.wp ? r1 * (r1 * ((tok ? g_tok * gm : gm) / a.H)) : 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < a.nvec) {
        const int64_t col = static_cast<int64_t>(v) * V;
        float f[V], g[V], w[V], h[V], tt[V];
        column(i, col, f, g, w, h, tt);
        float dh[V], o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dh[j] = fmaf(-c, h[j], tt[j]);
          const float n = f[j] * r1;  // without the post norm's weight
          awp[i][j] = fmaf(dh[j] * g[j], n, awp[i][j]);
          agc[i][j] = fmaf(dh[j], n * w[j], agc[i][j]);
        }
        if (d.dx) {
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = a.s * dh[j];
          store_pack<T, V>(static_cast<T*>(d.dx) + row + col, o);
        }
        if (d.df) {
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = fmaf(-k1, f[j], r1 * (g[j] * w[j]) * dh[j]);
          store_pack<T, V>(static_cast<T*>(d.df) + row + col, o);
        }
        if (a.gate == FMOE_GATE_FULL && d.dg_row) {
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = dh[j] * (f[j] * r1 * w[j]);
          if (a.g_f32) {
            float* dst = static_cast<float*>(d.dg_row) + row + col;
#pragma unroll
            for (int j = 0; j < V; ++j) dst[j] = o[j];
          } else {
            store_pack<T, V>(static_cast<T*>(d.dg_row) + row + col, o);
          }
        }
      }
    }
  }
  const int64_t plane = static_cast<int64_t>(gridDim.x) * a.H;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < a.nvec) {
      float* dst = d.part + static_cast<int64_t>(blockIdx.x) * a.H + static_cast<int64_t>(v) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (d.want_wp) dst[j] = awp[i][j];
        if (d.want_wq) dst[plane + j] = awq[i][j];
        if (d.want_gc) dst[2 * plane + j] = agc[i][j];
      }
    }
  }
}

// ------------------------------------------------------------------ ring kernels
// A group of G threads owns a row at a time; every thread copies the 16-byte granules that it will
// use itself into a ring of `stages` rows in shared memory (cp.async), so rows arrive while earlier
// ones are computed and no barrier guards the ring. A block holds gpb groups.
//
// With a row read straight into registers, each element converted and added by itself, the kernels
// were bound by their instructions (42 per element forward, 86 backward, at half the copy
// bandwidth). What depends on the column alone is therefore combined once per block: wg = wp *
// (channel gate) and wq, in fp32, in each thread's own part of shared memory; the arithmetic runs in
// packed pairs (fma.f32x2); and the sums over rows need one accumulator for wp and the channel gate
// together, since dwp = g * C and dg = wp * C with C = sum over rows of dh * f * r1 (the factor of a
// token or element gate inside).
//
// bf16 8192 x 7168 with a gate per token: forward 82 us (87% of the copy bandwidth; 112 from
// registers), gradients 149 (72%; 349), where one block of 448 threads fits an SM. 4096 x 7168 with
// a gate per channel: 44 and 69. 1024 threads per block were no faster.
//
// A row of H elements starts at a multiple of H, which for odd H is no multiple of 16 bytes. Its
// offset in its first granule, shift = (t * H) mod V, repeats every P = V / gcd(V, H) rows, so
// block b takes rows t = b mod P only: shift, and with it the columns of every thread, are the
// same for all its rows, and the sums over rows stay in registers. Elements of a neighbouring row
// in the first granule are read as zero; the last granule's copy stops at the row's end. 4096 x 4099
// takes 34 us forward and 76 backward.
constexpr int kRingThreads = 512;

struct RingGeom {
  int G;          // threads per row, a multiple of 32
  int gpb;        // rows in flight per block and stage
  int P;          // row classes
  int stages;
  int slots;      // granules of one row in the ring: G * VPT
  int row_step;   // between a group's rows
  int narr;       // row tensors in the ring
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the latest `later` groups of this thread have landed.
__device__ __forceinline__ void cp_async_wait(int later) {
  if (later >= 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (later == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Sums of N values over the G threads of a group, the same in each. buf: [N][16] of the group
// (zero beyond its warps), and another one at the next call (one barrier each). After the barrier
// every thread adds the warps' sums itself: four 16-byte reads and 15 additions are sooner done
// than five shuffles.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* buf, int group, int G) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_f32(v[i]);
  if (G == 32) return;
  const int lane = threadIdx.x & 31, w = (threadIdx.x - group * G) >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[i * 16 + w] = v[i];
  }
  named_bar_sync(1 + group, G);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 q = *reinterpret_cast<const float4*>(buf + i * 16 + 4 * j);
      sum += (q.x + q.y) + (q.z + q.w);
    }
    v[i] = sum;
  }
}

// One granule from shared memory; element j < skip (a neighbouring row's) reads as zero.
template <typename T>
__device__ __forceinline__ Gran<T> read_granule(const uint4* p, int skip) {
  Gran<T> r = gran_of<T>(*p);
  if (skip > 0) {
#pragma unroll
    for (int i = 0; i < Gran<T>::N; ++i) {
      if (2 * i < skip) r.p[i].x = 0.0f;
      if (2 * i + 1 < skip) r.p[i].y = 0.0f;
    }
  }
  return r;
}

// V columns of a parameter (of T or fp32) from global memory, zero outside the row. The columns of a
// shifted row are loaded one by one, without a branch between them, so that all loads are on their
// way together, and through L1: every block reads the same few lines, and from L2 alone they took
// 20 us at a kernel's start.
template <typename T, bool ODD>
__device__ __forceinline__ Gran<T> global_param(const void* p, int f32, int col0, int H) {
  float v[kV<T>];
  if constexpr (!ODD) {
    load_param<T, kV<T>>(p, f32, col0, v);
  } else {
    if (f32) {
#pragma unroll
      for (int j = 0; j < kV<T>; ++j)
        v[j] = static_cast<const float*>(p)[min(max(col0 + j, 0), H - 1)];
    } else {
      T e[kV<T>];
#pragma unroll
      for (int j = 0; j < kV<T>; ++j)
        e[j] = static_cast<const T*>(p)[min(max(col0 + j, 0), H - 1)];
#pragma unroll
      for (int j = 0; j < kV<T>; ++j) v[j] = to_f32(e[j]);
    }
#pragma unroll
    for (int j = 0; j < kV<T>; ++j)
      if (col0 + j < 0 || col0 + j >= H) v[j] = 0.0f;
  }
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) r.p[i] = make_float2(v[2 * i], v[2 * i + 1]);
  return r;
}

// wp * channel gate of V columns, ones where there is neither (zero outside the row, so that what
// a thread computes there is zero too).
template <typename T, bool ODD>
__device__ __forceinline__ Gran<T> branch_weight(const NormGeom& a, const NormIn& in, int col0) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; ++i) {
    const int c = col0 + 2 * i;
    r.p[i] = make_float2(c >= 0 && c < a.H ? 1.0f : 0.0f, c >= -1 && c + 1 < a.H ? 1.0f : 0.0f);
  }
  if (in.wp) r = global_param<T, ODD>(in.wp, a.wp_f32, col0, a.H);
  if (a.gate == FMOE_GATE_CHANNEL) r = mul(r, global_param<T, ODD>(in.g, a.g_f32, col0, a.H));
  return r;
}

// A granule of fp32 values in a thread's own part of shared memory: 16-byte pieces `stride` threads
// apart, so neighbouring threads' pieces are neighbours.
template <typename T>
__device__ __forceinline__ void put_own(float4* p, int stride, const Gran<T>& v) {
#pragma unroll
  for (int i = 0; i < Gran<T>::N; i += 2)
    p[(i / 2) * stride] = make_float4(v.p[i].x, v.p[i].y, v.p[i + 1].x, v.p[i + 1].y);
}
template <typename T>
__device__ __forceinline__ Gran<T> get_own(const float4* p, int stride) {
  Gran<T> r;
#pragma unroll
  for (int i = 0; i < Gran<T>::N; i += 2) {
    const float4 q = p[(i / 2) * stride];
    r.p[i] = make_float2(q.x, q.y);
    r.p[i + 1] = make_float2(q.z, q.w);
  }
  return r;
}

// V columns from column col0 on, whose place is p; columns outside the row stay.
template <typename T, bool ODD>
__device__ __forceinline__ void store_granule(T* p, int col0, int H, const Gran<T>& g) {
  constexpr int S = sizeof(T);
  const uint4 w = words_of(g);
  if constexpr (ODD)
    store_part<S>(reinterpret_cast<uint8_t*>(p), w, -col0 * S, (H - col0) * S);
  else
    *reinterpret_cast<uint4*>(p) = w;
}

// Where a thread stands: its group, its columns (granule i starts at col0 + i * step, of which the
// first `live` lie in the row) and its rows (t, then every row_step).
template <typename T, int VPT, bool ODD>
struct RowWalk {
  int group, g, shift, col0, step, live;
  int64_t t;
  __device__ RowWalk(const NormGeom& a, const RingGeom& r) {
    constexpr int V = kV<T>;
    group = threadIdx.x / r.G;
    g = threadIdx.x - group * r.G;
    const int cls = ODD ? blockIdx.x % r.P : 0;
    shift = ODD ? static_cast<int>((static_cast<int64_t>(cls) * a.H) % V) : 0;
    col0 = g * V - shift;
    step = r.G * V;
    live = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) live += col0 + i * step < a.H ? 1 : 0;
    t = cls + static_cast<int64_t>(r.P) * ((blockIdx.x / r.P) * r.gpb + group);
  }
  // elements of a neighbouring row at the start of granule i
  __device__ int skip(int i) const { return ODD && i == 0 && col0 < 0 ? shift : 0; }
};

// Copies the thread's granules of one tensor's row into its ring slots; off: the row's first
// element plus col0.
template <typename T, int VPT, bool ODD>
__device__ __forceinline__ void fetch_row(uint32_t dst, const void* src, int64_t off, int H,
                                          const RowWalk<T, VPT, ODD>& w, int G) {
  const T* p = static_cast<const T*>(src) + off;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i < w.live) {
      const int left = H - w.col0 - i * w.step;  // elements from the granule's start to the row's end
      cp_async16(dst + i * G * 16, p + i * w.step,
                 ODD && left < kV<T> ? left * static_cast<int>(sizeof(T)) : 16);
    }
  }
}

// COMMON: a block output, no gate per element, and both results wanted (forward) or both gradients
// given (backward); what is not common is decided at run time.
template <typename T, int VPT, bool ODD, bool COMMON>
__global__ void __launch_bounds__(kRingThreads, 2)
    k_norm_ring(const NormGeom a, const RingGeom r, const NormIn in, const NormOut out) {
  constexpr int V = kV<T>;
  extern __shared__ uint4 ring[];   // [stages][gpb][narr][slots], then wg and wq per thread
  __shared__ float4 sums[4][kRingThreads / 64][4];  // [row parity and call site][group]
  const RowWalk<T, VPT, ODD> w(a, r);
  const int H = a.H, G = r.G;
  const bool has_f = COMMON || in.f != nullptr, has_wq = COMMON || in.wq != nullptr;
  const bool has_h = COMMON || out.h != nullptr, full = !COMMON && a.gate == FMOE_GATE_FULL;
  float4* own = reinterpret_cast<float4*>(ring + static_cast<size_t>(r.stages) * r.gpb * r.narr * r.slots) +
                threadIdx.x;
  const int own_step = blockDim.x * (V / 4);
  for (int i = threadIdx.x; i < static_cast<int>(sizeof(sums) / 16); i += blockDim.x)
    (&sums[0][0][0])[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncthreads();
  // ring order: x, f, gate
  const int arr = r.slots, stage = r.gpb * r.narr * arr;
  const uint4* mine = ring + w.group * r.narr * arr + w.g;
  const uint32_t mine32 = smem_u32(mine);
  auto fetch = [&](int s, int64_t t, int64_t off) {
    if (t < a.T) {
      const uint32_t d = mine32 + s * stage * 16;
      fetch_row<T, VPT, ODD>(d, in.x, off, H, w, G);
      if (has_f) fetch_row<T, VPT, ODD>(d + arr * 16, in.f, off, H, w, G);
      if (full) fetch_row<T, VPT, ODD>(d + 2 * arr * 16, in.g, off, H, w, G);
    }
    cp_async_commit();
  };
  pdl_begin_in_order();
  const int64_t off_step = static_cast<int64_t>(r.row_step) * H;
  int64_t ahead = w.t, off = w.t * H + w.col0, off_ahead = off;
  for (int s = 0; s < r.stages; ++s, ahead += r.row_step, off_ahead += off_step)
    fetch(s, ahead, off_ahead);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i < w.live) {
      const int col = w.col0 + i * w.step;
      if (has_f) put_own(own + i * own_step, blockDim.x, branch_weight<T, ODD>(a, in, col));
      if (has_wq)
        put_own(own + (VPT + i) * own_step, blockDim.x,
                global_param<T, ODD>(in.wq, a.wq_f32, col, H));
    }
  }
  const float inv_h = 1.0f / H;
  const int gr = G == 32 ? 0 : w.group;
  const bool tok = a.gate == FMOE_GATE_TOKEN;
  // a token's gate is loaded a row ahead
  float g_next = tok && w.t < a.T ? load_scalar<T>(in.g, a.g_f32, w.t) : 1.0f;
  int s = 0, flip = 0;
  for (int64_t t = w.t; t < a.T; t += r.row_step, off += off_step, flip ^= 2) {
    const float g_tok = g_next;
    if (tok && t + r.row_step < a.T) g_next = load_scalar<T>(in.g, a.g_f32, t + r.row_step);
    cp_async_wait(r.stages - 1);
    const uint4* row = mine + s * stage;
    Gran<T> h[VPT];
    float r1 = 1.0f;
    if (has_f) {
      float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        zero(h[i]);
        if (i < w.live) h[i] = read_granule<T>(row + arr + i * G, w.skip(i));
        dot(sq, h[i], h[i]);
      }
      if (in.wp) {
        float sum[1] = {sq.x + sq.y};
        group_sum<1>(sum, &sums[flip][gr][0].x, w.group, G);
        r1 = rsqrtf(fmaf(sum[0], inv_h, a.eps));
      }
    }
    const float rg = r1 * g_tok;
    float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (i < w.live) {
        const Gran<T> x = mul(read_granule<T>(row + i * G, w.skip(i)), a.s);
        if (has_f) {
          h[i] = mul(h[i], rg);
          if (full) h[i] = mul(h[i], read_granule<T>(row + 2 * arr + i * G, w.skip(i)));
          h[i] = fma(h[i], get_own<T>(own + i * own_step, blockDim.x), x);
        } else {
          h[i] = x;
        }
        if (has_h)
          store_granule<T, ODD>(static_cast<T*>(out.h) + off + i * w.step, w.col0 + i * w.step, H,
                                h[i]);
        dot(sq, h[i], h[i]);
      }
    }
    fetch(s, ahead, off_ahead);  // the row's tensors are in registers now
    ahead += r.row_step;
    off_ahead += off_step;
    s = s + 1 == r.stages ? 0 : s + 1;
    if (!has_wq) {
      if (out.stats && w.g == 0) out.stats[2 * t] = r1;
      continue;
    }
    float sum[1] = {sq.x + sq.y};
    group_sum<1>(sum, &sums[flip + 1][gr][0].x, w.group, G);
    const float r2 = rsqrtf(fmaf(sum[0], inv_h, a.eps));
    if (out.stats && w.g == 0) {
      out.stats[2 * t] = r1;
      out.stats[2 * t + 1] = r2;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      // whole warps keep going for the e4m3 maximum: 128 columns are 128 / V neighbouring lanes
      const bool live = i < w.live;
      const int col = w.col0 + i * w.step;
      if (live) h[i] = mul(mul(h[i], r2), get_own<T>(own + (VPT + i) * own_step, blockDim.x));
      if constexpr (!ODD) {
        if (out.q) {
          float y[V];
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            y[2 * j] = live ? h[i].p[j].x : 0.0f;
            y[2 * j + 1] = live ? h[i].p[j].y : 0.0f;
          }
          float amax = 0.0f;
#pragma unroll
          for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(y[j]));
#pragma unroll
          for (int o = kBlock / V / 2; o > 0; o >>= 1)
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float scale = __fdiv_rn(fmaxf(amax, 1e-30f), 448.0f);
          if (live) {
            store_e4m3<V>(out.q + off + i * w.step, y, scale);
            if (col % kBlock == 0) out.q_scale[static_cast<int64_t>(col / kBlock) * a.T + t] = scale;
          }
          continue;
        }
      }
      if (live)
        store_granule<T, ODD>(static_cast<T*>(out.y) + off + i * w.step, col, H, h[i]);
    }
  }
  cp_async_wait(0);
}

// The gradients of a group's rows; this block's share of the sums over rows stays in registers and
// goes to part at the end, the groups added in order.
template <typename T, int VPT, bool ODD, bool COMMON>
__global__ void __launch_bounds__(kRingThreads, 1)
    k_norm_back_ring(const NormGeom a, const RingGeom r, const NormIn in, const NormGrad d) {
  constexpr int V = kV<T>;
  extern __shared__ uint4 ring[];   // [stages][gpb][narr][slots], then wg and wq per thread
  __shared__ float4 sums[2][kRingThreads / 64][3 * 4];  // [row parity][group][sum]
  const RowWalk<T, VPT, ODD> w(a, r);
  const int H = a.H, G = r.G;
  const bool has_f = COMMON || in.f != nullptr;
  const bool has_da = COMMON || d.da != nullptr, has_dy = COMMON || d.dy != nullptr;
  const bool tok = a.gate == FMOE_GATE_TOKEN, full = !COMMON && a.gate == FMOE_GATE_FULL;
  // piece p of granule i of parameter q of this thread: own[((q * VPT + i) * (V / 4) + p) * blockDim]
  float4* own = reinterpret_cast<float4*>(ring + static_cast<size_t>(r.stages) * r.gpb * r.narr * r.slots) +
                threadIdx.x;
  const int own_step = blockDim.x * (V / 4);
  for (int i = threadIdx.x; i < static_cast<int>(sizeof(sums) / 16); i += blockDim.x)
    (&sums[0][0][0])[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncthreads();
  const int gr = G == 32 ? 0 : w.group;
  // ring order: x, f, da, dy, gate, without those that are not there
  const int arr = r.slots, stage = r.gpb * r.narr * arr;
  const int fa = arr, da = fa + (has_f ? arr : 0), ya = da + (has_da ? arr : 0);
  const int ga = ya + (has_dy ? arr : 0);
  const uint4* mine = ring + w.group * r.narr * arr + w.g;
  const uint32_t mine32 = smem_u32(mine);
  // a row in two parts: what the first pass over it reads alone, and what both read
  auto fetch_first = [&](int s, int64_t t, int64_t off) {
    if (t < a.T) {
      const uint32_t p = mine32 + s * stage * 16;
      fetch_row<T, VPT, ODD>(p, in.x, off, H, w, G);
      if (has_da) fetch_row<T, VPT, ODD>(p + da * 16, d.da, off, H, w, G);
      if (has_dy) fetch_row<T, VPT, ODD>(p + ya * 16, d.dy, off, H, w, G);
    }
  };
  auto fetch_rest = [&](int s, int64_t t, int64_t off) {
    if (t < a.T) {
      const uint32_t p = mine32 + s * stage * 16;
      if (has_f) fetch_row<T, VPT, ODD>(p + fa * 16, in.f, off, H, w, G);
      if (full) fetch_row<T, VPT, ODD>(p + ga * 16, in.g, off, H, w, G);
    }
    cp_async_commit();
  };
  pdl_begin_in_order();
  const int64_t off_step = static_cast<int64_t>(r.row_step) * H;
  int64_t ahead = w.t, off = w.t * H + w.col0, off_ahead = off;
  for (int s = 0; s < r.stages; ++s, ahead += r.row_step, off_ahead += off_step) {
    fetch_first(s, ahead, off_ahead);
    fetch_rest(s, ahead, off_ahead);
  }
  Gran<T> C[VPT], Q[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    zero(C[i]);
    zero(Q[i]);
    if (i < w.live) {
      const int col = w.col0 + i * w.step;
      if (has_f) put_own(own + i * own_step, blockDim.x, branch_weight<T, ODD>(a, in, col));
      if (has_dy)
        put_own(own + (VPT + i) * own_step, blockDim.x,
                global_param<T, ODD>(in.wq, a.wq_f32, col, H));
    }
  }
  const float inv_h = 1.0f / H;
  // a row's statistics and token gate are loaded a row ahead
  float r1_next = 1.0f, r2_next = 0.0f, g_next = 1.0f;
  auto scalars = [&](int64_t t) {
    if (t >= a.T) return;
    if (in.wp) r1_next = __ldcg(d.stats + 2 * t);
    if (has_dy) r2_next = __ldcg(d.stats + 2 * t + 1);
    if (tok) g_next = load_scalar<T>(in.g, a.g_f32, t);
  };
  scalars(w.t);
  int s = 0, flip = 0;
  for (int64_t t = w.t; t < a.T; t += r.row_step, off += off_step, flip ^= 1) {
    const float r1 = r1_next, r2 = r2_next, g_tok = g_next, rg = r1 * g_tok;
    scalars(t + r.row_step);
    cp_async_wait(r.stages - 1);
    const uint4* row = mine + s * stage;
    Gran<T> h[VPT], tt[VPT];
    float2 s0 = make_float2(0.0f, 0.0f), s1 = s0, s2 = s0;  // u h; n t; n h (a token's gate apart)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (i < w.live) {
        h[i] = mul(read_granule<T>(row + i * G, w.skip(i)), a.s);
        Gran<T> m;
        zero(m);
        if (has_f) {
          m = mul(mul(read_granule<T>(row + fa + i * G, w.skip(i)), r1),
                  get_own<T>(own + i * own_step, blockDim.x));
          if (full) m = mul(m, read_granule<T>(row + ga + i * G, w.skip(i)));
          h[i] = fma(m, g_tok, h[i]);
        }
        zero(tt[i]);
        if (has_da) tt[i] = read_granule<T>(row + da + i * G, w.skip(i));
        if (has_dy) {
          const Gran<T> dy = read_granule<T>(row + ya + i * G, w.skip(i));
          const Gran<T> b = get_own<T>(own + (VPT + i) * own_step, blockDim.x);
          const Gran<T> p = mul(dy, h[i]);
          dot(s0, p, b);
          Q[i] = fma(p, r2, Q[i]);
          tt[i] = fma(mul(dy, b), r2, tt[i]);
        }
        dot(s1, m, tt[i]);
        dot(s2, m, h[i]);
      }
    }
    fetch_first(s, ahead, off_ahead);  // x, da and dy are in registers now, as h and t
    float sum[3] = {s0.x + s0.y, s1.x + s1.y, s2.x + s2.y};
    group_sum<3>(sum, &sums[flip][gr][0].x, w.group, G);
    const float c = r2 * (r2 * (r2 * (sum[0] * inv_h)));
    const float gm = sum[1] - c * sum[2];
    if (tok && d.dg_row && w.g == 0) {
      if (a.g_f32)
        static_cast<float*>(d.dg_row)[t] = gm;
      else
        from_f32(gm, static_cast<T*>(d.dg_row) + t);
    }
    const float k1 = in.wp ? r1 * (r1 * (g_tok * gm * inv_h)) : 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (i < w.live) {
        const int col = w.col0 + i * w.step;
        const int64_t at = off + i * w.step;
        const Gran<T> dh = fma(h[i], -c, tt[i]);
        if (d.dx)
          store_granule<T, ODD>(static_cast<T*>(d.dx) + at, col, H,
                                a.s == 1.0f ? dh : mul(dh, a.s));
        if (has_f) {
          const Gran<T> f = read_granule<T>(row + fa + i * G, w.skip(i));
          const Gran<T> wg = get_own<T>(own + i * own_step, blockDim.x);
          Gran<T> gd = mul(dh, rg);     // r1 * gate * dh, without a channel gate
          if (full) {
            if (d.dg_row)
              store_granule<T, ODD>(static_cast<T*>(d.dg_row) + at, col, H,
                                    mul(mul(f, wg), mul(dh, r1)));
            gd = mul(gd, read_granule<T>(row + ga + i * G, w.skip(i)));
          }
          C[i] = fma(gd, f, C[i]);
          if (d.df)
            store_granule<T, ODD>(static_cast<T*>(d.df) + at, col, H, fma(f, -k1, mul(gd, wg)));
        }
      }
    }
    fetch_rest(s, ahead, off_ahead);
    ahead += r.row_step;
    off_ahead += off_step;
    s = s + 1 == r.stages ? 0 : s + 1;
  }
  cp_async_wait(0);
  // the ring is free: the groups' sums meet there, and are added in order
  const int64_t plane = static_cast<int64_t>(gridDim.x) * H;
  float* acc = reinterpret_cast<float*>(ring);  // [gpb][slots * V]
  for (int which = 0; which < 2; ++which) {
    if (!(which == 0 ? d.want_wp || d.want_gc : d.want_wq)) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float4* dst = reinterpret_cast<float4*>(acc) + (w.group * arr + w.g + i * G) * (V / 4);
#pragma unroll
      for (int j = 0; j < V / 2; j += 2) {
        const float2 x = which == 0 ? C[i].p[j] : Q[i].p[j];
        const float2 y = which == 0 ? C[i].p[j + 1] : Q[i].p[j + 1];
        dst[j / 2] = make_float4(x.x, x.y, y.x, y.y);
      }
    }
    __syncthreads();
    float* dst = d.part + which * plane + static_cast<int64_t>(blockIdx.x) * H;
    for (int c = threadIdx.x; c < H; c += blockDim.x) {
      float x = acc[c + w.shift];
      for (int grp = 1; grp < r.gpb; ++grp) x += acc[grp * arr * V + c + w.shift];
      dst[c] = x;
    }
  }
}

// Sums over the blocks' shares, eight interleaved runs of blocks added in order. Plane 0 holds the
// sums behind the post norm's weight and a channel gate: C of the ring kernels (dwp = g * C, dg =
// wp * C), plane 1 dwq. The direct kernels store dwp, dwq and dg as they are, in three planes.
struct ColumnSums {
  void* out[3];          // dwp, dwq, dg
  int f32[3];
  const void* factor[3]; // what the plane is multiplied with, or null
  int factor_f32[3];
  int plane[3];
};

template <typename T>
__global__ void __launch_bounds__(256)
    k_column_sums(const float* part, int blocks, int H, const ColumnSums o) {
  pdl_begin_in_order();
  __shared__ float buf[8][33];
  const int which = blockIdx.y;
  if (!o.out[which]) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* p = part + static_cast<int64_t>(o.plane[which]) * blocks * H;
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
    if (o.factor[which]) sum *= load_scalar<T>(o.factor[which], o.factor_f32[which], c);
    if (o.f32[which])
      static_cast<float*>(o.out[which])[c] = sum;
    else
      from_f32(sum, static_cast<T*>(o.out[which]) + c);
  }
}

bool aligned16_or_null(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

NormGeom geom(const BlockNorm& p, int V) {
  NormGeom a{};
  a.T = p.T;
  a.H = p.H;
  a.nvec = p.H / V;
  a.gate = p.gate;
  a.wp_f32 = p.wp_dtype == FMOE_DTYPE_F32;
  a.wq_f32 = p.wq_dtype == FMOE_DTYPE_F32;
  a.g_f32 = p.g_dtype == FMOE_DTYPE_F32;
  a.s = p.s;
  a.eps = p.eps;
  return a;
}

int back_blocks(const BlockNorm& p, int sms) {
  const int b = sms < kMaxNormBlocks ? sms : kMaxNormBlocks;
  return static_cast<int>(p.T < b ? p.T : b);
}

NormGrad grads(const BlockNorm& p) {
  NormGrad d{};
  d.da = p.da;
  d.dy = p.dy;
  d.stats = p.stats;
  d.df = p.df;
  d.dx = p.dx;
  const bool channel = p.gate == FMOE_GATE_CHANNEL;
  d.dg_row = channel ? nullptr : p.dg;
  d.part = p.part;
  d.want_wp = p.dwp != nullptr;
  d.want_wq = p.dwq != nullptr;
  d.want_gc = channel && p.dg != nullptr;
  return d;
}

// The sums over the blocks' shares, if any are wanted.
template <typename T>
cudaError_t column_sums(const BlockNorm& p, const NormGeom& a, const NormGrad& d, int blocks,
                        bool ring, cudaStream_t s) {
  if (!(d.want_wp || d.want_wq || d.want_gc)) return cudaSuccess;
  ColumnSums o{};
  o.out[0] = p.dwp;
  o.out[1] = p.dwq;
  o.out[2] = d.want_gc ? p.dg : nullptr;
  o.f32[0] = a.wp_f32;
  o.f32[1] = a.wq_f32;
  o.f32[2] = a.g_f32;
  o.plane[1] = 1;
  o.plane[2] = ring ? 0 : 2;
  if (ring && p.gate == FMOE_GATE_CHANNEL) {
    o.factor[0] = p.g;
    o.factor_f32[0] = a.g_f32;
    o.factor[2] = p.wp;
    o.factor_f32[2] = a.wp_f32;
  }
  return launch_pdl(k_column_sums<T>, dim3((p.H + 31) / 32, 3), dim3(32, 8), 0, s,
                    static_cast<const float*>(p.part), blocks, p.H, o);
}

template <typename T, int V, int VPT, int MAXT>
cudaError_t norm_direct(const BlockNorm& p, int sms, cudaStream_t s) {
  if (V == 1 && p.q) return cudaErrorInvalidValue;  // the caller checks the alignment
  const NormGeom a = geom(p, V);
  const NormIn in{p.f, p.x, p.wp, p.g, p.wq};
  int threads = (a.nvec + VPT - 1) / VPT;
  threads = (threads + 31) / 32 * 32;
  if (!p.back) {
    const NormOut out{p.h, p.y, static_cast<uint8_t*>(p.q), p.q_scale, p.stats};
    return launch_pdl(k_block_norm<T, V, VPT, MAXT>, dim3(static_cast<unsigned>(p.T)),
                      dim3(threads), 0, s, a, in, out);
  }
  const NormGrad d = grads(p);
  const int blocks = back_blocks(p, sms);
  const cudaError_t e = launch_pdl(k_block_norm_back<T, V, VPT, MAXT>, dim3(blocks), dim3(threads),
                                   0, s, a, in, d);
  return e != cudaSuccess ? e : column_sums<T>(p, a, d, blocks, false, s);
}

// Dynamic shared memory of a block: two blocks per SM in the forward pass, whose barriers each
// other's work hides, and one in the backward pass, which holds its sums over rows in registers.
// Static shared memory (sums) comes on top.
constexpr int kNormSmem = 212 * 1024;

// The ring's shape for rows of ng granules, or stages = 0 if not even one stage fits.
template <typename T>
RingGeom ring_geom(const BlockNorm& p, int vpt, int ng, int cps, size_t* smem) {
  RingGeom r{};
  r.G = ((ng + vpt - 1) / vpt + 31) / 32 * 32;
  r.gpb = kRingThreads / r.G;  // at most 8 where groups need their named barriers (1 .. 8)
  r.slots = r.G * vpt;
  r.narr = 1 + (p.f ? 1 : 0) + (p.gate == FMOE_GATE_FULL ? 1 : 0) + (p.back && p.da ? 1 : 0) +
           (p.back && p.dy ? 1 : 0);
  // fewer rows at a time where the ring would not fit beside two parameters per thread; the
  // backward pass has, at its end, the fp32 sums of a row where the ring was
  for (; r.gpb >= 1; --r.gpb) {
    const size_t row = static_cast<size_t>(r.slots) * kV<T> * 4;
    const size_t stage = static_cast<size_t>(r.gpb) * r.narr * r.slots * 16;
    for (r.stages = 3; r.stages >= 1; --r.stages) {
      size_t bytes = r.stages * stage;
      if (p.back && bytes < r.gpb * row) bytes = r.gpb * row;
      bytes += 2 * r.gpb * row;
      if (bytes <= static_cast<size_t>(kNormSmem / cps)) {
        *smem = bytes;
        return r;
      }
    }
  }
  r.stages = 0;
  return r;
}

template <typename T, int VPT, bool ODD, bool COMMON>
cudaError_t norm_ring(const BlockNorm& p, RingGeom r, size_t smem, int cps, int sms,
                      cudaStream_t s) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(k_norm_ring<T, VPT, ODD, COMMON>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k_norm_back_ring<T, VPT, ODD, COMMON>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmem);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  const NormGeom a = geom(p, kV<T>);
  const NormIn in{p.f, p.x, p.wp, p.g, p.wq};
  r.P = 1;
  if (ODD)
    for (r.P = 2; (r.P * p.H) % kV<T> != 0;) r.P *= 2;
  int limit = cps * sms;
  if (p.back && limit > kMaxNormBlocks) limit = kMaxNormBlocks;
  limit = limit / r.P * r.P;
  r.row_step = limit * r.gpb;
  // block b's first row is b % P + P * gpb * (b / P), increasing in b: those that have one
  const int64_t per = static_cast<int64_t>(r.P) * r.gpb;
  int64_t blocks = p.T / per * r.P + (p.T % per < r.P ? p.T % per : r.P);
  if (blocks > limit) blocks = limit;
  const dim3 grid(static_cast<unsigned>(blocks)), block(r.G * r.gpb);
  if (!p.back) {
    const NormOut out{p.h, p.y, static_cast<uint8_t*>(p.q), p.q_scale, p.stats};
    return launch_pdl(k_norm_ring<T, VPT, ODD, COMMON>, grid, block, smem, s, a, r, in, out);
  }
  const NormGrad d = grads(p);
  const cudaError_t e =
      launch_pdl(k_norm_back_ring<T, VPT, ODD, COMMON>, grid, block, smem, s, a, r, in, d);
  return e != cudaSuccess ? e : column_sums<T>(p, a, d, static_cast<int>(blocks), true, s);
}

template <typename T>
cudaError_t norm_typed(const BlockNorm& p, int sms, cudaStream_t s) {
  constexpr int V = kV<T>;
  const bool odd = p.H % V != 0;
  bool rows16 = true, params16 = true;  // on 16-byte boundaries
  for (const void* q : {p.f, p.x, p.da, p.dy, static_cast<const void*>(p.h),
                        static_cast<const void*>(p.y), static_cast<const void*>(p.df),
                        static_cast<const void*>(p.dx)})
    rows16 = rows16 && aligned16_or_null(q);
  if (p.gate == FMOE_GATE_FULL) rows16 = rows16 && aligned16_or_null(p.g) && aligned16_or_null(p.dg);
  for (const void* q : {p.wp, p.wq, p.g}) params16 = params16 && aligned16_or_null(q);
  // parameters are staged in 16-byte pieces unless the rows are shifted
  const bool ring = rows16 && (odd || params16) &&
                    (p.gate != FMOE_GATE_FULL || p.g_dtype == p.dtype);
  if (ring) {
    // granules of a row at the largest shift
    const int ng = (p.H + V - 1) / V + (odd ? 1 : 0);
    if (ng <= 2048) {
      const int vpt = ng <= 32 ? 1 : ng <= 2 * kRingThreads ? 2 : 4;
      size_t smem = 0;
      int cps = p.back ? 1 : 2;
      RingGeom r = ring_geom<T>(p, vpt, ng, cps, &smem);
      if (r.stages == 0 && cps == 2) r = ring_geom<T>(p, vpt, ng, cps = 1, &smem);
      if (r.stages > 0) {
        // rows of more than 8192 16-bit columns do not have a variant of their own for the common case
        const bool common = vpt < 4 && p.f && p.gate != FMOE_GATE_FULL &&
                            (p.back ? p.da && p.dy : p.h && p.wq);
#define RUN(VPT, COMMON)                                                  \
  (odd ? norm_ring<T, VPT, true, COMMON>(p, r, smem, cps, sms, s)         \
       : norm_ring<T, VPT, false, COMMON>(p, r, smem, cps, sms, s))
        if (common) return vpt == 1 ? RUN(1, true) : RUN(2, true);
        return vpt == 1 ? RUN(1, false) : vpt == 2 ? RUN(2, false) : RUN(4, false);
#undef RUN
      }
    }
  }
  // 16384 columns are 2048 (16-bit) or 4096 (fp32) groups
  if (rows16 && params16 && !odd) return norm_direct<T, V, 4, sizeof(T) == 2 ? 512 : 1024>(p, sms, s);
  if (p.H <= 512) return norm_direct<T, 1, 1, 512>(p, sms, s);
  if (p.H <= 2048) return norm_direct<T, 1, 4, 512>(p, sms, s);
  return norm_direct<T, 1, 16, 1024>(p, sms, s);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNorm& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return norm_typed<float>(p, sms, s);
    case FMOE_DTYPE_BF16:
      return norm_typed<__nv_bfloat16>(p, sms, s);
    default:
      return norm_typed<__half>(p, sms, s);
  }
}

}  // namespace fmoe
