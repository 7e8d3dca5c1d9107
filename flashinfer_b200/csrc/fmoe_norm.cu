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
// Gradients, from da (of h), dy (of y) and the saved r1, r2: with u = dy * wq, t = da + r2 * u,
// m = f * wp (or f) and c = r2^3 / H * sum(u * h),
//   dh = t - c * h,  dx = s * dh,  dwq = sum over rows of dy * h * r2
//   df = r1 * (g * wp * dh) - f * r1^3 / H * S1,  S1 = sum(g * m * dh) = sum(g m t) - c * sum(g m h)
//   dwp = sum over rows of dh * g * f * r1,  dg = dh * n (summed over what the gate broadcasts to)
// so one pass over the row collects all three sums before anything is written.
// All sums and statistics are fp32; the sums over rows run in a fixed order (rows of a block
// ascending, then blocks ascending).
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
    const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(p) + i);
    unpack(r, v);
  }
}

template <typename T>
__device__ __forceinline__ float load_scalar(const void* p, int f32, int64_t i) {
  return f32 ? __ldcg(static_cast<const float*>(p) + i)
             : to_f32(load_pack<T, 1>(static_cast<const T*>(p) + i).e[0]);
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

// One row per block; a thread holds VPT groups of V columns.
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
          uint16_t b[V / 2];
#pragma unroll
          for (int j = 0; j < V; j += 2)
            b[j / 2] = pack_e4m3x2(__fdiv_rn(w[j], scale), __fdiv_rn(w[j + 1], scale));
          memcpy(out.q + row + col, b, V);
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
    float sum[3] = {0.0f, 0.0f, 0.0f};  // u h; (g) m t; (g) m h
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
          const float m = tok ? f[j] * w[j] : g[j] * f[j] * w[j];
          sum[1] = fmaf(m, tt[j], sum[1]);
          sum[2] = fmaf(m, h[j], sum[2]);
        }
      }
    }
    block_sum<3>(sum, buf[flip]);
    const float c = r2 * r2 * r2 * (sum[0] / a.H);
    const float gm = sum[1] - c * sum[2];
    if (tok && d.dg_row && threadIdx.x == 0) {
      if (a.g_f32)
        static_cast<float*>(d.dg_row)[t] = r1 * gm;
      else
        from_f32(r1 * gm, static_cast<T*>(d.dg_row) + t);
    }
    const float k1 = in.wp ? r1 * r1 * r1 * ((tok ? g_tok * gm : gm) / a.H) : 0.0f;
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

// out[c] = sum over blocks of part[b][c], eight interleaved runs of blocks added in order.
struct ColumnSums {
  void* out[3];
  int f32[3];
};

template <typename T>
__global__ void __launch_bounds__(256)
    k_column_sums(const float* part, int blocks, int H, const ColumnSums o) {
  pdl_begin_in_order();
  __shared__ float buf[8][33];
  const int which = blockIdx.y;
  if (!o.out[which]) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* p = part + static_cast<int64_t>(which) * blocks * H;
  float sum = 0.0f;
  if (c < H) {
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += 8) sum += __ldcg(p + static_cast<int64_t>(b) * H + c);
  }
  buf[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < H) {
    for (int i = 1; i < 8; ++i) sum += buf[i][threadIdx.x];
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
  int b = 2 * sms < kMaxNormBlocks ? 2 * sms : kMaxNormBlocks;
  return static_cast<int>(p.T < b ? p.T : b);
}

template <typename T, int V, int VPT, int MAXT>
cudaError_t norm_one(const BlockNorm& p, int sms, cudaStream_t s) {
  const NormGeom a = geom(p, V);
  const NormIn in{p.f, p.x, p.wp, p.g, p.wq};
  int threads = (a.nvec + VPT - 1) / VPT;
  threads = (threads + 31) / 32 * 32;
  if (!p.back) {
    const NormOut out{p.h, p.y, static_cast<uint8_t*>(p.q), p.q_scale, p.stats};
    return launch_pdl(k_block_norm<T, V, VPT, MAXT>, dim3(static_cast<unsigned>(p.T)),
                      dim3(threads), 0, s, a, in, out);
  }
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
  const int blocks = back_blocks(p, sms);
  cudaError_t e = launch_pdl(k_block_norm_back<T, V, VPT, MAXT>, dim3(blocks), dim3(threads), 0, s,
                             a, in, d);
  if (e != cudaSuccess || !(d.want_wp || d.want_wq || d.want_gc)) return e;
  ColumnSums o{};
  o.out[0] = p.dwp;
  o.out[1] = p.dwq;
  o.out[2] = d.want_gc ? p.dg : nullptr;
  o.f32[0] = a.wp_f32;
  o.f32[1] = a.wq_f32;
  o.f32[2] = a.g_f32;
  return launch_pdl(k_column_sums<T>, dim3((p.H + 31) / 32, 3), dim3(32, 8), 0, s,
                    static_cast<const float*>(p.part), blocks, p.H, o);
}

template <typename T>
cudaError_t norm_typed(const BlockNorm& p, int sms, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  bool vec = p.H % V == 0;
  for (const void* q : {p.f, p.x, p.wp, p.g, p.wq, p.da, p.dy, static_cast<const void*>(p.h),
                        static_cast<const void*>(p.y), static_cast<const void*>(p.df),
                        static_cast<const void*>(p.dx), static_cast<const void*>(p.dg)})
    vec = vec && aligned16_or_null(q);
  if (vec) {
    const int nvec = p.H / V;
    if (nvec <= 512) return norm_one<T, V, 1, 512>(p, sms, s);
    if (nvec <= 1024) return norm_one<T, V, 2, 512>(p, sms, s);
    if (nvec <= 2048) return norm_one<T, V, 4, 512>(p, sms, s);
    return norm_one<T, V, 4, 1024>(p, sms, s);  // fp32 rows of more than 8192 columns
  }
  if (p.H <= 512) return norm_one<T, 1, 1, 512>(p, sms, s);
  if (p.H <= 2048) return norm_one<T, 1, 4, 512>(p, sms, s);
  return norm_one<T, 1, 16, 1024>(p, sms, s);
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
