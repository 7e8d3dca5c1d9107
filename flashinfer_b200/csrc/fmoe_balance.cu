// fmoe_balance.cu -- the router's balance loss, the counts per expert it needs, and its gradient.
//
//   p[t, e]  = exp(u[t, e]) / sum_e' exp(u[t, e']),  u = logits, or log sigmoid(logits)
//   n[s, e]  = picks of expert e by the T_s tokens of sequence s
//   L_s      = sum_e  E n[s, e] / (K T_s) * (1 / T_s) sum_{t in s} p[t, e]
//   loss     = mean of L_s over the sequences that have tokens
// and with c[s, e] = E n[s, e] / (K T_s^2 S), S those sequences' number, g the gradient of the loss:
//   d logits = g p (c - sum_e p c) * (1, or sigmoid(-logits))
//
// Forward: every block takes a range of tokens and adds up p (in registers, a lane's columns) and the
// picks (in shared memory) of each sequence in it; one cluster then adds the blocks' shares in order.
// The picks are counted beside the scores and need no pass of their own, and nothing has to be
// zeroed first. Backward: one pass, a token per warp, the scores computed again. Logits are read once
// per pass: bound by HBM, at small sizes by the two launches.
#include <atomic>

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

// Warps of a block: what the registers of NV logits per lane leave room for, all on one SM. Few blocks have few
// shares to join.
constexpr int bal_warps(int NV) { return NV > 8 ? 16 : 32; }
constexpr int kBackWarps = 8;     // of the backward pass
constexpr int kBalCluster = 8;   // CTAs of the cluster that joins the shares
constexpr int kBalMaxSmem = 16 * kMaxBalanceExperts * 4 + kMaxBalanceExperts * 4 +
                            (kMaxBalanceSequences + 1) * 4;

struct BalArgs {
  const void* logits;      // [T, E], or null: counts only (loss null), or no tokens
  const int32_t* ids;      // [T, K]
  const int32_t* base;     // [S + 1], or null: one sequence of all rows
  int64_t T;
  int E, K, S, sigmoid;
  int rows;                // per block
  int blocks;
  float* part_p;           // [blocks + S][E]
  int32_t* part_n;         // [blocks + S][E]
  float* loss;
  int32_t* counts;         // [S, E]
  float* factor;           // [S]: E / (K T_s^2 S'), 0 for a sequence without tokens
  // backward
  const float* g;
  void* d_logits;
};

// The sequences' first rows, and the end of the last, to shared memory: clamped to [0, T], and as a running
// maximum, so that with a base that steps back no row belongs to two sequences. By the whole block, with a
// barrier at the end.
__device__ __forceinline__ void load_bases(const BalArgs& a, int* sbase) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int s0 = 0; s0 <= a.S; s0 += 32) {
      const int s = s0 + lane;
      int64_t b = 0;
      if (s <= a.S) b = a.base ? __ldcg(a.base + s) : s == 0 ? 0 : a.T;
      int most = max(carry, static_cast<int>(b < 0 ? 0 : b > a.T ? a.T : b));
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, most, o);
        if (lane >= o) most = max(most, up);
      }
      if (s <= a.S) sbase[s] = most;
      carry = __shfl_sync(0xffffffffu, most, 31);
    }
  }
  __syncthreads();
}

// The first sequence that ends behind the row (S: none).
__device__ __forceinline__ int sequence_of(const int* sbase, int S, int64_t row) {
  int lo = 0, hi = S;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sbase[mid + 1] > row)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// A lane's values of one row: NV values in units of V, unit u of lane l being number u * 32 + l.
template <typename T, int V, int NV>
__device__ __forceinline__ void load_logits(const BalArgs& a, int64_t row, float (&v)[NV]) {
  const int lane = threadIdx.x & 31, n = a.E / V;
  const T* p = static_cast<const T*>(a.logits) + row * a.E;
#pragma unroll
  for (int u = 0; u < NV / V; ++u) {
    const int i = u * 32 + lane;
    float w[V];
    if (i < n) {
      unpack(load_pack<T, V>(p + i * V), w);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[u * V + j] = w[j];
  }
}

// v: logits in, exp(u - m) out, with m such that the largest are of ordinary size; slope:
// d u / d logits (SLOPE). Returns 1 / sum, or 0 for a row whose logits are all -infinity (or whose
// sigmoids all are 0): it has no scores. A NaN among the logits makes the sum NaN.
//
// sigmoid(l) itself is taken as the exponential (m = 0) unless every logit is below -60, where they
// would run out of range: then sigmoid(l) exp(-m) = exp(l - m) / (1 + exp(l)) with m the largest logit.
template <int NV, bool SLOPE>
__device__ __forceinline__ float scores(float (&v)[NV], float (&slope)[SLOPE ? NV : 1], bool sigmoid) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, v[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float sum = 0.0f;
  if (!sigmoid || m < -60.0f) {
    const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // below -60 the factor 1 / (1 + exp(l)) is 1 to fp32, as is d u / d logits
      v[i] = expf(v[i] - shift);
      if constexpr (SLOPE) slope[i] = 1.0f;
      sum += v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float t = expf(-fabsf(v[i]));
      const float r = __fdividef(1.0f, 1.0f + t);
      const bool neg = v[i] <= 0.0f;
      const float e = (neg ? t : 1.0f) * r;
      if constexpr (SLOPE) slope[i] = (neg ? 1.0f : t) * r;
      v[i] = e;
      sum += e;
    }
  }
  sum = warp_sum_f32(sum);
  return sum == 0.0f ? 0.0f : 1.0f / sum;
}

// The shares of a block of rows: one for each sequence that has rows in it. The share of (block b,
// sequence s) is number b + s: along the rows either b or s goes up from one share to the next, so no
// two have the same number.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(bal_warps(NV) * 32) k_balance(const BalArgs a) {
  constexpr int WARPS = bal_warps(NV), THREADS = WARPS * 32;
  extern __shared__ float bal_smem[];
  float* sp = bal_smem;                                          // [WARPS][E]
  int* sn = reinterpret_cast<int*>(sp + (a.logits ? WARPS * a.E : 0));  // [E]
  int* sbase = sn + a.E;                                                   // [S + 1]
  pdl_begin_in_order();
  load_bases(a, sbase);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.rows;
  const int64_t r1 = min(r0 + a.rows, a.T);
  for (int s = sequence_of(sbase, a.S, r0); s < a.S && sbase[s] < r1; ++s) {
    const int64_t b0 = max(static_cast<int64_t>(sbase[s]), r0);
    const int64_t b1 = min(static_cast<int64_t>(sbase[s + 1]), r1);
    if (b0 >= b1) continue;
    float next[NV];  // the logits of this warp's next row
    int64_t row = b0 + warp;
    if (a.logits && row < b1) load_logits<T, V, NV>(a, row, next);
    for (int e = threadIdx.x; e < a.E; e += THREADS) sn[e] = 0;
    __syncthreads();
    const int64_t p1 = b1 * a.K;
    for (int64_t p = b0 * a.K + threadIdx.x; p < p1; p += THREADS) {
      const int id = __ldcg(a.ids + p);
      if (id >= 0 && id < a.E) atomicAdd(sn + id, 1);
    }
    if (a.logits) {
      float acc[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
      for (; row < b1; row += WARPS) {
        float v[NV], none[1];
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = next[i];
        if (row + WARPS < b1) load_logits<T, V, NV>(a, row + WARPS, next);
        const float inv = scores<NV, false>(v, none, a.sigmoid);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = fmaf(v[i], inv, acc[i]);
      }
#pragma unroll
      for (int u = 0; u < NV / V; ++u) {
        const int i = u * 32 + lane;
        if (i < a.E / V) {
#pragma unroll
          for (int j = 0; j < V; ++j) sp[warp * a.E + i * V + j] = acc[u * V + j];
        }
      }
    }
    __syncthreads();
    const int64_t at = (static_cast<int64_t>(blockIdx.x) + s) * a.E;
    for (int e = threadIdx.x; e < a.E; e += THREADS) {
      a.part_n[at + e] = sn[e];
      if (a.logits) {
        float sum = 0.0f;
#pragma unroll 8
        for (int w = 0; w < WARPS; ++w) sum += sp[w * a.E + e];
        a.part_p[at + e] = sum;
      }
    }
    __syncthreads();
  }
}

// Adds the blocks' shares. The cluster's CTAs take the (sequence, 32 experts) pieces in turn, a warp every 32nd
// share of a piece; the terms of the loss are added in double, in an order that is the same in every run.
constexpr int kJoinThreads = 1024;

__global__ void __launch_bounds__(kJoinThreads) k_balance_join(const BalArgs a) {
  extern __shared__ float bal_smem[];
  int* sbase = reinterpret_cast<int*>(bal_smem);  // [S + 1]
  __shared__ float bp[32][33];
  __shared__ int bn[32][33];
  __shared__ double part[32];
  __shared__ double shares[kBalCluster];  // of every CTA, in the first one
  __shared__ int live_seqs;
  cluster_arrive();  // once all have arrived their shared memory can be written to
  pdl_begin_in_order();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  if (threadIdx.x == 0) live_seqs = 0;
  load_bases(a, sbase);
  int mine = 0;
  for (int s = threadIdx.x; s < a.S; s += kJoinThreads) mine += sbase[s + 1] > sbase[s];
  if (mine) atomicAdd(&live_seqs, mine);
  __syncthreads();
  const float live = static_cast<float>(live_seqs);
  const int chunks = (a.E + 31) / 32;
  const int64_t pieces = static_cast<int64_t>(a.S) * chunks;
  double sum = 0.0;  // of each warp's first lane
  for (int64_t piece = rank; piece < pieces; piece += kBalCluster) {
    const int s = static_cast<int>(piece / chunks);
    const int e = static_cast<int>(piece - static_cast<int64_t>(s) * chunks) * 32 + lane;
    const int64_t b0 = sbase[s], b1 = sbase[s + 1];
    float p = 0.0f;
    int n = 0;
    if (b0 < b1 && e < a.E) {
      const int first = static_cast<int>(b0 / a.rows), last = static_cast<int>((b1 - 1) / a.rows);
      const float* pp = a.part_p + static_cast<int64_t>(s) * a.E + e;
      const int32_t* pn = a.part_n + static_cast<int64_t>(s) * a.E + e;
      for (int b = first + warp; b <= last; b += 32 * 4) {
        float tp[4];
        int tn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = b + 32 * i <= last;
          const int64_t at = static_cast<int64_t>(b + 32 * i) * a.E;
          tn[i] = in ? __ldcg(pn + at) : 0;
          tp[i] = in && a.loss ? __ldcg(pp + at) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p += tp[i];
          n += tn[i];
        }
      }
    }
    bp[warp][lane] = p;
    bn[warp][lane] = n;
    __syncthreads();
    // a warp per expert adds its 32 parts
    p = warp_sum_f32(bp[lane][warp]);
    n = __reduce_add_sync(0xffffffffu, bn[lane][warp]);
    const int mine = e - lane + warp;
    if (lane == 0 && mine < a.E) {
      a.counts[static_cast<int64_t>(s) * a.E + mine] = n;
      if (a.loss) {
        const float len = static_cast<float>(b1 - b0);
        const float factor = b0 < b1 ? static_cast<float>(a.E) / (static_cast<float>(a.K) * live * len * len) : 0.0f;
        if (b0 < b1) sum += static_cast<double>(factor * n) * p;
        if (mine == 0) a.factor[s] = factor;
      }
    }
    __syncthreads();
  }
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  cluster_wait();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < 32; ++i) t += part[i];
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&shares[rank])), "r"(0));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(t) : "memory");
  }
  cluster_arrive();
  cluster_wait();
  if (a.loss && rank == 0 && threadIdx.x == 0) {
    double t = 0.0;
    for (int r = 0; r < kBalCluster; ++r) t += shares[r];
    *a.loss = static_cast<float>(t);
  }
}

// A token per warp, neighbouring tokens one after the other; c = counts * factor of its sequence stays in
// registers while the sequence does. Rows of no sequence get zeros.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(kBackWarps * 32) k_balance_back(const BalArgs a) {
  extern __shared__ float bal_smem[];
  int* sbase = reinterpret_cast<int*>(bal_smem);  // [S + 1]
  pdl_begin_in_order();
  load_bases(a, sbase);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = a.E / V;
  const int64_t r0 = (static_cast<int64_t>(blockIdx.x) * kBackWarps + warp) * a.rows;
  const int64_t r1 = min(r0 + a.rows, a.T);
  if (r0 >= r1) return;
  const float g = *a.g;
  int s = sequence_of(sbase, a.S, r0);
  float c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) c[i] = 0.0f;
  int64_t b0 = 0, b1 = r0;  // of sequence s; in the rows behind the last sequence, none
  float next[NV];           // the next row's logits
  load_logits<T, V, NV>(a, r0, next);
  for (int64_t row = r0; row < r1; ++row) {
    if (row >= b1) {
      while (s < a.S && sbase[s + 1] <= row) ++s;
      b0 = s < a.S ? sbase[s] : a.T;
      b1 = s < a.S ? sbase[s + 1] : a.T;
      if (s < a.S) {
        const float f = a.factor[s] * g;
        const int32_t* cn = a.counts + static_cast<int64_t>(s) * a.E;
#pragma unroll
        for (int u = 0; u < NV / V; ++u) {
          const int i = u * 32 + lane;
          if (i < n) {
            // through L1: every warp of the grid reads the same few lines (past it, 16384 x 256 took 22 us)
            if constexpr (V > 1) {
#pragma unroll
              for (int j = 0; j < V; j += 4) {
                const int4 w = *reinterpret_cast<const int4*>(cn + i * V + j);
                c[u * V + j] = static_cast<float>(w.x) * f;
                c[u * V + j + 1] = static_cast<float>(w.y) * f;
                c[u * V + j + 2] = static_cast<float>(w.z) * f;
                c[u * V + j + 3] = static_cast<float>(w.w) * f;
              }
            } else {
              c[u] = static_cast<float>(cn[i]) * f;
            }
          }
        }
      }
    }
    float v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = next[i];
    if (row + 1 < r1) load_logits<T, V, NV>(a, row + 1, next);
    if (row < b0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = 0.0f;
    } else {
      float slope[NV];
      const float inv = scores<NV, true>(v, slope, a.sigmoid);
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        v[i] *= inv;
        dot = fmaf(v[i], c[i], dot);
      }
      dot = warp_sum_f32(dot);
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = v[i] * (c[i] - dot) * slope[i];
    }
    T* out = static_cast<T*>(a.d_logits) + row * a.E;
#pragma unroll
    for (int u = 0; u < NV / V; ++u) {
      const int i = u * 32 + lane;
      float w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = v[u * V + j];
      if (i < n) store_pack(out + i * V, w);
    }
  }
}

template <typename T, int V, int NV>
cudaError_t run(const BalArgs& given, void* workspace, bool back, int sms, cudaStream_t s) {
  static std::atomic<bool> done[64];
  BalArgs a = given;
  const size_t bases = static_cast<size_t>(a.S + 1) * 4;
  if (back) {
    // the warps that run at a time share the rows evenly
    const int64_t most = static_cast<int64_t>(sms) * (NV > 8 ? 16 : 32);
    a.rows = static_cast<int>((a.T + most - 1) / most);
    const int64_t warps = (a.T + a.rows - 1) / a.rows;
    return launch_pdl(k_balance_back<T, V, NV>,
                      dim3(static_cast<unsigned>((warps + kBackWarps - 1) / kBackWarps)),
                      dim3(kBackWarps * 32), bases, s, a);
  }
  // one block per SM, of a row per warp or more
  constexpr int WARPS = bal_warps(NV);
  const int64_t most = sms < kMaxBalanceBlocks ? sms : kMaxBalanceBlocks;
  const int64_t even = ((a.T > 0 ? a.T : 1) + most - 1) / most;
  a.rows = static_cast<int>((even + WARPS - 1) / WARPS * WARPS);
  a.blocks = static_cast<int>((a.T + a.rows - 1) / a.rows);
  a.part_n = static_cast<int32_t*>(workspace);
  a.part_p = reinterpret_cast<float*>(a.part_n + (static_cast<int64_t>(a.blocks) + a.S) * a.E);
  const size_t smem = ((a.logits ? WARPS * a.E : 0) + a.E) * 4 + bases;
  if (smem > 48 * 1024) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev].load(std::memory_order_acquire)) {
      const cudaError_t e = cudaFuncSetAttribute(
          k_balance<T, V, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBalMaxSmem);
      if (e != cudaSuccess) return e;
      done[dev].store(true, std::memory_order_release);
    }
  }
  if (a.blocks > 0) {
    const cudaError_t e = launch_pdl(k_balance<T, V, NV>, dim3(a.blocks), dim3(WARPS * 32), smem, s, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl_cluster(k_balance_join, dim3(kBalCluster), dim3(kJoinThreads), bases, s,
                            kBalCluster, a);
}

template <typename T>
cudaError_t typed(const BalArgs& a, void* workspace, bool back, int sms, cudaStream_t s) {
  const bool wide = a.E % kV<T> == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.d_logits) & 15u) == 0 &&
                    (!back || (reinterpret_cast<uintptr_t>(a.counts) & 15u) == 0);
  if (a.E <= 256)
    return wide ? run<T, kV<T>, 8>(a, workspace, back, sms, s) : run<T, 1, 8>(a, workspace, back, sms, s);
  return wide ? run<T, kV<T>, 32>(a, workspace, back, sms, s) : run<T, 1, 32>(a, workspace, back, sms, s);
}

}  // namespace

cudaError_t launch_balance(const Balance& p, int sms, cudaStream_t s) {
  BalArgs a{};
  a.logits = p.back || p.loss ? p.logits : nullptr;
  a.ids = p.ids;
  a.base = p.base;
  a.T = p.T;
  a.E = p.E;
  a.K = p.K;
  a.S = p.S;
  a.sigmoid = p.sigmoid;
  a.loss = p.loss;
  a.counts = p.counts;
  a.factor = p.factor;
  a.g = p.grad_loss;
  a.d_logits = p.grad_logits;
  switch (p.dtype) {
    case FMOE_DTYPE_F32:
      return typed<float>(a, p.workspace, p.back, sms, s);
    case FMOE_DTYPE_BF16:
      return typed<__nv_bfloat16>(a, p.workspace, p.back, sms, s);
    default:
      return typed<__half>(a, p.workspace, p.back, sms, s);
  }
}

}  // namespace fmoe
