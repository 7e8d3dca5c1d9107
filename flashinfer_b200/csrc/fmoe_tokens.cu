// fmoe_tokens.cu -- tokens sorted by expert and back, with weights applied, and the gradients.
//
// Pick p = t * K + k of topk_ids is local if key(p) = topk_ids[p] - offset lies in [0, E). Its
// row is base[key] + (how many earlier picks have the same key): a stable counting sort, so the
// tables do not depend on the order in which blocks or threads run. base[e] are the sums of the
// counts, each rounded up to `align`.
//   order    expert_base [E + 1], row_pick [R] (-1 = no pick), pick_row [T, K] (-1 = no row)
//   sort     rows[r] = x[row_pick[r] / K]
//   unsort   y[t] = sum over k ascending of w[t, k] * rows[pick_row[t, k]], fp32, one rounding
//   backward of sort: unsort without weights; backward of unsort: drows[r] = w * dy[t] and
//   dw[t, k] = <dy[t], rows[pick_row[t, k]]> in fp32
#include "fmoe_elem.cuh"
#include "fmoe_internal.h"

namespace fmoe {
namespace {

constexpr int kOrderThreads = 256;       // threads of a multi-block order kernel
constexpr int kOrderChunk = 1024;        // picks of one block, at least
constexpr int kOrderMaxBlocks = 64;      // chunk grows beyond kOrderChunk * kOrderMaxBlocks picks
constexpr int kOrderSingle = 4096;       // up to this many picks one block does everything

struct OrderShape {
  int64_t picks;
  int chunk;    // picks per block (multiple of 32 * warps)
  int blocks;
  int threads;
};

OrderShape order_shape(int64_t picks, int E) {
  OrderShape s{};
  s.picks = picks;
  // every warp keeps a count per expert in shared memory: 32 KB for 32 warps and 256 experts,
  // the same for 8 warps and 1024
  if (picks <= kOrderSingle) {
    s.threads = E <= 256 ? (picks <= 256 ? 256 : 1024) : 256;
    s.blocks = 1;
    const int64_t step = s.threads;
    s.chunk = static_cast<int>((picks + step - 1) / step * step);
  } else {
    s.threads = kOrderThreads;
    int64_t chunk = (picks + kOrderMaxBlocks - 1) / kOrderMaxBlocks;
    if (chunk < kOrderChunk) chunk = kOrderChunk;
    s.chunk = static_cast<int>((chunk + kOrderThreads - 1) / kOrderThreads * kOrderThreads);
    s.blocks = static_cast<int>((picks + s.chunk - 1) / s.chunk);
  }
  return s;
}

__device__ __forceinline__ int pick_key(const int32_t* ids, int64_t p, int64_t end, int E,
                                        int offset) {
  if (p >= end) return -1;
  const int64_t key = static_cast<int64_t>(ids[p]) - offset;
  return key >= 0 && key < E ? static_cast<int>(key) : -1;
}

// hist[b][e]: picks of expert e in block b's chunk.
__global__ void __launch_bounds__(kOrderThreads)
    k_order_count(const int32_t* ids, int64_t picks, int chunk, int E, int offset,
                  int32_t* hist) {
  pdl_begin_in_order();
  __shared__ int cnt[kMaxOrderExperts];
  for (int e = threadIdx.x; e < E; e += blockDim.x) cnt[e] = 0;
  __syncthreads();
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * chunk;
  const int64_t end = min(picks, p0 + chunk);
  for (int64_t p = p0 + threadIdx.x; p < end; p += blockDim.x) {
    const int key = pick_key(ids, p, end, E, offset);
    if (key >= 0) atomicAdd(&cnt[key], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x)
    hist[static_cast<size_t>(blockIdx.x) * E + e] = cnt[e];
}

// Ranks every pick of the block's chunk and writes the tables. Each warp owns a contiguous piece
// of the chunk and walks it 32 picks at a time; picks of one expert inside the 32 are ranked by
// lane (match_any), so rows follow the picks' order. With several blocks, the counts of the
// others come from hist.
__global__ void __launch_bounds__(1024)
    k_order_place(const int32_t* ids, int64_t picks, int chunk, int E, int offset, int align,
                  int64_t R, const int32_t* hist, int32_t* expert_base, int32_t* row_pick,
                  int32_t* pick_row) {
  pdl_begin_in_order();
  extern __shared__ int sm[];
  const int nwarp = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* cnt = sm;                 // [nwarp][E]
  int* first = sm + nwarp * E;   // [E]: base of the expert plus the counts of earlier blocks
  __shared__ int warp_tot[32];
  __shared__ int carry;
  for (int i = threadIdx.x; i < nwarp * E; i += blockDim.x) cnt[i] = 0;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  const int per_warp = chunk / nwarp;  // a multiple of 32
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * chunk + static_cast<int64_t>(warp) * per_warp;
  const int64_t wend = min(picks, w0 + per_warp);
  int* mine = cnt + warp * E;
  for (int64_t p = w0; p < wend; p += 32) {
    const int key = pick_key(ids, p + lane, wend, E, offset);
    const unsigned peers = __match_any_sync(0xffffffffu, key);
    if (key >= 0 && lane == __ffs(peers) - 1) mine[key] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  // experts in rounds of blockDim: totals, then an exclusive scan of the padded totals
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0, padded = 0;
    if (e < E) {
      int run = 0;
      for (int w = 0; w < nwarp; ++w) {
        const int c = cnt[w * E + e];
        cnt[w * E + e] = run;
        run += c;
      }
      total = run;
      if (hist) {
        total = 0;
#pragma unroll 8
        for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
          const int c = __ldcg(hist + static_cast<size_t>(b) * E + e);
          if (b < static_cast<int>(blockIdx.x)) before += c;
          total += c;
        }
      }
      padded = (total + align - 1) / align * align;
    }
    int incl = padded;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int t = lane < nwarp ? warp_tot[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += up;
      }
      if (lane < nwarp) warp_tot[lane] = t;
    }
    __syncthreads();
    const int base = carry + incl - padded + (warp > 0 ? warp_tot[warp - 1] : 0);
    if (e < E) {
      first[e] = base + before;
      if (blockIdx.x == 0) expert_base[e] = base;
      // the padding rows of expert e hold no pick
      if (e % gridDim.x == blockIdx.x)
        for (int r = base + total; r < base + padded; ++r) row_pick[r] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) carry += warp_tot[nwarp - 1];
    __syncthreads();
  }
  const int live = carry;
  if (blockIdx.x == 0 && threadIdx.x == 0) expert_base[E] = live;
  for (int64_t p = w0; p < wend; p += 32) {
    const int key = pick_key(ids, p + lane, wend, E, offset);
    const unsigned peers = __match_any_sync(0xffffffffu, key);
    int row = -1;
    if (key >= 0) row = first[key] + mine[key] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (key >= 0 && lane == __ffs(peers) - 1) mine[key] += __popc(peers);
    __syncwarp();
    if (p + lane < wend) pick_row[p + lane] = row;
    if (row >= 0) row_pick[row] = static_cast<int32_t>(p + lane);
  }
  // rows behind the last expert's hold no pick
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t r = live + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; r < R; r += step)
    row_pick[r] = -1;
}

// Zeroes the rows without a pick among [0, limit): blocks b of nb, a warp looks at 32 rows at a
// time. U: the access unit, nvec of them per row.
template <typename U>
__device__ __forceinline__ void zero_rows(U* rows, const int32_t* row_pick, int64_t limit,
                                          int64_t nvec, int b, int nb) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int nwarp = (blockDim.x * blockDim.y) >> 5, warp = tid >> 5, lane = tid & 31;
  const int64_t step = static_cast<int64_t>(nb) * nwarp * 32;
  for (int64_t r0 = (static_cast<int64_t>(b) * nwarp + warp) * 32; r0 < limit; r0 += step) {
    const bool none = r0 + lane < limit && __ldcg(row_pick + r0 + lane) < 0;
    unsigned todo = __ballot_sync(0xffffffffu, none);
    while (todo) {
      const int64_t r = r0 + __ffs(todo) - 1;
      todo &= todo - 1;
      for (int64_t v = lane; v < nvec; v += 32) rows[r * nvec + v] = U{};
    }
  }
}

struct RowsArgs {
  const int32_t* expert_base;
  const int32_t* row_pick;
  const int32_t* pick_row;
  int T, K, E;
  int64_t R;
  int64_t nvec;     // access units per row
  int chunks;       // blocks along a row
  int copy_blocks;  // blocks that take tokens; the others zero rows
  int zero_tail;    // rows from expert_base[E] on are zeroed too
};

__device__ __forceinline__ int64_t zero_limit(const RowsArgs& a) {
  if (a.zero_tail) return a.R;
  const int64_t live = __ldcg(a.expert_base + a.E);
  return live < a.R ? live : a.R;
}

// Copies token rows to their picks' rows: each token is read once and stored K times.
template <typename U>
__global__ void __launch_bounds__(256) k_sort_rows(const U* x, U* rows, const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(rows, a.row_pick, zero_limit(a), a.nvec, blockIdx.x - a.copy_blocks,
              gridDim.x - a.copy_blocks);
    return;
  }
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(a.chunks) * blockDim.x;
  if (t >= a.T) return;
  const int32_t* pr = a.pick_row + t * a.K;
  for (int64_t v = static_cast<int64_t>(blockIdx.x % a.chunks) * blockDim.x + threadIdx.x;
       v < a.nvec; v += step) {
    const U val = x[t * a.nvec + v];
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = __ldcg(pr + k);
      if (r >= 0 && r < a.R) rows[r * a.nvec + v] = val;
    }
  }
}

// Up to eight picks of a token from k0 on: their rows (-1: none) and weights.
struct Picks {
  int r[8];
  float f[8];
};

__device__ __forceinline__ Picks load_picks(const RowsArgs& a, const float* w, int64_t t, int k0) {
  Picks p;
  const int64_t at = t * a.K + k0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool has = k0 + j < a.K;
    p.r[j] = has ? __ldcg(a.pick_row + at + j) : -1;
    p.f[j] = has && w ? __ldcg(w + at + j) : 1.0f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (p.r[j] >= a.R) p.r[j] = -1;
    if (p.r[j] < 0) p.f[j] = 0.0f;  // a weight without a row is not used, whatever it holds
  }
  return p;
}

// The picks k0 .. k0 + 31 of one token, one per lane (a warp works on one token at a time).
struct LanePick {
  int r;    // row, -1: none
  float f;  // weight, 0 without a row, whatever the weight holds
};

__device__ __forceinline__ LanePick lane_pick(const RowsArgs& a, const float* w, int64_t t, int k0) {
  const int k = k0 + (threadIdx.x & 31);
  LanePick p{-1, 0.0f};
  if (t < a.T && k < a.K) {
    p.r = __ldcg(a.pick_row + t * a.K + k);
    if (p.r >= a.R) p.r = -1;
    if (p.r >= 0) p.f = w ? __ldcg(w + t * a.K + k) : 1.0f;
  }
  return p;
}

// y[t] = sum_k w[t, k] * rows[pick_row[t, k]] (w null: 1), k ascending, in fp32. Eight rows' loads
// are in flight per thread; a pick without a row adds 0 * 0, so the sums have no branches. With
// single conversions and a branch per pick the kernel issued 75 instructions per row and granule.
template <typename T>
__global__ void __launch_bounds__(256, 3)
    k_unsort_granules(const T* rows, const float* w, T* y, const RowsArgs a) {
  pdl_begin_in_order();
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(a.chunks) * blockDim.x;
  if (t >= a.T) return;
  const uint4* in = reinterpret_cast<const uint4*>(rows);
  for (int64_t v = static_cast<int64_t>(blockIdx.x % a.chunks) * blockDim.x + threadIdx.x;
       v < a.nvec; v += step) {
    Gran<T> acc;
    zero(acc);
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      const Picks p = load_picks(a, w, t, k0);
      uint4 q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[j] = make_uint4(0u, 0u, 0u, 0u);
        if (p.r[j] >= 0) q[j] = __ldcg(in + p.r[j] * a.nvec + v);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc = fma(gran_of<T>(q[j]), p.f[j], acc);
    }
    reinterpret_cast<uint4*>(y)[t * a.nvec + v] = words_of(acc);
  }
}

// The same by single elements, for rows that are no multiple of 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256)
    k_unsort_elements(const T* rows, const float* w, T* y, const RowsArgs a) {
  pdl_begin_in_order();
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(a.chunks) * blockDim.x;
  if (t >= a.T) return;
  for (int64_t v = static_cast<int64_t>(blockIdx.x % a.chunks) * blockDim.x + threadIdx.x;
       v < a.nvec; v += step) {
    float acc = 0.0f;
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      const Picks p = load_picks(a, w, t, k0);
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        e[j] = p.r[j] >= 0 ? to_f32(load_pack<T, 1>(rows + p.r[j] * a.nvec + v).e) : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc = fmaf(p.f[j], e[j], acc);
    }
    from_f32(acc, y + t * a.nvec + v);
  }
}

// The eight sums of a block's threads, added in a fixed order (lane tree, warps ascending), to
// dw[t, k0 ..]. One barrier: the next call uses another `part`.
__device__ __forceinline__ void store_dots(float (&dot)[8], float* dw, int64_t t, int k0, int K,
                                           float (*part)[8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float s = warp_sum_f32(dot[j]);
    if (lane == 0) part[warp][j] = s;
  }
  __syncthreads();
  if (threadIdx.x < 8 && k0 + static_cast<int>(threadIdx.x) < K) {
    float s = 0.0f;
    for (int i = 0; i < nwarp; ++i) s += part[i][threadIdx.x];
    dw[t * K + k0 + threadIdx.x] = s;
  }
}

// One block per token at a time: drows[pick_row[t, k]] = w[t, k] * dy[t]; dw[t, k] =
// <dy[t], rows[..]> (dw null: rows are not read; drows null: not written). Eight picks at a time.
template <typename T>
__global__ void __launch_bounds__(256, 3)
    k_unsort_back_granules(const T* dy, const T* rows, const float* w, T* drows, float* dw,
                           const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(reinterpret_cast<uint4*>(drows), a.row_pick, zero_limit(a), a.nvec,
              blockIdx.x - a.copy_blocks, gridDim.x - a.copy_blocks);
    return;
  }
  __shared__ float part[2][8][8];
  const int nvec = static_cast<int>(a.nvec);
  const uint4* in = reinterpret_cast<const uint4*>(rows);
  uint4* out = reinterpret_cast<uint4*>(drows);
  int flip = 0;
  int64_t t = blockIdx.x;
  LanePick next = lane_pick(a, w, t, 0);
  for (; t < a.T; t += a.copy_blocks) {
    const uint4* g_in = reinterpret_cast<const uint4*>(dy) + t * nvec;
    LanePick p = next;
    next = lane_pick(a, w, t + a.copy_blocks, 0);
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      const int k = k0 & 31;
      if (k0 > 0 && k == 0) p = lane_pick(a, w, t, k0);
      float2 dot2[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) dot2[j] = make_float2(0.0f, 0.0f);
      // whole warps keep going for the shuffles
      for (int v0 = 0; v0 < nvec; v0 += blockDim.x) {
        const int v = v0 + threadIdx.x;
        uint4 gq = make_uint4(0u, 0u, 0u, 0u), q[8];
        if (v < nvec) gq = __ldcg(g_in + v);
        if (dw) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = __shfl_sync(0xffffffffu, p.r, k + j);
            q[j] = make_uint4(0u, 0u, 0u, 0u);
            if (r >= 0 && v < nvec) q[j] = __ldcg(in + static_cast<int64_t>(r) * nvec + v);
          }
        }
        const Gran<T> g = gran_of<T>(gq);
        if (drows) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = __shfl_sync(0xffffffffu, p.r, k + j);
            const float f = __shfl_sync(0xffffffffu, p.f, k + j);
            if (r >= 0 && v < nvec) out[static_cast<int64_t>(r) * nvec + v] = words_of(mul(g, f));
          }
        }
        if (dw) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const Gran<T> e = gran_of<T>(q[j]);
#pragma unroll
            for (int i = 0; i < Gran<T>::N; ++i) dot2[j] = __ffma2_rn(g.p[i], e.p[i], dot2[j]);
          }
        }
      }
      if (dw) {
        float dot[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)  // a gradient that is no number stays out of absent picks
          dot[j] = __shfl_sync(0xffffffffu, p.r, k + j) >= 0 ? dot2[j].x + dot2[j].y : 0.0f;
        store_dots(dot, dw, t, k0, a.K, part[flip]);
        flip ^= 1;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_unsort_back_elements(const T* dy, const T* rows, const float* w, T* drows, float* dw,
                           const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(reinterpret_cast<Pack<T, 1>*>(drows), a.row_pick, zero_limit(a), a.nvec,
              blockIdx.x - a.copy_blocks, gridDim.x - a.copy_blocks);
    return;
  }
  __shared__ float part[2][8][8];
  const int64_t t = blockIdx.x;
  for (int k0 = 0; k0 < a.K; k0 += 8) {
    const Picks p = load_picks(a, w, t, k0);
    float dot[8] = {};
    for (int64_t v = threadIdx.x; v < a.nvec; v += blockDim.x) {
      const float g = to_f32(load_pack<T, 1>(dy + t * a.nvec + v).e);
      float e[8];
      if (dw) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          e[j] = p.r[j] >= 0 ? to_f32(load_pack<T, 1>(rows + p.r[j] * a.nvec + v).e) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (drows && p.r[j] >= 0) from_f32(p.f[j] * g, drows + p.r[j] * a.nvec + v);
        if (dw && p.r[j] >= 0) dot[j] = fmaf(g, e[j], dot[j]);
      }
    }
    if (dw) store_dots(dot, dw, t, k0, a.K, part[(k0 >> 3) & 1]);
  }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Block shape for rows of nvec units: up to 256 threads along the row, several tokens per block
// where a row is shorter.
struct RowGrid {
  dim3 block;
  int chunks;
  int64_t blocks;
};

RowGrid row_grid(int64_t T, int64_t nvec, int per_thread) {
  RowGrid g{};
  if (nvec < 256) {
    int tx = 1;
    while (tx < nvec) tx *= 2;
    g.block = dim3(tx, 256 / tx);
    g.chunks = 1;
  } else {
    // blocks of equal length along the row, a multiple of a warp each
    const int64_t units = (nvec + per_thread - 1) / per_thread;
    g.chunks = static_cast<int>((units + 255) / 256);
    const int64_t tx = ((units + g.chunks - 1) / g.chunks + 31) / 32 * 32;
    g.block = dim3(static_cast<unsigned>(tx), 1);
  }
  g.blocks = (T + g.block.y - 1) / g.block.y * g.chunks;
  return g;
}

RowsArgs rows_args(const TokenOrder& o, int64_t nvec) {
  RowsArgs a{};
  a.expert_base = o.expert_base;
  a.row_pick = o.row_pick;
  a.pick_row = o.pick_row;
  a.T = o.T;
  a.K = o.K;
  a.E = o.E;
  a.R = o.R;
  a.nvec = nvec;
  return a;
}

int zero_blocks(int64_t R, int num_sms) {
  const int64_t b = (R + 255) / 256;
  return static_cast<int>(b < 2 * num_sms ? b : 2 * num_sms);
}

template <typename U>
cudaError_t sort_rows(const void* x, void* rows, const TokenOrder& o, int64_t row_bytes,
                      int zero_tail, int num_sms, cudaStream_t s) {
  RowsArgs a = rows_args(o, row_bytes / static_cast<int64_t>(sizeof(U)));
  const RowGrid g = row_grid(o.T, a.nvec, sizeof(U) == 16 ? 1 : 4);
  a.chunks = g.chunks;
  a.copy_blocks = static_cast<int>(g.blocks);
  a.zero_tail = zero_tail;
  return launch_pdl(k_sort_rows<U>, dim3(static_cast<unsigned>(g.blocks + zero_blocks(o.R, num_sms))),
                    g.block, 0, s, static_cast<const U*>(x), static_cast<U*>(rows), a);
}

template <typename T>
cudaError_t unsort_rows(const void* rows, const float* w, void* y, const TokenOrder& o, int64_t H,
                        bool vec, cudaStream_t s) {
  RowsArgs a = rows_args(o, vec ? H / kV<T> : H);
  const RowGrid g = row_grid(o.T, a.nvec, vec ? 1 : 4);
  a.chunks = g.chunks;
  return launch_pdl(vec ? k_unsort_granules<T> : k_unsort_elements<T>,
                    dim3(static_cast<unsigned>(g.blocks)), g.block, 0, s,
                    static_cast<const T*>(rows), w, static_cast<T*>(y), a);
}

template <typename T>
cudaError_t unsort_back(const void* dy, const void* rows, const float* w, void* drows, float* dw,
                        const TokenOrder& o, int64_t H, bool vec, int num_sms, cudaStream_t s) {
  RowsArgs a = rows_args(o, vec ? H / kV<T> : H);
  int64_t threads = (a.nvec + 31) / 32 * 32;
  if (threads > 256) threads = 256;
  a.copy_blocks = o.T;
  const int64_t most = static_cast<int64_t>(num_sms) * (768 / threads);
  if (vec && a.copy_blocks > most) a.copy_blocks = static_cast<int>(most);
  a.zero_tail = 1;
  const int64_t blocks = a.copy_blocks + (drows ? zero_blocks(o.R, num_sms) : 0);
  return launch_pdl(vec ? k_unsort_back_granules<T> : k_unsort_back_elements<T>,
                    dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), 0, s,
                    static_cast<const T*>(dy), static_cast<const T*>(rows), w,
                    static_cast<T*>(drows), dw, a);
}

}  // namespace

size_t order_scratch_bytes(int64_t picks, int E) {
  const OrderShape s = order_shape(picks, E);
  return s.blocks > 1 ? static_cast<size_t>(s.blocks) * E * 4 : 0;
}

cudaError_t launch_order(const int32_t* ids, const TokenOrder& o, int offset, int align,
                         int32_t* expert_base, int32_t* row_pick, int32_t* pick_row,
                         int32_t* hist, cudaStream_t s) {
  const OrderShape sh = order_shape(static_cast<int64_t>(o.T) * o.K, o.E);
  const int32_t* counts = nullptr;
  if (sh.blocks > 1) {
    const cudaError_t e = launch_pdl(k_order_count, dim3(sh.blocks), dim3(kOrderThreads), 0, s,
                                     ids, sh.picks, sh.chunk, o.E, offset, hist);
    if (e != cudaSuccess) return e;
    counts = hist;
  }
  const size_t smem = (static_cast<size_t>(sh.threads / 32) + 1) * o.E * 4;  // at most 36 KB
  return launch_pdl(k_order_place, dim3(sh.blocks), dim3(sh.threads), smem, s, ids, sh.picks,
                    sh.chunk, o.E, offset, align, o.R, counts, expert_base, row_pick, pick_row);
}

cudaError_t launch_sort_rows(const void* x, void* rows, const TokenOrder& o, int64_t row_bytes,
                             int zero_tail, int num_sms, cudaStream_t s) {
  const auto fits = [&](int64_t n) {
    return row_bytes % n == 0 && aligned(x, n) && aligned(rows, n);
  };
  if (fits(16)) return sort_rows<uint4>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  if (fits(4)) return sort_rows<uint32_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  if (fits(2)) return sort_rows<uint16_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  return sort_rows<uint8_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
}

cudaError_t launch_unsort_rows(const void* rows, const float* w, void* y, int dtype,
                               const TokenOrder& o, int64_t H, cudaStream_t s) {
  const int64_t bytes = H * (dtype == FMOE_DTYPE_F32 ? 4 : 2);
  const bool vec = bytes % 16 == 0 && aligned(rows, 16) && aligned(y, 16);
  switch (dtype) {
    case FMOE_DTYPE_F32:
      return unsort_rows<float>(rows, w, y, o, H, vec, s);
    case FMOE_DTYPE_BF16:
      return unsort_rows<__nv_bfloat16>(rows, w, y, o, H, vec, s);
    default:
      return unsort_rows<__half>(rows, w, y, o, H, vec, s);
  }
}

cudaError_t launch_unsort_back(const void* dy, const void* rows, const float* w, void* drows,
                               float* dw, int dtype, const TokenOrder& o, int64_t H, int num_sms,
                               cudaStream_t s) {
  const int64_t bytes = H * (dtype == FMOE_DTYPE_F32 ? 4 : 2);
  const bool vec = bytes % 16 == 0 && aligned(dy, 16) && aligned(drows, 16) &&
                   (!dw || aligned(rows, 16));
  switch (dtype) {
    case FMOE_DTYPE_F32:
      return unsort_back<float>(dy, rows, w, drows, dw, o, H, vec, num_sms, s);
    case FMOE_DTYPE_BF16:
      return unsort_back<__nv_bfloat16>(dy, rows, w, drows, dw, o, H, vec, num_sms, s);
    default:
      return unsort_back<__half>(dy, rows, w, drows, dw, o, H, vec, num_sms, s);
  }
}

}  // namespace fmoe
