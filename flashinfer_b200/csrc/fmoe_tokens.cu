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
#include <initializer_list>

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"
#include "fmoe_ptx.cuh"

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

// The lanes of the warp whose key equals this lane's, by a vote per bit. match_any gives the same;
// with it the cluster kernel took 11.8 us for 32768 picks, not 9.2.
__device__ __forceinline__ unsigned same_key(int key, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (key >> b) & 1;
    const unsigned v = __ballot_sync(0xffffffffu, one);
    same &= one ? v : ~v;
  }
  return same;
}

// Bits that tell the keys -1 .. E - 1 apart: no key but -1 has all of them set.
__device__ __forceinline__ int key_bits(int E) { return 32 - __clz(E); }

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
// lane, so rows follow the picks' order. With several blocks, the counts of the
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
  const int bits = key_bits(E);
  for (int64_t p = w0; p < wend; p += 32) {
    const int key = pick_key(ids, p + lane, wend, E, offset);
    const unsigned peers = same_key(key, bits);
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
    const unsigned peers = same_key(key, bits);
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

// The same as a count and a place kernel in one launch: a cluster of eight CTAs takes up to 65536
// picks, the counts of the others come through distributed shared memory, and each pick's expert
// stays in a register between counting and placing. 32768 picks of 256 experts take 9.2 us, in two
// launches 11.0; 7422 picks of 20 experts 5.2 against 7.0.
constexpr int kClusterCtas = 8;
constexpr int kClusterRounds = 8;                          // of 32 picks per warp
constexpr int kClusterPicks = kClusterCtas * 1024 * kClusterRounds;
constexpr int kClusterExperts = 256;                       // 32 warps' counts: 32 KB

__global__ void __launch_bounds__(1024)
    k_order_cluster(const int32_t* ids, int64_t picks, int chunk, int E, int offset, int align,
                    int64_t R, int32_t* expert_base, int32_t* row_pick, int32_t* pick_row) {
  pdl_begin_in_order();
  extern __shared__ int sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* cnt = sm;                // [32][E]
  int* total_of = sm + 32 * E;  // [E] this CTA's counts
  int* first = total_of + E;    // [E]
  __shared__ int warp_tot[32];
  const int cta = static_cast<int>(cluster_ctarank());
  for (int i = threadIdx.x; i < 32 * E; i += 1024) cnt[i] = 0;
  const int rounds = chunk / 1024;  // at most kClusterRounds
  const int64_t w0 = static_cast<int64_t>(cta) * chunk + warp * rounds * 32;
  int key[kClusterRounds];
#pragma unroll
  for (int i = 0; i < kClusterRounds; ++i)
    key[i] = i < rounds ? pick_key(ids, w0 + i * 32 + lane, picks, E, offset) : -1;
  __syncthreads();
  int* mine = cnt + warp * E;
  const int bits = key_bits(E);
#pragma unroll
  for (int i = 0; i < kClusterRounds; ++i) {
    if (i >= rounds) break;
    const unsigned peers = same_key(key[i], bits);
    if (key[i] >= 0 && lane == __ffs(peers) - 1) mine[key[i]] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < E) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < 32; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = run;
      run += c;
    }
    total_of[e] = run;
  }
  cluster_arrive();
  cluster_wait();
  int total = 0, before = 0;
  if (e < E) {
#pragma unroll
    for (int c = 0; c < kClusterCtas; ++c) {
      const int n = ld_dsmem_s32(&total_of[e], c);
      if (c < cta) before += n;
      total += n;
    }
  }
  cluster_arrive();  // this CTA no longer reads the others' counts
  const int padded = (total + align - 1) / align * align;
  int incl = padded;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_tot[warp] = incl;
  __syncthreads();
  int base = incl - padded;
  int live = 0;
#pragma unroll
  for (int w = 0; w < kClusterExperts / 32; ++w) {  // warps beyond have no expert
    if (w < warp) base += warp_tot[w];
    live += warp_tot[w];
  }
  if (e < E) {
    first[e] = base + before;
    if (cta == 0) expert_base[e] = base;
    if (e % kClusterCtas == cta)
      for (int r = base + total; r < base + padded; ++r) row_pick[r] = -1;
  }
  if (cta == 0 && e == 0) expert_base[E] = live;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kClusterRounds; ++i) {
    if (i >= rounds) break;
    const int k = key[i];
    const int64_t p = w0 + i * 32 + lane;
    const unsigned peers = same_key(k, bits);
    int row = -1;
    if (k >= 0) row = first[k] + mine[k] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (k >= 0 && lane == __ffs(peers) - 1) mine[k] += __popc(peers);
    __syncwarp();
    if (p < picks) pick_row[p] = row;
    if (row >= 0) row_pick[row] = static_cast<int32_t>(p);
  }
  for (int64_t r = live + static_cast<int64_t>(cta) * 1024 + threadIdx.x; r < R;
       r += kClusterCtas * 1024)
    row_pick[r] = -1;
  cluster_wait();
}

// Zeroes the rows without a pick among [0, limit): blocks b of nb, a warp looks at four rows at a
// time. Whatever the rows' size, all but their ends goes in 16-byte stores.
__device__ __forceinline__ void zero_rows(void* rows, const int32_t* row_pick, int64_t limit,
                                          int64_t row_bytes, int b, int nb) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int nwarp = (blockDim.x * blockDim.y) >> 5, warp = tid >> 5, lane = tid & 31;
  const int64_t step = static_cast<int64_t>(nb) * nwarp * 4;
  for (int64_t r0 = (static_cast<int64_t>(b) * nwarp + warp) * 4; r0 < limit; r0 += step) {
    const bool none = lane < 4 && r0 + lane < limit && __ldcg(row_pick + r0 + lane) < 0;
    unsigned todo = __ballot_sync(0xffffffffu, none);
    while (todo) {
      const int64_t r = r0 + __ffs(todo) - 1;
      todo &= todo - 1;
      uint8_t* p = static_cast<uint8_t*>(rows) + r * row_bytes;
      int64_t head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15;
      if (head > row_bytes) head = row_bytes;
      if (lane < head) p[lane] = 0;
      const int64_t n = (row_bytes - head) / 16;
      uint4* q = reinterpret_cast<uint4*>(p + head);
      for (int64_t v = lane; v < n; v += 32) q[v] = make_uint4(0u, 0u, 0u, 0u);
      const int64_t done = head + n * 16;
      if (lane < row_bytes - done) p[done + lane] = 0;
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
  int64_t bytes;    // per row
  int chunks;       // blocks along a row
  int copy_blocks;  // blocks that take tokens; the others zero rows
  int zero_tail;    // rows from expert_base[E] on are zeroed too
};

__device__ __forceinline__ int64_t zero_limit(const RowsArgs& a) {
  if (a.zero_tail) return a.R;
  const int64_t live = __ldcg(a.expert_base + a.E);
  return live < a.R ? live : a.R;
}

// Copies token rows to their picks' rows: each token is read once and stored K times. Bound by the
// stores: 4096 x 7168 (bf16, top 8) takes 87 us, 93% of the copy bandwidth over its 529 MB.
template <typename U>
__global__ void __launch_bounds__(256) k_sort_rows(const U* x, U* rows, const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(rows, a.row_pick, zero_limit(a), a.bytes, blockIdx.x - a.copy_blocks,
              gridDim.x - a.copy_blocks);
    return;
  }
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(a.chunks) * blockDim.x;
  if (t >= a.T) return;
  const int32_t* pr = a.pick_row + t * a.K;
  for (int64_t v = static_cast<int64_t>(blockIdx.x % a.chunks) * blockDim.x + threadIdx.x;
       v < a.nvec; v += step) {
    const U val = __ldcg(x + t * a.nvec + v);
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      int r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = k0 + j < a.K ? __ldcg(pr + k0 + j) : -1;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r[j] >= 0 && r[j] < a.R) rows[r[j] * a.nvec + v] = val;
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
// single conversions and a branch per pick the kernel issued 75 instructions per row and granule and
// took 135 us for 4096 x 7168 (bf16, top 8); it takes 100, 81% of the copy bandwidth, and waits for
// its rows, which lie all over the input. A grid that stays resident was no faster.
template <typename T>
__global__ void __launch_bounds__(256, 4)
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
        if (p.r[j] >= 0) q[j] = load_row16(in + p.r[j] * a.nvec + v);
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

// N (4 or 8) sums of a block's threads, added in a fixed order (lane tree, warps ascending), to
// dw[t, k0 ..]. One barrier: the next call uses another `part`.
template <int N>
__device__ __forceinline__ void store_dots(float (&dot)[N], float* dw, int64_t t, int k0, int K,
                                           float (*part)[8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float s = warp_sum_f32(dot[j]);
    if (lane == 0) part[warp][j] = s;
  }
  __syncthreads();
  if (threadIdx.x < N && k0 + static_cast<int>(threadIdx.x) < K) {
    float s = 0.0f;
    for (int i = 0; i < nwarp; ++i) s += part[i][threadIdx.x];
    dw[t * K + k0 + threadIdx.x] = s;
  }
}

// One block per token at a time: drows[pick_row[t, k]] = w[t, k] * dy[t]; dw[t, k] =
// <dy[t], rows[..]> (dw null: rows are not read; drows null: not written). Eight picks at a time:
// their rows are loaded before dy is used. 4096 x 7168 (bf16, top 8) takes 164 us, 93% of the copy
// bandwidth.
template <typename T>
__global__ void __launch_bounds__(256, 3)
    k_unsort_back_granules(const T* dy, const T* rows, const float* w, T* drows, float* dw,
                           const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(drows, a.row_pick, zero_limit(a), a.bytes,
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
      const bool any = (__ballot_sync(0xffffffffu, p.r >= 0) >> k & 0xffu) != 0;
      for (int v0 = 0; any && v0 < nvec; v0 += blockDim.x) {
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
    zero_rows(drows, a.row_pick, zero_limit(a), a.bytes,
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

// ------------------------------------------------------------------ rows of any size
// Rows that are no multiple of 16 bytes, in tensors that start on a 16-byte boundary: all accesses
// still go by aligned 16-byte granules. A row's granules are those that hold a byte of it; the
// first and last may hold bytes of its neighbours. Moving a row to one with another offset in its
// granules shifts two neighbouring granules against each other. Single-element accesses took 70 us
// to sort 4096 x 2047 (bf16, top 8); it takes 30 this way (2048: 27), unsort 50 (26) and its gradients
// 106 (51): there the shifts and the edges of eight rows are most of the instructions.

// Granule g of a tensor of `total` bytes; bytes outside the tensor read as zero.
__device__ __forceinline__ uint4 granule(const uint8_t* base, int64_t g, int64_t total) {
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if (g >= 0 && g * 16 + 16 <= total) {
    q = __ldcg(reinterpret_cast<const uint4*>(base) + g);
  } else if (g >= 0 && g * 16 < total) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    const int n = static_cast<int>(total - g * 16);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) w[i / 4] |= static_cast<uint32_t>(__ldcg(base + g * 16 + i)) << (8 * (i % 4));
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return q;
}

// The granule of a row's reader: rows before the tensor's last (`last` is uniform) have at least
// 512 bytes behind them, so only the lane's place in its own row needs a look.
__device__ __forceinline__ uint4 row_granule(const uint8_t* base, int64_t g, int64_t total, bool last,
                                             bool near) {
  if (last || g < 0) return granule(base, g, total);
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if (near) q = __ldcg(reinterpret_cast<const uint4*>(base) + g);
  return q;
}

// Bytes [by, by + 16) of the 32 bytes lo, hi (0 <= by < 16, the same in the whole warp).
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, int by) {
  const int bits = (by & 3) * 8;
  switch (by >> 2) {
    case 0:
      return make_uint4(__funnelshift_r(lo.x, lo.y, bits), __funnelshift_r(lo.y, lo.z, bits),
                        __funnelshift_r(lo.z, lo.w, bits), __funnelshift_r(lo.w, hi.x, bits));
    case 1:
      return make_uint4(__funnelshift_r(lo.y, lo.z, bits), __funnelshift_r(lo.z, lo.w, bits),
                        __funnelshift_r(lo.w, hi.x, bits), __funnelshift_r(hi.x, hi.y, bits));
    case 2:
      return make_uint4(__funnelshift_r(lo.z, lo.w, bits), __funnelshift_r(lo.w, hi.x, bits),
                        __funnelshift_r(hi.x, hi.y, bits), __funnelshift_r(hi.y, hi.z, bits));
    default:
      return make_uint4(__funnelshift_r(lo.w, hi.x, bits), __funnelshift_r(hi.x, hi.y, bits),
                        __funnelshift_r(hi.y, hi.z, bits), __funnelshift_r(hi.z, hi.w, bits));
  }
}

__device__ __forceinline__ uint4 shfl_granule(const uint4& q, int from) {
  return make_uint4(__shfl_sync(0xffffffffu, q.x, from), __shfl_sync(0xffffffffu, q.y, from),
                    __shfl_sync(0xffffffffu, q.z, from), __shfl_sync(0xffffffffu, q.w, from));
}

// A granule of a token's row and its two neighbours, for shifting it to any other offset. Lanes hold
// consecutive granules; only the outer lanes load their missing neighbour.
struct Granules3 {
  uint4 before, at, after;
};

__device__ __forceinline__ Granules3 load3(const uint8_t* base, int64_t g, int64_t total, bool last,
                                           bool near) {
  const int lane = threadIdx.x & 31;
  Granules3 t;
  t.at = row_granule(base, g, total, last, near);
  t.before = shfl_granule(t.at, lane - 1 < 0 ? 0 : lane - 1);
  t.after = shfl_granule(t.at, lane + 1 > 31 ? 31 : lane + 1);
  if (lane == 0) t.before = row_granule(base, g - 1, total, last, near);
  if (lane == 31) t.after = row_granule(base, g + 1, total, last, near);
  return t;
}

// The token's bytes for the granule of a row at the same index: `from` and `to` are the offsets of
// the two rows in their first granules.
__device__ __forceinline__ uint4 move(const Granules3& t, int from, int to) {
  const int by = from - to;  // > -16 and < 16
  return by >= 0 ? shifted(t.at, t.after, by) : shifted(t.before, t.at, by + 16);
}

// rows[pick_row[t, k]] = x[t], element size E.
template <int E>
__global__ void __launch_bounds__(256)
    k_sort_shifted(const uint8_t* x, uint8_t* rows, const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(rows, a.row_pick, zero_limit(a), a.bytes, blockIdx.x - a.copy_blocks,
              gridDim.x - a.copy_blocks);
    return;
  }
  const int64_t t = blockIdx.x / a.chunks;
  // whole warps take part in the exchange of neighbours
  const int64_t v = static_cast<int64_t>(blockIdx.x % a.chunks) * blockDim.x + threadIdx.x;
  const int64_t start = t * a.bytes;
  const int from = static_cast<int>(start & 15);
  const bool near = v * 16 < a.bytes + 32;
  const Granules3 g = load3(x, start / 16 + v, a.T * a.bytes, t == a.T - 1, near);
  const int32_t* pr = a.pick_row + t * a.K;
  for (int k0 = 0; k0 < a.K; k0 += 8) {
    int picks[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) picks[j] = k0 + j < a.K ? __ldcg(pr + k0 + j) : -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t r = picks[j];
      if (r < 0 || r >= a.R) continue;
      const int to = static_cast<int>((r * a.bytes) & 15);
      const int64_t lo = to - v * 16, hi = to + a.bytes - v * 16;  // the row's bytes in this granule
      if (hi <= 0) continue;
      store_part<E>(rows + (r * a.bytes - to) + v * 16, move(g, from, to),
                    static_cast<int>(lo < 0 ? 0 : lo), static_cast<int>(hi > 16 ? 16 : hi));
    }
  }
}

// As k_unsort_granules. Each of the eight rows is read at this token's offset: a granule and its
// neighbour, which the next lane has; the last lane of a warp only lends its granule, so a warp
// finishes 31.
template <typename T>
__global__ void __launch_bounds__(256, 3)
    k_unsort_shifted(const T* rows, const float* w, T* y, const RowsArgs a) {
  pdl_begin_in_order();
  const int64_t t = blockIdx.x / a.chunks;
  const int lane = threadIdx.x & 31;
  const int warp = (blockIdx.x % a.chunks) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t v = static_cast<int64_t>(warp) * 31 + lane;
  const uint8_t* in = reinterpret_cast<const uint8_t*>(rows);
  const int64_t start = t * a.bytes, total = a.R * a.bytes;
  const int to = static_cast<int>(start & 15);
  const bool near = v * 16 < a.bytes + 32;
  Gran<T> acc;
  zero(acc);
  for (int k0 = 0; k0 < a.K; k0 += 8) {
    const Picks p = load_picks(a, w, t, k0);
    uint4 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = make_uint4(0u, 0u, 0u, 0u);
      if (p.r[j] >= 0) {
        // this granule's bytes lie at row start + v * 16 - to
        const int64_t at = p.r[j] * a.bytes + v * 16 - to;
        q[j] = row_granule(in, at >= 0 ? at / 16 : -1, total, p.r[j] == a.R - 1, near);  // at > -16
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (p.r[j] < 0) continue;  // the same in the whole warp
      const uint4 next = shfl_granule(q[j], lane < 31 ? lane + 1 : 31);
      const int by = static_cast<int>((p.r[j] * a.bytes + 16 - to) & 15);
      acc = fma(gran_of<T>(shifted(q[j], next, by)), p.f[j], acc);
    }
  }
  const int64_t lo = to - v * 16, hi = to + a.bytes - v * 16;
  if (hi > 0 && lane < 31)
    store_part<sizeof(T)>(reinterpret_cast<uint8_t*>(y) + (start - to) + v * 16, words_of(acc),
                          static_cast<int>(lo < 0 ? 0 : lo), static_cast<int>(hi > 16 ? 16 : hi));
}

// As k_unsort_back_granules: dy is shifted to each row's offset; bytes of neighbouring rows count
// as zero in the sums.
template <typename T>
__global__ void __launch_bounds__(256, 3)
    k_unsort_back_shifted(const T* dy, const T* rows, const float* w, T* drows, float* dw,
                          const RowsArgs a) {
  pdl_begin_in_order();
  if (static_cast<int>(blockIdx.x) >= a.copy_blocks) {
    zero_rows(drows, a.row_pick, zero_limit(a), a.bytes, blockIdx.x - a.copy_blocks,
              gridDim.x - a.copy_blocks);
    return;
  }
  __shared__ float part[2][8][8];
  const int64_t t = blockIdx.x;
  const int64_t start = t * a.bytes, total = a.R * a.bytes;
  const int from = static_cast<int>(start & 15);
  const uint8_t* in = reinterpret_cast<const uint8_t*>(rows);
  // four picks at a time: eight take 120 registers (4096 x 2047: 115 us with eight, 106 with four)
  for (int k0 = 0; k0 < a.K; k0 += 4) {
    const Picks p = load_picks(a, w, t, k0);
    float2 dot2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) dot2[j] = make_float2(0.0f, 0.0f);
    const bool any = p.r[0] >= 0 || p.r[1] >= 0 || p.r[2] >= 0 || p.r[3] >= 0;
    for (int64_t v0 = 0; any && v0 < a.nvec; v0 += blockDim.x) {
      const int64_t v = v0 + threadIdx.x;
      uint4 q[4];
      if (dw) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[j] = make_uint4(0u, 0u, 0u, 0u);
          if (p.r[j] >= 0 && v < a.nvec)
            q[j] = row_granule(in, p.r[j] * a.bytes / 16 + v, total, p.r[j] == a.R - 1, true);
        }
      }
      const Granules3 g3 = load3(reinterpret_cast<const uint8_t*>(dy), start / 16 + v, a.T * a.bytes,
                                 t == a.T - 1, v < a.nvec);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (p.r[j] < 0) continue;
        const int to = static_cast<int>((p.r[j] * a.bytes) & 15);
        const int64_t lo64 = to - v * 16, hi64 = to + a.bytes - v * 16;
        if (hi64 <= 0) continue;
        const int lo = static_cast<int>(lo64 < 0 ? 0 : lo64), hi = static_cast<int>(hi64 > 16 ? 16 : hi64);
        Gran<T> g = gran_of<T>(move(g3, from, to));
        if (drows)
          store_part<sizeof(T)>(reinterpret_cast<uint8_t*>(drows) + (p.r[j] * a.bytes - to) + v * 16,
                                words_of(mul(g, p.f[j])), lo, hi);
        if (dw) {
          Gran<T> e = gran_of<T>(q[j]);
          if (lo > 0 || hi < 16) {
            constexpr int S = sizeof(T);
#pragma unroll
            for (int i = 0; i < Gran<T>::N; ++i) {
              if (2 * i * S < lo || 2 * i * S >= hi) g.p[i].x = e.p[i].x = 0.0f;
              if ((2 * i + 1) * S < lo || (2 * i + 1) * S >= hi) g.p[i].y = e.p[i].y = 0.0f;
            }
          }
#pragma unroll
          for (int i = 0; i < Gran<T>::N; ++i) dot2[j] = __ffma2_rn(g.p[i], e.p[i], dot2[j]);
        }
      }
    }
    if (dw) {
      float dot[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) dot[j] = p.r[j] >= 0 ? dot2[j].x + dot2[j].y : 0.0f;
      store_dots(dot, dw, t, k0, a.K, part[(k0 >> 2) & 1]);
    }
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

RowsArgs rows_args(const TokenOrder& o, int64_t nvec, int64_t bytes) {
  RowsArgs a{};
  a.bytes = bytes;
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
  const int64_t b = (R + 31) / 32;  // four rows per warp
  return static_cast<int>(b < 2 * num_sms ? b : 2 * num_sms);
}

template <typename U>
cudaError_t sort_rows(const void* x, void* rows, const TokenOrder& o, int64_t row_bytes,
                      int zero_tail, int num_sms, cudaStream_t s) {
  RowsArgs a = rows_args(o, row_bytes / static_cast<int64_t>(sizeof(U)), row_bytes);
  const RowGrid g = row_grid(o.T, a.nvec, sizeof(U) == 16 ? 1 : 4);
  a.chunks = g.chunks;
  a.copy_blocks = static_cast<int>(g.blocks);
  a.zero_tail = zero_tail;
  return launch_pdl(k_sort_rows<U>, dim3(static_cast<unsigned>(g.blocks + zero_blocks(o.R, num_sms))),
                    g.block, 0, s, static_cast<const U*>(x), static_cast<U*>(rows), a);
}

// Rows from 512 bytes on, of any size, go by granules (a warp holds 32 of one row); shorter rows
// that are no multiple of 16 bytes go by elements.
enum RowPath { kGranules, kShifted, kElements };

RowPath row_path(int64_t bytes, std::initializer_list<const void*> tensors) {
  for (const void* p : tensors)
    if (!aligned(p, 16)) return kElements;
  return bytes % 16 == 0 ? kGranules : bytes >= 512 ? kShifted : kElements;
}

// Blocks along the granules of a shifted row (at most two more than its size gives), of which a warp
// finishes per_warp.
RowGrid shifted_grid(int64_t T, int64_t bytes, int per_warp) {
  const int64_t warps = (bytes / 16 + 2 + per_warp - 1) / per_warp;
  RowGrid g{};
  g.chunks = static_cast<int>((warps + 7) / 8);
  g.block = dim3(static_cast<unsigned>((warps + g.chunks - 1) / g.chunks * 32), 1);
  g.blocks = T * g.chunks;
  return g;
}

template <int E>
cudaError_t sort_shifted(const void* x, void* rows, const TokenOrder& o, int64_t row_bytes,
                         int zero_tail, int num_sms, cudaStream_t s) {
  RowsArgs a = rows_args(o, 0, row_bytes);
  const RowGrid g = shifted_grid(o.T, row_bytes, 32);
  a.chunks = g.chunks;
  a.copy_blocks = static_cast<int>(g.blocks);
  a.zero_tail = zero_tail;
  return launch_pdl(k_sort_shifted<E>, dim3(static_cast<unsigned>(g.blocks + zero_blocks(o.R, num_sms))),
                    g.block, 0, s, static_cast<const uint8_t*>(x), static_cast<uint8_t*>(rows), a);
}

template <typename T>
cudaError_t unsort_rows(const void* rows, const float* w, void* y, const TokenOrder& o, int64_t H,
                        cudaStream_t s) {
  const int64_t bytes = H * static_cast<int64_t>(sizeof(T));
  const RowPath path = row_path(bytes, {rows, y});
  RowsArgs a = rows_args(o, path == kGranules ? H / kV<T> : H, bytes);
  const RowGrid g = path == kShifted ? shifted_grid(o.T, bytes, 31)
                                     : row_grid(o.T, a.nvec, path == kGranules ? 1 : 4);
  a.chunks = g.chunks;
  return launch_pdl(path == kGranules  ? k_unsort_granules<T>
                    : path == kShifted ? k_unsort_shifted<T>
                                       : k_unsort_elements<T>,
                    dim3(static_cast<unsigned>(g.blocks)), g.block, 0, s,
                    static_cast<const T*>(rows), w, static_cast<T*>(y), a);
}

template <typename T>
cudaError_t unsort_back(const void* dy, const void* rows, const float* w, void* drows, float* dw,
                        const TokenOrder& o, int64_t H, int num_sms, cudaStream_t s) {
  const int64_t bytes = H * static_cast<int64_t>(sizeof(T));
  const RowPath path = row_path(bytes, {dy, dw ? rows : nullptr, drows});
  RowsArgs a = rows_args(o, path == kGranules ? H / kV<T> : path == kShifted ? bytes / 16 + 2 : H, bytes);
  // passes of equal length along the row
  const int64_t passes = (a.nvec + 255) / 256;
  const int64_t threads = ((a.nvec + passes - 1) / passes + 31) / 32 * 32;
  a.copy_blocks = o.T;
  const int64_t most = static_cast<int64_t>(num_sms) * (768 / threads);
  if (path == kGranules && a.copy_blocks > most) a.copy_blocks = static_cast<int>(most);
  a.zero_tail = 1;
  const int64_t blocks = a.copy_blocks + (drows ? zero_blocks(o.R, num_sms) : 0);
  return launch_pdl(path == kGranules  ? k_unsort_back_granules<T>
                    : path == kShifted ? k_unsort_back_shifted<T>
                                       : k_unsort_back_elements<T>,
                    dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), 0, s,
                    static_cast<const T*>(dy), static_cast<const T*>(rows), w,
                    static_cast<T*>(drows), dw, a);
}

// One launch: a block up to kOrderSingle picks, a cluster up to kClusterPicks of few experts.
bool order_by_cluster(int64_t picks, int E) {
  return picks > kOrderSingle && picks <= kClusterPicks && E <= kClusterExperts;
}

}  // namespace

size_t order_scratch_bytes(int64_t picks, int E) {
  const OrderShape s = order_shape(picks, E);
  if (order_by_cluster(picks, E)) return 0;
  return s.blocks > 1 ? static_cast<size_t>(s.blocks) * E * 4 : 0;
}

cudaError_t launch_order(const int32_t* ids, const TokenOrder& o, int offset, int align,
                         int32_t* expert_base, int32_t* row_pick, int32_t* pick_row,
                         int32_t* hist, cudaStream_t s) {
  const OrderShape sh = order_shape(static_cast<int64_t>(o.T) * o.K, o.E);
  if (order_by_cluster(sh.picks, o.E)) {
    const int64_t part = (sh.picks + kClusterCtas - 1) / kClusterCtas;
    const int chunk = static_cast<int>((part + 1023) / 1024 * 1024);
    return launch_pdl_cluster(k_order_cluster, dim3(kClusterCtas), dim3(1024),
                              static_cast<size_t>(34) * o.E * 4, s, kClusterCtas, ids, sh.picks,
                              chunk, o.E, offset, align, o.R, expert_base, row_pick, pick_row);
  }
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
  const bool shift = row_path(row_bytes, {x, rows}) == kShifted;
  if (fits(16)) return sort_rows<uint4>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  if (fits(4))
    return shift ? sort_shifted<4>(x, rows, o, row_bytes, zero_tail, num_sms, s)
                 : sort_rows<uint32_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  if (fits(2))
    return shift ? sort_shifted<2>(x, rows, o, row_bytes, zero_tail, num_sms, s)
                 : sort_rows<uint16_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
  return shift ? sort_shifted<1>(x, rows, o, row_bytes, zero_tail, num_sms, s)
               : sort_rows<uint8_t>(x, rows, o, row_bytes, zero_tail, num_sms, s);
}

cudaError_t launch_unsort_rows(const void* rows, const float* w, void* y, int dtype,
                               const TokenOrder& o, int64_t H, cudaStream_t s) {
  switch (dtype) {
    case FMOE_DTYPE_F32:
      return unsort_rows<float>(rows, w, y, o, H, s);
    case FMOE_DTYPE_BF16:
      return unsort_rows<__nv_bfloat16>(rows, w, y, o, H, s);
    default:
      return unsort_rows<__half>(rows, w, y, o, H, s);
  }
}

cudaError_t launch_unsort_back(const void* dy, const void* rows, const float* w, void* drows,
                               float* dw, int dtype, const TokenOrder& o, int64_t H, int num_sms,
                               cudaStream_t s) {
  switch (dtype) {
    case FMOE_DTYPE_F32:
      return unsort_back<float>(dy, rows, w, drows, dw, o, H, num_sms, s);
    case FMOE_DTYPE_BF16:
      return unsort_back<__nv_bfloat16>(dy, rows, w, drows, dw, o, H, num_sms, s);
    default:
      return unsort_back<__half>(dy, rows, w, drows, dw, o, H, num_sms, s);
  }
}

}  // namespace fmoe
