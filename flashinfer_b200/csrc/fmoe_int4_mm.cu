// fmoe_int4_mm.cu -- products of 16-bit activations with 4-bit weights on the tensor cores, for one
// matrix or one per expert, many tokens (fmoe_int4.cu has the format and the kernel for few).
//
// The weight rows are the M side of the MMA (128 per tile) and the tokens its N side (up to BN per tile,
// the instruction's N chosen per tile), as in the int8 products. Eight warps widen the weights: 16 bytes of
// a row at a time, loaded D stages ahead into registers, become 32 16-bit values in the 128-byte swizzled
// rows that the MMA reads, while a TMA warp brings the tokens' rows; the widened matrix never exists in
// global memory. The widening of a tile's K block is the same work however many tokens the tile has:
// with 256 it is hidden behind the MMAs, with few it is what the tile costs.
//
// A weight is scale * (q - zero) rounded once to the activations' type, since the MMA sums over groups: off
// by at most half a step of that type, as each output is. (A sum per group, scaled in fp32 as the kernel for
// few tokens does it, would have to take the accumulator out of tensor memory once per group.) For fp16 the
// scales of a row are moved by a power of two, such that the largest is in [2^9, 2^10), and the output back:
// small scales then lose nothing to fp16's range, and a weight cannot overflow. An fp32 scale enters as the
// sum of two 16-bit values.
#include <cuda.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "fmoe_int4.cuh"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

constexpr int kI4Threads = 640;   // warp 0 loads tokens, 1 issues MMAs, 4..11 widen, 12..19 store
constexpr int kI4Widen0 = 4, kI4WidenWarps = 8;
constexpr int kI4Epi0 = 12, kI4EpiWarps = 8;
constexpr int kI4Rows = 128;      // weight rows per tile
constexpr int kI4KB = 64;         // values of a K block: one 128-byte row
constexpr int kI4MaxStages = 8;
constexpr int kI4Invs = 16;       // tiles that the widening may be ahead of the stores, rounded up

// SUB: K blocks per stage. D: stages whose weights are on their way in registers.
template <int BN>
struct I4Cfg {
  static constexpr int SUB = BN == 64 ? 2 : 1;
  static constexpr int D = 4;
  static constexpr int BLOCK_A = kI4Rows * 128, BLOCK_B = BN * 128;
  static constexpr int STAGE = SUB * (BLOCK_A + BLOCK_B);
  static constexpr int NS = 192 * 1024 / STAGE;
  static constexpr int BOX = BN == 64 ? 32 : 64;  // token rows per TMA box
  static constexpr int COLS = 2 * BN;
  static_assert(NS <= kI4MaxStages && NS + 2 < kI4Invs, "barrier arrays, factors in flight");
};

struct alignas(16) I4Tail {
  uint64_t bfull[kI4MaxStages];  // tokens: the TMA copies
  uint64_t afull[kI4MaxStages];  // weights: one arrival per widening warp
  uint64_t empty[kI4MaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint64_t never;
  uint32_t tmem_base;
  int abort_flag;
  int tiles;
  int live;
  int last_issue[kI4MaxStages];
  alignas(16) float inv[kI4Invs][kI4Rows];  // fp16: what an output is multiplied with
  int ebase[kMaxLocalExperts + 1];
  int etile[kMaxLocalExperts + 1];          // token tiles before expert e
};

template <int BN>
constexpr size_t i4_smem_bytes() {
  return static_cast<size_t>(I4Cfg<BN>::NS) * I4Cfg<BN>::STAGE + sizeof(I4Tail) + 1024;
}
static_assert(i4_smem_bytes<64>() <= 227 * 1024 && i4_smem_bytes<128>() <= 227 * 1024 &&
                  i4_smem_bytes<256>() <= 227 * 1024,
              "shared memory per CTA");

struct I4Run {
  int nkb, S;                 // K blocks, and the parts that K is split into
  uint32_t group_magic;       // about 2^32 / (group / 32), see group_of
  unsigned long long wait_ns; // limit of every wait
  int inject;                 // failure-path test: the MMA warp first waits for what never comes
};

// D[tmem] (+)= A[smem] * B[smem]^T, 16-bit operands of one type, fp32 sums.
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: D fp32, A and B bf16 (1) or fp16 (0), both K-major.
template <typename T>
__device__ __forceinline__ uint32_t idesc_16(int M, int N) {
  constexpr uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Set by a product whose bounded wait ran out, until take_int4_status takes it to g_int4_taken.
__device__ int32_t g_int4_status;
__device__ int32_t g_int4_taken;

// Reads and clears in one step: a product on another stream may set the word at any time.
__global__ void k_take_int4_status() { g_int4_taken = atomicExch(&g_int4_status, 0); }

__device__ __forceinline__ void i4_abort(I4Tail* t) {
  *reinterpret_cast<volatile int*>(&t->abort_flag) = 1;
  atomicOr(&g_int4_status, FMOE_STATUS_TIMEOUT_INT4);
}

// A unit of work: a part of K of a tile. Order: expert, weight tile, token tile, part of K (fastest), so
// that CTAs that run side by side share weight tiles. An expert's tokens are cut into equal tiles of at
// most BN.
struct I4Unit {
  int e, n0;         // expert, first weight row (channel)
  int64_t row0;      // first token row
  int rows, cols;    // tokens in the tile, and the MMA's N (a multiple of 16)
  int part, kb0, kb1;
};

template <int BN>
__device__ __forceinline__ I4Unit decode_unit(int unit, int NT, const I4Tail* t, int E, const I4Run& r) {
  I4Unit u;
  const int tile = unit / r.S;
  u.part = unit - tile * r.S;
  int lo = 0, hi = E - 1;
  while (lo < hi) {  // first expert e with tile < etile[e + 1] * NT
    const int mid = (lo + hi) >> 1;
    if (tile < t->etile[mid + 1] * NT)
      hi = mid;
    else
      lo = mid + 1;
  }
  const int mt = t->etile[lo + 1] - t->etile[lo];
  const int local = tile - t->etile[lo] * NT;
  const int n = local / mt;
  const int m = local - n * mt;
  const int count = t->ebase[lo + 1] - t->ebase[lo];
  // at most BN: count <= mt * BN, and BN is a multiple of 16
  const int per = ((count + mt - 1) / mt + 15) / 16 * 16;
  u.e = lo;
  u.n0 = n * kI4Rows;
  u.row0 = t->ebase[lo] + static_cast<int64_t>(m) * per;
  u.rows = max(0, min(per, count - m * per));
  u.cols = max(16, (u.rows + 15) / 16 * 16);
  u.kb0 = u.part * r.nkb / r.S;
  u.kb1 = (u.part + 1) * r.nkb / r.S;
  return u;
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
  uint32_t v[4];
  widen8<T>(q, zp, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F32S)
      v[i] = fma2(type, hi, v[i], mul2(type, lo, v[i]));
    else
      v[i] = mul2(type, hi, v[i]);
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                    __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
}

// The epilogue of one warp: its 32 channels (one per lane) of the tile's columns c0, c0 + c_step, ...; out
// is the element of the tile's first token at this warp's first channel. PAIRS (outputs at 4-byte
// boundaries): neighbouring lanes exchange halves of their tokens, so that a lane stores two channels at
// once. O float: the partial sums of a split product.
template <typename O, bool PAIRS>
__device__ __forceinline__ void store_tile(uint32_t taddr, int c0, int c_step, int cols, int rows,
                                           float factor, float bias, O* out, int N, int live) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1;
  O* mine = out + (PAIRS ? lane & ~1 : lane);
  const bool writes = lane < live;  // N is even with PAIRS, so both channels of a pair exist
  for (int c = c0; c < cols; c += c_step) {
    __syncwarp();
    float v[16];
    tmem_ld_32x32b_x16(taddr + c, v);
    tmem_ld_wait16(v);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = fmaf(v[i], factor, bias);
    if constexpr (PAIRS) {
      uint32_t w[8];  // even lanes take tokens c .. c + 7, odd lanes c + 8 .. c + 15
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 8], 1);
        w[i] = odd ? pack2(static_cast<O*>(nullptr), other, v[i + 8])
                   : pack2(static_cast<O*>(nullptr), v[i], other);
      }
      if (writes) {
        O* p = mine + static_cast<int64_t>(c + (odd ? 8 : 0)) * N;
        const int left = rows - c - (odd ? 8 : 0);
#pragma unroll
        for (int i = 0; i < 8; ++i, p += N)
          if (i < left) *reinterpret_cast<uint32_t*>(p) = w[i];
      }
    } else if (writes) {
      O* p = mine + static_cast<int64_t>(c) * N;
      const int left = rows - c;
#pragma unroll
      for (int i = 0; i < 16; ++i, p += N)
        if (i < left) from_f32(v[i], p);
    }
  }
  __syncwarp();
}

template <typename T, int BN, bool F32S>
__global__ void __launch_bounds__(kI4Threads, 1)
    k_int4_mm(const __grid_constant__ CUtensorMap tm_x, const I4Args args, const I4Run run) {
  using C = I4Cfg<BN>;
  constexpr int NS = C::NS, SUB = C::SUB, D = C::D;
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  I4Tail* tail = reinterpret_cast<I4Tail*>(smem + NS * C::STAGE);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = args.E;
  const int NT = (args.N + kI4Rows - 1) / kI4Rows;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&tail->bfull[s], 1);
      mbar_init(&tail->afull[s], kI4WidenWarps);
      mbar_init(&tail->empty[s], 1);
      tail->last_issue[s] = -1;
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tail->tfull[b], 1);
      mbar_init(&tail->tempty[b], kI4EpiWarps * 32);
    }
    mbar_init(&tail->drain, 1);
    mbar_init(&tail->never, 1);
    tail->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, C::COLS);
    tmem_relinquish();
  }
  // everything this kernel reads may have been written by the previous grid
  pdl_begin_in_order();
  if (warp == 0) {
    // the bases as a running maximum, token tiles per expert and their running sum
    int most = 0, tiles = 0;
    for (int e0 = 0; e0 <= E; e0 += 32) {
      const int e = e0 + lane;
      int64_t b = 0;
      if (e <= E) b = args.expert_base ? __ldcg(args.expert_base + e) : e == 0 ? 0 : args.M;
      int v = max(most, static_cast<int>(b < 0 ? 0 : b > args.M ? args.M : b));
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, up);
      }
      // tiles of the expert before base e
      const int before = __shfl_up_sync(0xffffffffu, v, 1);
      int mt = e == 0 || e > E ? 0 : (v - (lane == 0 ? most : before) + BN - 1) / BN;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, mt, o);
        if (lane >= o) mt += up;
      }
      if (e <= E) {
        tail->ebase[e] = v;
        tail->etile[e] = tiles + mt;
      }
      most = __shfl_sync(0xffffffffu, v, 31);
      tiles += __shfl_sync(0xffffffffu, mt, 31);
    }
    __syncwarp();
    if (lane == 0) {
      tail->tiles = tail->etile[E] * NT;
      tail->live = tail->ebase[E];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  const int units = tail->tiles * run.S;

  if (warp == 0) {
    // ---------------------------------------------------------------- tokens
    if (elect_one()) {
      const uint64_t pol = policy_evict_last();
      int it = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
        const I4Unit u = decode_unit<BN>(unit, NT, tail, E, run);
        const int boxes = (u.cols + C::BOX - 1) / C::BOX;
        for (int kb = u.kb0; kb < u.kb1; kb += SUB, ++it) {
          const int s = it % NS, r = it / NS;
          if (r > 0 && !parked_wait(&tail->empty[s], (r & 1) ^ 1, abort_flag, run.wait_ns)) {
            i4_abort(tail);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::STAGE + SUB * C::BLOCK_A;
          const int blocks = min(SUB, u.kb1 - kb);
          mbar_arrive_expect_tx(&tail->bfull[s], blocks * boxes * C::BOX * 128);
          for (int j = 0; j < blocks; ++j, st += C::BLOCK_B)
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(st + b * C::BOX * 128, &tm_x, &tail->bfull[s], (kb + j) * 128,
                          static_cast<int>(u.row0) + b * C::BOX, pol);
          tail->last_issue[s] = r;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    if (elect_one()) {
      int it = 0, n = 0;
      bool ok = run.inject == 0 || parked_wait(&tail->never, 0, abort_flag, run.wait_ns);
      for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x, ++n) {
        const I4Unit u = decode_unit<BN>(unit, NT, tail, E, run);
        const uint32_t idesc = idesc_16<T>(kI4Rows, u.cols);
        const int b = n & 1, rb = n >> 1;
        const uint32_t d = tmem + b * BN;
        if (rb > 0 && !parked_wait(&tail->tempty[b], (rb & 1) ^ 1, abort_flag, run.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t more = 0;  // the unit's first MMA overwrites
        for (int kb = u.kb0; kb < u.kb1; kb += SUB, ++it) {
          const int s = it % NS, r = it / NS;
          if (!parked_wait(&tail->afull[s], r & 1, abort_flag, run.wait_ns) ||
              !parked_wait(&tail->bfull[s], r & 1, abort_flag, run.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t sa = smem_u32(smem + s * C::STAGE), sb = sa + SUB * C::BLOCK_A;
          for (int left = min(SUB, u.kb1 - kb); left > 0; --left, sa += C::BLOCK_A, sb += C::BLOCK_B) {
            const uint64_t wd = smem_desc_k128(sa), xd = smem_desc_k128(sb);
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 16 values of K each
              mma_f16(d, wd + 2 * j, xd + 2 * j, idesc, more);
              more = 1u;
            }
          }
          mma_commit(&tail->empty[s]);
        }
        if (ok) mma_commit(&tail->tfull[b]);
      }
      if (!ok) i4_abort(tail);
      mma_commit(&tail->drain);
      (void)mbar_wait(&tail->drain, 0);
    }
  } else if (warp >= kI4Widen0 && warp < kI4Widen0 + kI4WidenWarps) {
    // ---------------------------------------------------------------- widening
    // Two threads per weight row, each with 32 of a block's 64 values.
    T* type = nullptr;
    const int tid = threadIdx.x - kI4Widen0 * 32;
    const int r = tid >> 1, h = tid & 1;
    const uint32_t swz = static_cast<uint32_t>(r & 7);
    const auto group_of = [&](int k) {
      const uint32_t k32 = static_cast<uint32_t>(k >> 5);
      return static_cast<int>(run.group_magic == 0 ? k32 : __umulhi(k32, run.group_magic));
    };
    struct Cursor {
      int unit, kb, kb0, kb1;
      int64_t wrow;
    };
    const auto open = [&](Cursor& c) {
      if (c.unit >= units) return;
      const I4Unit u = decode_unit<BN>(c.unit, NT, tail, E, run);
      c.kb = c.kb0 = u.kb0;
      c.kb1 = u.kb1;
      // rows behind the last are the last, and are not stored
      c.wrow = static_cast<int64_t>(u.e) * args.N + min(u.n0 + r, args.N - 1);
    };
    const auto advance = [&](Cursor& c) {
      c.kb += SUB;
      if (c.kb >= c.kb1) {
        c.unit += gridDim.x;
        open(c);
      }
    };
    uint4 q[D][SUB];
    uint32_t sc[D][SUB], zp[D][SUB];
    const auto fetch = [&](Cursor& c, uint4 (&to)[SUB], uint32_t (&ts)[SUB], uint32_t (&tz)[SUB]) {
      if (c.unit >= units) return;
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        const int k = (c.kb + j) * kI4KB + 32 * h;
        if (c.kb + j < c.kb1 && k < args.K) {
          to[j] = __ldcg(reinterpret_cast<const uint4*>(args.w + c.wrow * (args.K / 2) + k / 2));
          const int64_t at = c.wrow * args.groups + group_of(k);
          ts[j] = F32S ? __ldcg(static_cast<const uint32_t*>(args.scale) + at)
                       : static_cast<uint32_t>(__ldcg(static_cast<const uint16_t*>(args.scale) + at));
          tz[j] = args.zero ? __ldcg(args.zero + at) : 8u;
        }
      }
      advance(c);
    };
    Cursor ahead{static_cast<int>(blockIdx.x), 0, 0, 0, 0};
    open(ahead);
    Cursor now = ahead;
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(ahead, q[d], sc[d], zp[d]);
    int it = 0, n = 0;
    bool ok = true;
    float factor = 1.0f;
    while (now.unit < units && ok) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (now.unit >= units || !ok) break;
        if (HALF && now.kb == now.kb0) {
          // the largest scale of the unit's groups to [2^9, 2^10); the row's two threads share the search
          const int g0 = group_of(now.kb0 * kI4KB), g1 = group_of(min(now.kb1 * kI4KB, args.K) - 1);
          float most = 0.0f;
          for (int i = g0 + h; i <= g1; i += 2)
            most = fmaxf(most, fabsf(scale_at(args.scale, F32S, type, now.wrow * args.groups + i)));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127 - 9;
          if (most == 0.0f || ex > 110) ex = 0;  // nothing, or infinite
          if (ex < -120) ex = -120;
          factor = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
          if (h == 0) tail->inv[n % kI4Invs][r] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
        }
        const int s = it % NS, round = it / NS;
        if (round > 0)
          ok = __all_sync(0xffffffffu, parked_wait(&tail->empty[s], (round & 1) ^ 1, abort_flag,
                                                   run.wait_ns));
        if (!ok) {
          if (lane == 0) i4_abort(tail);
          break;
        }
        uint8_t* st = smem + s * C::STAGE + r * 128;
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
          if (now.kb + j >= now.kb1) break;
          uint4* row = reinterpret_cast<uint4*>(st + j * C::BLOCK_A);
          if ((now.kb + j) * kI4KB + 32 * h < args.K) {
            uint32_t hi, lo = 0;
            if constexpr (F32S || HALF) {
              float f = F32S ? __uint_as_float(sc[d][j])
                             : __half2float(__ushort_as_half(static_cast<uint16_t>(sc[d][j])));
              f *= factor;
              T a;
              from_f32(f, &a);
              hi = pack2(type, to_f32(a), to_f32(a));
              // what the rounding left; nothing of an infinite scale
              const float rest = fabsf(f) < INFINITY && fabsf(to_f32(a)) < INFINITY ? f - to_f32(a) : 0.0f;
              if (F32S) lo = pack2(type, rest, rest);
            } else {
              hi = sc[d][j] * 0x00010001u;
            }
            const uint32_t z = nibble_base(type) + (zp[d][j] & 15u) * 0x00010001u;
            const uint32_t w[4] = {q[d][j].x, q[d][j].y, q[d][j].z, q[d][j].w};
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) row[(4 * h + c) ^ swz] = weights8<T, F32S>(w[c], z, hi, lo);
          } else {
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) row[(4 * h + c) ^ swz] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fetch(ahead, q[d], sc[d], zp[d]);
        fence_async_smem();  // the MMAs read through the asynchronous proxy
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->afull[s]);
        ++it;
        const int was = now.unit;
        advance(now);
        if (now.unit != was) ++n;
      }
    }
  } else if (warp >= kI4Epi0) {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;              // TMEM lanes of this warp
    const int g = (warp - kI4Epi0) >> 2;       // which 16 of 32 columns
    if (args.zero_tail) {                      // rows of no expert
      const int64_t tid = static_cast<int64_t>(blockIdx.x) * (kI4EpiWarps * 32) + threadIdx.x - kI4Epi0 * 32;
      const int64_t threads = static_cast<int64_t>(gridDim.x) * (kI4EpiWarps * 32);
      zero_rows16(args.out, args.N, 0, tail->ebase[0], tid, threads);
      zero_rows16(args.out, args.N, tail->live, args.M, tid, threads);
    }
    const bool pairs = (args.N & 1) == 0 && (reinterpret_cast<uintptr_t>(args.out) & 3u) == 0;
    int n = 0;
    bool ok = true;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++n) {
      const I4Unit u = decode_unit<BN>(unit, NT, tail, E, run);
      const int b = n & 1, rb = n >> 1;
      const int ch = u.n0 + quarter * 32 + lane;
      const float bias = run.S == 1 && args.bias && ch < args.N ? __ldcg(args.bias + ch) : 0.0f;
      if (ok) ok = __all_sync(0xffffffffu, parked_wait(&tail->tfull[b], rb & 1, abort_flag, run.wait_ns));
      if (!ok) {
        if (lane == 0) i4_abort(tail);
        break;
      }
      tc_fence_after();
      const float factor = HALF ? tail->inv[n % kI4Invs][quarter * 32 + lane] : 1.0f;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * BN;
      const int n0 = u.n0 + quarter * 32, live = args.N - n0;
      const int64_t at = u.row0 * args.N + n0;
      if (run.S > 1)
        store_tile<float, false>(taddr, g * 16, 32, u.cols, u.rows, factor, 0.0f,
                                 args.part + static_cast<int64_t>(u.part) * args.M * args.N + at, args.N,
                                 live);
      else if (pairs)
        store_tile<T, true>(taddr, g * 16, 32, u.cols, u.rows, factor, bias,
                            static_cast<T*>(args.out) + at, args.N, live);
      else
        store_tile<T, false>(taddr, g * 16, 32, u.cols, u.rows, factor, bias,
                             static_cast<T*>(args.out) + at, args.N, live);
      tc_fence_before();
      mbar_arrive(&tail->tempty[b]);
    }
  }

  tc_fence_before();
  __syncthreads();
  // Never leave a bulk copy in flight into shared memory that is about to be released: after an abort, wait
  // for each stage's latest issued round (without one the MMA warp has seen them all).
  if (threadIdx.x == 0 && *abort_flag) {
    for (int s = 0; s < NS; ++s)
      if (tail->last_issue[s] >= 0) (void)mbar_wait(&tail->bfull[s], tail->last_issue[s] & 1);
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// The parts' sums of a split product, added in order, with the bias: rows that have an expert, four channels
// per thread (V = 4) or one.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_int4_finish(const I4Args a, int S) {
  pdl_begin_in_order();
  int64_t first = 0, end = a.M, none;
  if (a.expert_base) {
    expert_rows(a.expert_base, 0, a.M, &first, &none);
    expert_rows(a.expert_base, a.E - 1, a.M, &none, &end);
  }
  const int64_t per = a.N / V, all = a.M * a.N;
  const int64_t last = end * per;
  for (int64_t i = first * per + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < last;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    for (int s = 0; s < S; ++s) {
      const float* p = a.part + s * all + i * V;
      if constexpr (V == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
        sum[0] += v.x;
        sum[1] += v.y;
        sum[2] += v.z;
        sum[3] += v.w;
      } else {
        sum[0] += __ldcg(p);
      }
    }
    const int ch = static_cast<int>(i % per) * V;
    T* out = static_cast<T*>(a.out) + i * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (a.bias) sum[j] += __ldcg(a.bias + ch + j);
      if (V == 1) from_f32(sum[j], out);
    }
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2(static_cast<T*>(nullptr), sum[0], sum[1]),
                                                  pack2(static_cast<T*>(nullptr), sum[2], sum[3]));
  }
}

// ------------------------------------------------------------------ launches
template <typename T, int BN, bool F32S>
cudaError_t launch_mm(const Int4Product& p, const I4Args& a, const Int4Plan& plan, int sms,
                      cudaStream_t s) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(k_int4_mm<T, BN, F32S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(i4_smem_bytes<BN>()));
    if (e != cudaSuccess) return e;
    done[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tm_x;
  const uint64_t row = static_cast<uint64_t>(p.K) * 2;
  if (!tensor_map_u8(&tm_x, p.x, row, p.M, row, 128, I4Cfg<BN>::BOX)) return cudaErrorInvalidValue;
  I4Run r{};
  r.nkb = (p.K + kI4KB - 1) / kI4KB;
  r.S = plan.S;
  const uint32_t g32 = static_cast<uint32_t>(p.group / 32);
  // (k / 32) (2^32 / g32 + 1) >> 32 is k / 32 / g32: k / 32 <= 4096 makes its error less than 2^-20, and
  // g32 <= 4096. 0: a group is 32 values; 1: the row is one group
  r.group_magic = g32 == 1 ? 0u : g32 > 4096 ? 1u : static_cast<uint32_t>((1ull << 32) / g32 + 1);
  r.wait_ns = p.wait_ns != 0 ? p.wait_ns : FMOE_WAIT_NS;
  r.inject = p.wait_ns != 0;
  const int64_t used = p.M < p.E ? p.M : p.E;
  const int64_t most = (p.expert_base ? p.M / BN + used : (p.M + BN - 1) / BN) *
                       ((p.N + kI4Rows - 1) / kI4Rows) * plan.S;
  const int grid = static_cast<int>(most < sms ? most : sms);
  cudaError_t e = launch_pdl(k_int4_mm<T, BN, F32S>, dim3(grid), dim3(kI4Threads), i4_smem_bytes<BN>(), s,
                             tm_x, a, r);
  if (e != cudaSuccess || plan.S == 1) return e;
  const bool four = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7u) == 0;
  const int64_t blocks = (p.M * p.N / (four ? 4 : 1) + 255) / 256;
  const dim3 fgrid(static_cast<unsigned>(blocks < 8 * sms ? blocks : 8 * sms));
  if (four) return launch_pdl(k_int4_finish<T, 4>, fgrid, dim3(256), 0, s, a, plan.S);
  return launch_pdl(k_int4_finish<T, 1>, fgrid, dim3(256), 0, s, a, plan.S);
}

template <typename T, bool F32S>
cudaError_t launch_mm(const Int4Product& p, const I4Args& a, const Int4Plan& plan, int sms,
                      cudaStream_t s) {
  switch (plan.bn) {
    case 64:
      return launch_mm<T, 64, F32S>(p, a, plan, sms, s);
    case 128:
      return launch_mm<T, 128, F32S>(p, a, plan, sms, s);
    default:
      return launch_mm<T, 256, F32S>(p, a, plan, sms, s);
  }
}

}  // namespace

cudaError_t launch_int4_mm(const Int4Product& p, const I4Args& a, const Int4Plan& plan, int sms,
                           cudaStream_t s) {
  if (p.dtype == FMOE_DTYPE_BF16)
    return a.scale_f32 ? launch_mm<__nv_bfloat16, true>(p, a, plan, sms, s)
                       : launch_mm<__nv_bfloat16, false>(p, a, plan, sms, s);
  return a.scale_f32 ? launch_mm<__half, true>(p, a, plan, sms, s)
                     : launch_mm<__half, false>(p, a, plan, sms, s);
}

cudaError_t take_int4_status(int32_t* status, cudaStream_t s) {
  static std::mutex one_at_a_time;  // g_int4_taken is one call's until it has been copied out
  const std::lock_guard<std::mutex> hold(one_at_a_time);
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_int4_taken);
  if (e != cudaSuccess) return e;
  k_take_int4_status<<<1, 1, 0, s>>>();
  e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, sizeof(int32_t), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e;
}

}  // namespace fmoe
