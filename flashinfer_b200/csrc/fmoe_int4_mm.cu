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
// a row of small scales then loses nothing to fp16's range, and a weight cannot overflow. What is left of the
// range is 2^-24, fp16's last step: a scale and a product that end in it are off by 2^-25, a weight by 16 or 17 of
// those, 2^-29 of the row's largest scale. An fp32 scale enters as the sum of two 16-bit values.
#include <cuda.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "fmoe_int4.cuh"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

constexpr int kI4Threads = 640;   // warp 0 loads tokens, 1 issues MMAs, 4..15 widen, 16..19 store
constexpr int kI4Widen0 = 4;
constexpr int kI4Groups = 3;      // of four widening warps, one thread per weight row
constexpr int kI4Epi0 = kI4Widen0 + 4 * kI4Groups, kI4EpiWarps = 4;
constexpr int kI4Rows = 128;      // weight rows per tile
constexpr int kI4KB = 64;         // values of a K block: one 128-byte row
constexpr int kI4MaxStages = 8;
constexpr int kI4Ahead = 2;       // blocks whose weights are on their way in a thread's registers
constexpr int kI4Invs = 16;       // tiles that the widening may be ahead of the stores, rounded up

template <int BN>
struct I4Cfg {
  static constexpr int BLOCK_A = kI4Rows * 128, BLOCK_B = BN * 128;
  static constexpr int STAGE = BLOCK_A + BLOCK_B;
  static constexpr int NS = 192 * 1024 / STAGE;
  static constexpr int BOX = BN == 64 ? 32 : 64;  // token rows per TMA box
  static constexpr int COLS = 2 * BN;
  static_assert(NS > kI4Groups && NS <= kI4MaxStages && NS + 2 < kI4Invs, "barrier arrays, factors in flight");
};

struct alignas(16) I4Tail {
  uint64_t bfull[kI4MaxStages];  // tokens: the TMA copies
  uint64_t afull[kI4MaxStages];  // weights: one arrival per warp of a widening group
  uint64_t empty[kI4MaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint64_t never;
  uint32_t tmem_base;
  int abort_flag;
  int tiles;
  int live;
  int last_issue[kI4MaxStages];  // the latest round of copies that this CTA issued into the stage,
  int last_bytes[kI4MaxStages];  // -1 for none, and (pairs) its bytes
  int gave_up;                   // pairs: set in both CTAs after the leader's abort
  alignas(16) float inv[kI4Invs][kI4Rows];  // fp16: what an output is multiplied with
  int ebase[kMaxLocalExperts + 1];
  int etile[kMaxLocalExperts + 1];          // token tiles before expert e
};

template <int BN>
constexpr size_t i4_smem_bytes() {
  return static_cast<size_t>(I4Cfg<BN>::NS) * I4Cfg<BN>::STAGE + sizeof(I4Tail) + 1024;
}
static_assert(i4_smem_bytes<64>() <= 227 * 1024 && i4_smem_bytes<128>() <= 227 * 1024,
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

__device__ __forceinline__ void st_shared_v4(uint32_t to, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
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

// The bases as a running maximum, the token tiles (of bn) per expert and their running sum. By one warp.
__device__ __forceinline__ void plan_tiles(const I4Args& args, int bn, int NT, I4Tail* tail) {
  const int lane = threadIdx.x & 31, E = args.E;
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
    int mt = e == 0 || e > E ? 0 : (v - (lane == 0 ? most : before) + bn - 1) / bn;
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

// A unit of work: a part of K of a tile. Order: expert, weight tile, token tile, part of K (fastest), so
// that CTAs that run side by side share weight tiles. An expert's tokens are cut into equal tiles of at
// most BN.
struct I4Unit {
  int e, n0;         // expert, first weight row (channel)
  int64_t row0;      // first token row
  int rows, cols;    // tokens in the tile, and the MMA's N
  int part, kb0, kb1;
};

// STEP: what a tile's tokens are a multiple of. ROWS: its weight rows.
template <int STEP, int ROWS>
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
  // at most BN: count <= mt * BN, and BN is a multiple of STEP
  const int per = ((count + mt - 1) / mt + STEP - 1) / STEP * STEP;
  u.e = lo;
  u.n0 = n * ROWS;
  u.row0 = t->ebase[lo] + static_cast<int64_t>(m) * per;
  u.rows = max(0, min(per, count - m * per));
  u.cols = max(STEP, (u.rows + STEP - 1) / STEP * STEP);
  u.kb0 = u.part * r.nkb / r.S;
  u.kb1 = (u.part + 1) * r.nkb / r.S;
  return u;
}

// The largest absolute value of the scales `at` + g0 .. `at` + g1 of a row of fp16 weights, or of whole 16-byte
// pieces around them where rows have such (a bound of other groups' scales too does as well): one load per
// scale, every lane in a row of its own, took a third of 37 x 2047 x 7168 in groups of 32. NaN counts as
// infinite.
template <bool F32S>
__device__ __forceinline__ float largest_scale(const I4Args& args, int64_t at, int g0, int g1) {
  constexpr int SB = F32S ? 4 : 2, PER = 16 / SB;
  const uint8_t* row = static_cast<const uint8_t*>(args.scale) + at * SB;
  uint32_t m = 0;
  if (args.groups % PER == 0 && (reinterpret_cast<uintptr_t>(args.scale) & 15u) == 0) {
#pragma unroll 4
    for (int c = g0 / PER; c <= g1 / PER; ++c) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + c * 16);
      if constexpr (F32S)
        m = max(m, max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu)));
      else
        m = __vmaxu2(__vmaxu2(m, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)),
                     __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    }
  } else {
#pragma unroll 8
    for (int g = g0; g <= g1; ++g)
      m = max(m, F32S ? reinterpret_cast<const uint32_t*>(row)[g] & 0x7fffffffu
                      : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[g]) & 0x7fffu);
  }
  if constexpr (F32S) return __uint_as_float(m);
  m = max(m & 0xffffu, m >> 16);  // as integers non-negative floats keep their order
  return __half2float(__ushort_as_half(static_cast<uint16_t>(m)));
}

// Three groups of four warps, a thread per weight row: a group takes every third block of 64 values, so
// that one is loading and waiting while the others store. With all warps on every block, two threads per
// row, a block took 1,100 cycles (its MMAs take 512), with two groups 1,000: instruction latency, one
// after the other.
// first, step, units: the CTA's units of work; decode: a unit with the first of this CTA's own 128 weight
// rows; arrive: counts a warp on the barrier of a stage's weights.
template <typename T, bool F32S, int NS, int STAGE, typename Decode, typename Arrive>
__device__ __forceinline__ void widen_blocks(const I4Args& args, const I4Run& run, I4Tail* tail,
                                             uint8_t* smem, int first, int step, int units,
                                             const Decode& decode, const Arrive& arrive) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T* type = nullptr;
  const int r = threadIdx.x & 127;
  const int grp = (warp - kI4Widen0) >> 2;
  const bool g32 = run.group_magic == 0;
  const bool whole = (args.K & 63) == 0;  // no row ends inside a block
  const bool wide = whole && (reinterpret_cast<uintptr_t>(args.w) & 31u) == 0;
  const auto group_of = [&](int k) {
    const uint32_t k32 = static_cast<uint32_t>(k >> 5);
    return static_cast<int>(g32 ? k32 : __umulhi(k32, run.group_magic));
  };
  // The blocks of all of this CTA's units, one after the other; where the next to be loaded is.
  int total = 0;
  for (int unit = first; unit < units; unit += step) {
    const int part = unit % run.S;
    total += (part + 1) * run.nkb / run.S - part * run.nkb / run.S;
  }
  int unit = first, kb = 0, kb1 = 0;
  // of the row of this thread: its values, scales and zero points
  const uint8_t *wr = nullptr, *sr = nullptr, *zr = nullptr;
  constexpr int SB = F32S ? 4 : 2;
  const auto row_of = [&](const I4Unit& u) {
    // rows behind the last are the last, and are not stored
    return static_cast<int64_t>(u.e) * args.N + min(u.n0 + r, args.N - 1);
  };
  const auto open = [&]() {
    const I4Unit u = decode(unit);
    const int64_t row = row_of(u);
    wr = args.w + row * (args.K / 2);
    sr = static_cast<const uint8_t*>(args.scale) + row * args.groups * SB;
    zr = args.zero ? args.zero + row * args.groups : nullptr;
    return u;
  };
  // to the unit that a position behind a unit's end belongs to
  const auto settle = [&]() {
    while (kb >= kb1 && unit < units) {
      const int over = kb - kb1;
      unit += step;
      if (unit >= units) break;
      const I4Unit u = open();
      kb = u.kb0 + over;
      kb1 = u.kb1;
    }
  };
  // z1 kSame: the second half's scale and zero point are the first half's (not copied: a copy of a value
  // that is still being loaded would wait for it)
  constexpr uint32_t kSame = 0x100u;
  struct Ahead {
    uint32_t w[8], s0, s1, z0, z1;
  };
  Ahead q[kI4Ahead];
  const auto fetch = [&](Ahead& to) {
    if (unit >= units) return;
    const uint8_t* w = wr + kb * 32;
    const int at = group_of(kb * kI4KB);
    const auto scale = [&](int i) {
      return F32S ? reinterpret_cast<const uint32_t*>(sr)[i]
                  : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(sr)[i]);
    };
    to.s0 = scale(at);
    to.z0 = zr ? zr[at] : 8u;
    to.z1 = kSame;
    if (wide) {
      ld_global_v8(w, to.w);
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(w);
      to.w[0] = a.x, to.w[1] = a.y, to.w[2] = a.z, to.w[3] = a.w;
    }
    if (g32 || !wide) {
      if (whole || kb * kI4KB + 32 < args.K) {
        if (!wide) {
          const uint4 b = *reinterpret_cast<const uint4*>(w + 16);
          to.w[4] = b.x, to.w[5] = b.y, to.w[6] = b.z, to.w[7] = b.w;
        }
        if (g32) {
          to.s1 = scale(at + 1);
          to.z1 = zr ? zr[at + 1] : 8u;
        }
      } else {
        to.s1 = 0;  // behind the row's end: zeros, whatever the values
        to.z1 = 8u;
      }
    }
    kb += kI4Groups;
    settle();
  };
  float factor = 1.0f;
  const auto scales = [&](uint32_t raw, uint32_t& hi, uint32_t& lo) {
    if constexpr (F32S || HALF) {
      float f = F32S ? __uint_as_float(raw) : __half2float(__ushort_as_half(static_cast<uint16_t>(raw)));
      f *= factor;
      T a;
      from_f32(f, &a);
      hi = pack2(type, to_f32(a), to_f32(a));
      if constexpr (F32S) {  // what the rounding left; nothing of an infinite scale
        const float rest = fabsf(f) < INFINITY && fabsf(to_f32(a)) < INFINITY ? f - to_f32(a) : 0.0f;
        lo = pack2(type, rest, rest);
      }
    } else {
      hi = raw * 0x00010001u;
    }
  };
  if (unit < units) {
    const I4Unit u = open();
    kb = u.kb0 + grp;
    kb1 = u.kb1;
    settle();
  }
#pragma unroll
  for (int d = 0; d < kI4Ahead; ++d) fetch(q[d]);
  // fp16: the unit of the block at hand, its blocks behind this one, its number, its factor
  int mine = first - step, left = 0, n = -1;
  int skip = grp + 1;
  const uint32_t base = smem_u32(smem) + r * 128;
  const uint32_t swz = static_cast<uint32_t>(r & 7) << 4;
  int s = grp, round = 0;
  bool ok = true;
  for (int it = grp; it < total && ok;) {
#pragma unroll
    for (int d = 0; d < kI4Ahead; ++d) {
      if (it >= total) break;
      if constexpr (HALF) {
        bool entered = false;
        while (left < skip) {
          skip -= left;
          mine += step;
          ++n;
          const int part = mine % run.S;
          left = (part + 1) * run.nkb / run.S - part * run.nkb / run.S;
          entered = true;
        }
        left -= skip;
        skip = kI4Groups;
        if (entered) {
          // the largest scale of the unit's groups to [2^9, 2^10)
          const I4Unit u = decode(mine);
          const int g0 = group_of(u.kb0 * kI4KB), g1 = group_of(min(u.kb1 * kI4KB, args.K) - 1);
          const float most = largest_scale<F32S>(args, row_of(u) * args.groups, g0, g1);
          int ex = static_cast<int>(__float_as_uint(most) >> 23) - 127 - 9;
          if (most == 0.0f || ex > 110) ex = 0;  // nothing, or infinite
          if (ex < -120) ex = -120;
          factor = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
          // every group writes the same
          tail->inv[n % kI4Invs][r] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
        }
      }
      if (round > 0)
        ok = __all_sync(0xffffffffu, parked_wait(&tail->empty[s], (round & 1) ^ 1, abort_flag,
                                                 run.wait_ns));
      if (!ok) {
        if (lane == 0) i4_abort(tail);
        break;
      }
      const uint32_t to = (base + s * STAGE) ^ swz;
      uint32_t hi, lo = 0;
      scales(q[d].s0, hi, lo);
      uint32_t z = nibble_base(type) + (q[d].z0 & 15u) * 0x00010001u;
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) st_shared_v4(to ^ (c << 4), weights8<T, F32S>(q[d].w[c], z, hi, lo));
      if (q[d].z1 != kSame) {
        scales(q[d].s1, hi, lo);
        z = nibble_base(type) + (q[d].z1 & 15u) * 0x00010001u;
      }
#pragma unroll
      for (uint32_t c = 4; c < 8; ++c) st_shared_v4(to ^ (c << 4), weights8<T, F32S>(q[d].w[c], z, hi, lo));
      fence_async_smem();  // the MMAs read through the asynchronous proxy
      __syncwarp();
      if (lane == 0) arrive(s);
      fetch(q[d]);  // behind the fence, which would wait for the loads
      it += kI4Groups;
      s += kI4Groups;
      if (s >= NS) {
        s -= NS;
        ++round;
      }
    }
  }
}

// The epilogue of one warp: its 32 channels (one per lane) of the tile's columns; out is the element of the
// tile's first token at this warp's first channel. PAIRS (outputs at 4-byte
// boundaries): neighbouring lanes exchange halves of their tokens, so that a lane stores two channels at
// once. O float: the partial sums of a split product.
template <typename O, bool PAIRS>
__device__ __forceinline__ void store_tile(uint32_t taddr, int cols, int rows, float factor, float bias,
                                           O* out, int N, int live) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1;
  O* mine = out + (PAIRS ? lane & ~1 : lane);
  const bool writes = lane < live;  // N is even with PAIRS, so both channels of a pair exist
  for (int c = 0; c < cols; c += 16) {
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

// Zeroes the rows of no expert, by the epilogue warps of all CTAs.
__device__ __forceinline__ void zero_rows_beside(const I4Args& args, const I4Tail* tail) {
  if (!args.zero_tail) return;
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * (kI4EpiWarps * 32) + threadIdx.x - kI4Epi0 * 32;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * (kI4EpiWarps * 32);
  zero_rows16(args.out, args.N, 0, tail->ebase[0], tid, threads);
  zero_rows16(args.out, args.N, tail->live, args.M, tid, threads);
}

// One epilogue warp's share of a unit, the n-th of this CTA, from its lanes of the accumulator at taddr.
template <typename T, bool HALF>
__device__ __forceinline__ void store_unit(const I4Args& args, const I4Run& run, const I4Tail* tail,
                                           const I4Unit& u, int n, uint32_t taddr, bool pairs) {
  const int at_row = (threadIdx.x >> 5 & 3) * 32, lane = threadIdx.x & 31;
  const int n0 = u.n0 + at_row, live = args.N - n0;
  const float bias = run.S == 1 && args.bias && lane < live ? __ldcg(args.bias + n0 + lane) : 0.0f;
  const float factor = HALF ? tail->inv[n % kI4Invs][at_row + lane] : 1.0f;
  const int64_t at = u.row0 * args.N + n0;
  if (run.S > 1)
    store_tile<float, false>(taddr, u.cols, u.rows, factor, 0.0f,
                             args.part + static_cast<int64_t>(u.part) * args.M * args.N + at, args.N, live);
  else if (pairs)
    store_tile<T, true>(taddr, u.cols, u.rows, factor, bias, static_cast<T*>(args.out) + at, args.N, live);
  else
    store_tile<T, false>(taddr, u.cols, u.rows, factor, bias, static_cast<T*>(args.out) + at, args.N, live);
}

template <typename T, int BN, bool F32S>
__global__ void __launch_bounds__(kI4Threads, 1)
    k_int4_mm(const __grid_constant__ CUtensorMap tm_x, const I4Args args, const I4Run run) {
  using C = I4Cfg<BN>;
  constexpr int NS = C::NS;
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
      mbar_init(&tail->afull[s], 4);
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
  if (warp == 0) plan_tiles(args, BN, NT, tail);
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
        const I4Unit u = decode_unit<16, kI4Rows>(unit, NT, tail, E, run);
        const int boxes = (u.cols + C::BOX - 1) / C::BOX;
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++it) {
          const int s = it % NS, r = it / NS;
          if (r > 0 && !parked_wait(&tail->empty[s], (r & 1) ^ 1, abort_flag, run.wait_ns)) {
            i4_abort(tail);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::STAGE + C::BLOCK_A;
          mbar_arrive_expect_tx(&tail->bfull[s], boxes * C::BOX * 128);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(st + b * C::BOX * 128, &tm_x, &tail->bfull[s], kb * 128,
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
        const I4Unit u = decode_unit<16, kI4Rows>(unit, NT, tail, E, run);
        const uint32_t idesc = idesc_16<T>(kI4Rows, u.cols);
        const int b = n & 1, rb = n >> 1;
        const uint32_t d = tmem + b * BN;
        if (rb > 0 && !parked_wait(&tail->tempty[b], (rb & 1) ^ 1, abort_flag, run.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t more = 0;  // the unit's first MMA overwrites
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++it) {
          const int s = it % NS, r = it / NS;
          if (!parked_wait(&tail->afull[s], r & 1, abort_flag, run.wait_ns) ||
              !parked_wait(&tail->bfull[s], r & 1, abort_flag, run.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * C::STAGE);
          const uint64_t wd = smem_desc_k128(sa), xd = smem_desc_k128(sa + C::BLOCK_A);
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // 16 values of K each
            mma_f16(d, wd + 2 * j, xd + 2 * j, idesc, more);
            more = 1u;
          }
          mma_commit(&tail->empty[s]);
        }
        if (ok) mma_commit(&tail->tfull[b]);
      }
      if (!ok) i4_abort(tail);
      mma_commit(&tail->drain);
      (void)mbar_wait(&tail->drain, 0);
    }
  } else if (warp >= kI4Widen0 && warp < kI4Epi0) {
    // ---------------------------------------------------------------- widening
    widen_blocks<T, F32S, NS, C::STAGE>(
        args, run, tail, smem, blockIdx.x, gridDim.x, units,
        [&](int unit) { return decode_unit<16, kI4Rows>(unit, NT, tail, E, run); },
        [&](int s) { mbar_arrive(&tail->afull[s]); });
  } else if (warp >= kI4Epi0) {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;              // TMEM lanes of this warp
    zero_rows_beside(args, tail);
    const bool pairs = (args.N & 1) == 0 && (reinterpret_cast<uintptr_t>(args.out) & 3u) == 0;
    int n = 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++n) {
      const I4Unit u = decode_unit<16, kI4Rows>(unit, NT, tail, E, run);
      const int b = n & 1, rb = n >> 1;
      if (!__all_sync(0xffffffffu, parked_wait(&tail->tfull[b], rb & 1, abort_flag, run.wait_ns))) {
        if (lane == 0) i4_abort(tail);
        break;
      }
      tc_fence_after();
      store_unit<T, HALF>(args, run, tail, u, n,
                          tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * BN, pairs);
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

// ------------------------------------------------------------------ CTA pairs
// For many tokens: two CTAs share a tile of 256 weight rows x up to 256 tokens. One MMA (cta_group::2,
// M = 256) reads both CTAs' shared memory: each widens its own 128 weight rows and loads half of the tokens,
// so a K block fills 32 KB of an SM's shared memory instead of 48 for the same 128 x 256 outputs. That fill
// bounds a single CTA: with 256 tokens per tile its blocks took 800 cycles (540 with the widening left
// out), at 75 to 92 bytes a cycle that shared memory takes beside the MMAs' reads.
//
// Both CTAs count on the leader's (rank 0's) barriers; the leader issues the MMAs and commits to the barriers
// of both. Each CTA stores its own weight rows' outputs.
constexpr int kI4PairTokens = 256;
constexpr int kI4PairBlock = kI4Rows * 128;               // weights, and as much again of tokens
constexpr int kI4PairStage = 2 * kI4PairBlock;
constexpr int kI4PairStages = 6;
constexpr int kI4PairBox = 32;                            // token rows per TMA box
constexpr size_t kI4PairSmem =
    static_cast<size_t>(kI4PairStages) * kI4PairStage + sizeof(I4Tail) + 1024;
static_assert(kI4PairSmem <= 227 * 1024, "pair shared memory");
static_assert(kI4PairStages <= kI4MaxStages && kI4PairStages + 2 < kI4Invs, "arrays");

__device__ __forceinline__ uint32_t at_cta(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}

// Loads a box into this CTA's shared memory, its bytes counted on a barrier of the pair.
__device__ __forceinline__ void load_box_pair(void* dst, const void* tmap, uint32_t bar, int32_t c0,
                                              int32_t c1, uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "l"(hint)
      : "memory");
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on the barrier at `bar`'s place in both CTAs when the issued MMAs have finished.
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The arrival of a warp's weights on the leader's barrier. They are in this CTA's own shared memory, and
// fence.proxy.async, before this, has handed them to the asynchronous proxy, through which the pair's MMAs
// read them: the arrival carries no data of its own and has to follow that fence only. With .release.cluster it
// also waits for the loads that the warp has under way: 8192 x 4096 x 7168 took 559 us with it, 418 without,
// and 609 with a warp of its own that passes the arrivals on.
__device__ __forceinline__ void arrive_weights(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// parked_wait for a phase that threads of the other CTA arrive on as well: acquires at cluster scope.
__device__ __forceinline__ bool parked_wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                 uint64_t limit_ns) {
  uint64_t t0 = 0;
  for (uint32_t polls = 1;; ++polls) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
        : "memory");
    if (ok) return true;
    if ((polls & 15u) == 0) {
      if (*abort_flag) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > limit_ns) return false;
    }
  }
}

// After an abort, by the leader once no role of either CTA issues any more: waits (bounded) until the copies
// issued into every stage have landed, in both CTAs. A round needs both CTAs' copies and the next needs
// both CTAs' stages, so a CTA is at most one round ahead of the other; the half of a round that was never
// issued is taken off what the barrier expects.
__device__ __forceinline__ void drain_pair(I4Tail* t) {
  for (int s = 0; s < kI4PairStages; ++s) {
    const int mine = t->last_issue[s], other = ld_dsmem_s32(&t->last_issue[s], 1);
    const int r = max(mine, other);
    if (r < 0) continue;
    if (mine < r) {
      mbar_arrive_expect_tx(&t->bfull[s], ld_dsmem_s32(&t->last_bytes[s], 1));
    } else if (other < r) {
      asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(
                       smem_u32(&t->bfull[s])),
                   "r"(t->last_bytes[s])
                   : "memory");
    }
    (void)mbar_wait(&t->bfull[s], r & 1);
  }
}

template <typename T, bool F32S>
__global__ void __launch_bounds__(kI4Threads, 1)
    k_int4_pair(const __grid_constant__ CUtensorMap tm_x, const I4Args args, const I4Run run) {
  constexpr int NS = kI4PairStages;
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  I4Tail* tail = reinterpret_cast<I4Tail*>(smem + NS * kI4PairStage);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = args.E;
  const int NT = (args.N + 2 * kI4Rows - 1) / (2 * kI4Rows);
  const int rank = static_cast<int>(cluster_ctarank());

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&tail->bfull[s], 1);
      mbar_init(&tail->afull[s], 2 * 4);
      mbar_init(&tail->empty[s], 1);
      tail->last_issue[s] = -1;
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tail->tfull[b], 1);
      mbar_init(&tail->tempty[b], 2 * kI4EpiWarps);
    }
    mbar_init(&tail->drain, 1);
    mbar_init(&tail->never, 1);
    tail->abort_flag = 0;
    tail->gave_up = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tail->tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  pdl_begin_in_order();
  if (warp == 0) plan_tiles(args, kI4PairTokens, NT, tail);
  tc_fence_before();
  __syncthreads();
  // both CTAs' barriers are initialised and both have their tensor memory
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  const int units = tail->tiles * run.S;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    // ---------------------------------------------------------------- tokens
    if (elect_one()) {
      const uint64_t pol = policy_evict_last();
      int it = 0;
      // the injected failure also leaves a stage that one CTA of the pair alone has filled
      const int stop = run.inject != 0 ? 2 - rank : -1;
      bool ok = true;
      for (int unit = first; unit < units && ok; unit += step) {
        const I4Unit u = decode_unit<32, 2 * kI4Rows>(unit, NT, tail, E, run);
        const int half = u.cols / 2;
        const int boxes = (half + kI4PairBox - 1) / kI4PairBox;
        const int bytes = boxes * kI4PairBox * 128;
        const int row = static_cast<int>(u.row0) + rank * half;
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++it) {
          const int s = it % NS, r = it / NS;
          if (it == stop) {
            ok = false;
            break;
          }
          if (r > 0 && !parked_wait(&tail->empty[s], (r & 1) ^ 1, abort_flag, run.wait_ns)) {
            i4_abort(tail);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kI4PairStage + kI4PairBlock;
          if (rank == 0) mbar_arrive_expect_tx(&tail->bfull[s], 2 * bytes);
          const uint32_t bar = at_cta(&tail->bfull[s], 0);
          for (int b = 0; b < boxes; ++b)
            load_box_pair(st + b * kI4PairBox * 128, &tm_x, bar, kb * 128, row + b * kI4PairBox, pol);
          tail->last_issue[s] = r;
          tail->last_bytes[s] = bytes;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs (the leader's)
    if (rank == 0 && elect_one()) {
      int it = 0, n = 0;
      bool ok = run.inject == 0 || parked_wait(&tail->never, 0, abort_flag, run.wait_ns);
      for (int unit = first; unit < units && ok; unit += step, ++n) {
        const I4Unit u = decode_unit<32, 2 * kI4Rows>(unit, NT, tail, E, run);
        const uint32_t idesc = idesc_16<T>(2 * kI4Rows, u.cols);
        const int b = n & 1, rb = n >> 1;
        const uint32_t d = tmem + b * kI4PairTokens;
        if (rb > 0 && !parked_wait_pair(&tail->tempty[b], (rb & 1) ^ 1, abort_flag, run.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t more = 0;
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++it) {
          const int s = it % NS, r = it / NS;
          if (!parked_wait_pair(&tail->afull[s], r & 1, abort_flag, run.wait_ns) ||
              !parked_wait(&tail->bfull[s], r & 1, abort_flag, run.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * kI4PairStage);
          const uint64_t wd = smem_desc_k128(sa), xd = smem_desc_k128(sa + kI4PairBlock);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_f16_pair(d, wd + 2 * j, xd + 2 * j, idesc, more);
            more = 1u;
          }
          commit_both(&tail->empty[s]);
        }
        if (ok) commit_both(&tail->tfull[b]);
      }
      if (!ok) i4_abort(tail);
      commit_both(&tail->drain);
    }
    if (lane == 0) (void)mbar_wait(&tail->drain, 0);
  } else if (warp >= kI4Widen0 && warp < kI4Epi0) {
    // ---------------------------------------------------------------- widening
    widen_blocks<T, F32S, NS, kI4PairStage>(
        args, run, tail, smem, first, step, units,
        [&](int unit) {
          I4Unit u = decode_unit<32, 2 * kI4Rows>(unit, NT, tail, E, run);
          u.n0 += rank * kI4Rows;
          return u;
        },
        [&](int s) { arrive_weights(at_cta(&tail->afull[s], 0)); });
  } else if (warp >= kI4Epi0) {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    zero_rows_beside(args, tail);
    const bool pairs = (args.N & 1) == 0 && (reinterpret_cast<uintptr_t>(args.out) & 3u) == 0;
    int n = 0;
    for (int unit = first; unit < units; unit += step, ++n) {
      I4Unit u = decode_unit<32, 2 * kI4Rows>(unit, NT, tail, E, run);
      u.n0 += rank * kI4Rows;
      const int b = n & 1, rb = n >> 1;
      if (!__all_sync(0xffffffffu, parked_wait(&tail->tfull[b], rb & 1, abort_flag, run.wait_ns))) {
        if (lane == 0) i4_abort(tail);
        break;
      }
      tc_fence_after();
      store_unit<T, HALF>(args, run, tail, u, n,
                          tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * kI4PairTokens, pairs);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(at_cta(&tail->tempty[b], 0));
    }
  }

  tc_fence_before();
  __syncthreads();
  // Never leave a bulk copy in flight into shared memory that is about to be released. Without an abort of
  // the leader its MMAs have waited for all of them.
  if (threadIdx.x == 0 && rank == 0 && *abort_flag)
    for (int c = 0; c < 2; ++c)
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at_cta(&tail->gave_up, c)), "r"(1)
                   : "memory");
  cluster_arrive();  // the pair's MMAs are done
  cluster_wait();
  tc_fence_after();
  if (*reinterpret_cast<volatile int*>(&tail->gave_up)) {
    if (threadIdx.x == 0 && rank == 0) drain_pair(tail);
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
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
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(bytes));
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  return e;
}

template <typename T, int BN, bool F32S>
cudaError_t launch_single(const CUtensorMap& tm_x, const I4Args& a, const I4Run& r, int64_t units, int sms,
                          cudaStream_t s) {
  static std::atomic<bool> done[64];
  const cudaError_t e = allow_smem(k_int4_mm<T, BN, F32S>, i4_smem_bytes<BN>(), done);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_int4_mm<T, BN, F32S>, dim3(static_cast<unsigned>(units < sms ? units : sms)),
                    dim3(kI4Threads), i4_smem_bytes<BN>(), s, tm_x, a, r);
}

template <typename T, bool F32S>
cudaError_t launch_pair(const CUtensorMap& tm_x, const I4Args& a, const I4Run& r, int64_t units, int sms,
                        cudaStream_t s) {
  static std::atomic<bool> done[64];
  const cudaError_t e = allow_smem(k_int4_pair<T, F32S>, kI4PairSmem, done);
  if (e != cudaSuccess) return e;
  const int64_t clusters = units < sms / 2 ? units : sms / 2;
  return launch_pdl_cluster(k_int4_pair<T, F32S>, dim3(static_cast<unsigned>(2 * clusters)),
                            dim3(kI4Threads), kI4PairSmem, s, 2, tm_x, a, r);
}

template <typename T, bool F32S>
cudaError_t launch_mm(const Int4Product& p, const I4Args& a, const Int4Plan& plan, int sms,
                      cudaStream_t s) {
  const int box = plan.bn == 64 ? I4Cfg<64>::BOX : plan.bn == 128 ? I4Cfg<128>::BOX : kI4PairBox;
  CUtensorMap tm_x;
  const uint64_t row = static_cast<uint64_t>(p.K) * 2;
  if (!tensor_map_u8(&tm_x, p.x, row, p.M, row, 128, box)) return cudaErrorInvalidValue;
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
  const int rows = plan.bn == kI4PairTokens ? 2 * kI4Rows : kI4Rows;
  const int64_t units = (p.expert_base ? p.M / plan.bn + used : (p.M + plan.bn - 1) / plan.bn) *
                        ((p.N + rows - 1) / rows) * plan.S;
  cudaError_t e;
  if (plan.bn == 64)
    e = launch_single<T, 64, F32S>(tm_x, a, r, units, sms, s);
  else if (plan.bn == 128)
    e = launch_single<T, 128, F32S>(tm_x, a, r, units, sms, s);
  else
    e = launch_pair<T, F32S>(tm_x, a, r, units, sms, s);
  if (e != cudaSuccess || plan.S == 1) return e;
  const bool four = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7u) == 0;
  const int64_t blocks = (p.M * p.N / (four ? 4 : 1) + 255) / 256;
  const dim3 fgrid(static_cast<unsigned>(blocks < 8 * sms ? blocks : 8 * sms));
  if (four) return launch_pdl(k_int4_finish<T, 4>, fgrid, dim3(256), 0, s, a, plan.S);
  return launch_pdl(k_int4_finish<T, 1>, fgrid, dim3(256), 0, s, a, plan.S);
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
