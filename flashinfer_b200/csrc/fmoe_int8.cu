// fmoe_int8.cu -- 8-bit integer products with one scale per token and one per output channel,
// for one weight matrix or one per expert, and the quantisation of their activations.
//
//   q[t, k] = round_half_even(127 x[t, k] / amax_t),  a_scale[t] = amax_t / 127,
//             amax_t = max(max_k |x[t, k]|, 1e-30)
//   y[t, n] = a_scale[t] * w_scale[n] * sum_k a[t, k] * w[n, k] (+ bias[n])
// The sum is exact in int32 (127 * 127 * K and -128 * -128 * K stay below 2^31 for K <= 131071);
// the scaling is fp32 and rounded once to the output type.
//
// The weight rows are the M side of the MMA (128 per tile) and the tokens its N side (16..256 per
// tile, the instruction's N chosen per tile): a decode step then fills the 128 MMA rows with
// weights, which are all that costs, and a tile with few tokens issues a narrow MMA instead of
// padding. A tile's accumulator has one weight row per TMEM lane, so each epilogue thread keeps
// its channel's scale and bias in a register and a warp stores 32 neighbouring channels of a
// token at a time.
#include <cuda.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "fmoe_elem.cuh"
#include "fmoe_internal.h"
#include "fmoe_ptx.cuh"

namespace fmoe {
namespace {

// ------------------------------------------------------------------ quantisation
// Elementwise maximum of absolute values of 16-bit pairs; a NaN stays.
__device__ __forceinline__ uint32_t abs_max2(__nv_bfloat16*, uint32_t a, uint32_t b) {
  b &= 0x7fff7fffu;
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t abs_max2(__half*, uint32_t a, uint32_t b) {
  b &= 0x7fff7fffu;
  const __half2 m =
      __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// Two values as 127 x / amax rounded to the nearest integer, ties to even; the integers are the low
// bytes of the result. With both operands scaled by 2^-8, p = 127 x and den = amax are exact for
// 16-bit inputs and stay finite. v = p * inv is within two units of the quotient and p - v * den is
// exact, so the corrected v is the rounded quotient: a quotient halfway between integers comes out
// as that, and any other is 2^-18 (relative) or more away from halfway, x and amax having at most
// 11 bits. Adding 1.5 * 2^23 then rounds to the even integer. Against one IEEE division per
// element, quantising 8192 x 7168 took 84.9 us with it (58.1 without division but with a tie test).
__device__ __forceinline__ uint2 quant2(float2 x, float den, float inv) {
  const float2 c = make_float2(127.0f / 256.0f, 127.0f / 256.0f);
  const float2 i2 = make_float2(inv, inv), d2 = make_float2(-den, -den);
  const float2 p = __fmul2_rn(x, c);
  float2 v = __fmul2_rn(p, i2);
  v = __ffma2_rn(__ffma2_rn(v, d2, p), i2, v);
  v = __fadd2_rn(v, make_float2(12582912.0f, 12582912.0f));
  return make_uint2(__float_as_uint(v.x), __float_as_uint(v.y));
}

// A group (a warp with WARP, eight groups per block; else the block) takes rows first, first + step,
// .... Up to VPT 16-byte granules (VEC; else single elements) of a row per thread stay in registers
// between the maximum and the rounding, and the next row's are on their way meanwhile; what a longer
// row has beyond them is read a second time. One row per block, without the next row's loads:
// 8192 x 7168 took 44.7 us; it takes 31.5 (86% of the copy bandwidth over its 176 MB).
template <typename T, bool VEC, int VPT, bool WARP>
__global__ void __launch_bounds__(256, 4)
    k_quantize_int8(const T* x, int64_t rows, int64_t K, int8_t* q, float* scale) {
  pdl_begin_in_order();
  using Unit = typename std::conditional<VEC, uint4, uint16_t>::type;
  __shared__ uint32_t part[2][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = WARP ? 32 : blockDim.x;
  const int g = WARP ? lane : static_cast<int>(threadIdx.x);
  T* type = nullptr;
  const int64_t n = VEC ? K / 8 : K;
  const Unit* xu = reinterpret_cast<const Unit*>(x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 8 : 1);
  int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  Unit next[VPT];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (r < rows && g + i * G < n) next[i] = __ldcg(xu + r * n + g + i * G);
  };
  fetch(row);
  int flip = 0;
  for (; row < rows; row += step, flip ^= 1) {
    Unit in[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) in[i] = next[i];
    fetch(row + step);
    const Unit* xr = xu + row * n;
    int8_t* qr = q + row * K;
    uint32_t m2 = 0;
    auto maximum = [&](const Unit& u) {
      if constexpr (VEC) {
        m2 = abs_max2(type, m2, u.x);
        m2 = abs_max2(type, m2, u.y);
        m2 = abs_max2(type, m2, u.z);
        m2 = abs_max2(type, m2, u.w);
      } else {
        m2 = abs_max2(type, m2, u);
      }
    };
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (g + i * G < n) maximum(in[i]);
    for (int64_t v = g + static_cast<int64_t>(VPT) * G; v < n; v += G) maximum(__ldcg(xr + v));
    // as ordered integers the bits of non-negative floats keep their order, NaN above infinity
    const float2 halves = unpack2(type, m2);
    uint32_t m = max(__float_as_uint(halves.x), __float_as_uint(halves.y)) & 0x7fffffffu;
    m = __reduce_max_sync(0xffffffffu, m);
    if (!WARP) {  // one barrier: the next row uses the other buffer
      if (lane == 0) part[flip][warp] = m;
      __syncthreads();
      for (int i = 0; i < (G >> 5); ++i) m = max(m, part[flip][i]);
    }
    m = max(m, __float_as_uint(1e-30f));
    const float amax = __uint_as_float(m);
    if (g == 0) scale[row] = __fdiv_rn(amax, 127.0f);
    const bool finite = m < 0x7f800000u;  // else the row's values are zeros
    const float den = amax * (1.0f / 256.0f);
    const float inv = 1.0f / den;
    auto put = [&](const Unit& u, int64_t v) {
      if constexpr (VEC) {
        const uint2 a = quant2(unpack2(type, u.x), den, inv), b = quant2(unpack2(type, u.y), den, inv);
        const uint2 c = quant2(unpack2(type, u.z), den, inv), d = quant2(unpack2(type, u.w), den, inv);
        uint2 w;
        w.x = __byte_perm(__byte_perm(a.x, a.y, 0x0040), __byte_perm(b.x, b.y, 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(c.x, c.y, 0x0040), __byte_perm(d.x, d.y, 0x0040), 0x5410);
        reinterpret_cast<uint2*>(qr)[v] = finite ? w : make_uint2(0u, 0u);
      } else {
        qr[v] = finite ? static_cast<int8_t>(quant2(unpack2(type, u), den, inv).x) : int8_t{0};
      }
    };
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (g + i * G < n) put(in[i], g + i * G);
    for (int64_t v = g + static_cast<int64_t>(VPT) * G; v < n; v += G) put(__ldcg(xr + v), v);
  }
}

template <typename T, bool VEC>
cudaError_t quantize_rows(const void* x, int64_t rows, int64_t K, void* q, float* scale, int sms,
                          cudaStream_t s) {
  // a row of up to four units per lane is a warp's; a longer one a block's, with as few threads
  // as hold four units each; as many blocks as run at a time (64 registers per thread)
  const int64_t n = VEC ? K / 8 : K;
  const T* xt = static_cast<const T*>(x);
  int8_t* qt = static_cast<int8_t*>(q);
  if (n <= 32 * 4) {
    const int64_t blocks = (rows + 7) / 8, most = static_cast<int64_t>(sms) * 4;
    return launch_pdl(k_quantize_int8<T, VEC, 4, true>,
                      dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, s,
                      xt, rows, K, qt, scale);
  }
  int64_t threads = (n + 127) / 128 * 32;
  if (threads > 256) threads = 256;
  const int64_t most = static_cast<int64_t>(sms) * (1024 / threads);
  return launch_pdl(k_quantize_int8<T, VEC, 4, false>,
                    dim3(static_cast<unsigned>(rows < most ? rows : most)),
                    dim3(static_cast<unsigned>(threads)), 0, s, xt, rows, K, qt, scale);
}

// ------------------------------------------------------------------ product
constexpr int kI8Threads = 640;   // warps 0, 2, 3 load, warp 1 issues MMAs, 4..19 store
constexpr int kI8Producers = 3;
constexpr int kI8Epi0 = 4;
constexpr int kI8EpiWarps = 16;   // with 8 the stores of 8192 x 7168 outputs took 70 us at any K
constexpr int kI8EpiCols = kI8EpiWarps / 4 * 16;  // columns that the warps take at a time
constexpr int kWRows = 128;       // weight rows per tile (MMA M)
constexpr int kKB = 128;          // K bytes of a block (one 128-byte swizzled row)
// K blocks per stage. A stage costs the MMA warp's loop time beside its MMAs: with one block per stage
// 8192 x 4096 x 7168 took 176 us, with two 167. Three would leave two stages in flight.
constexpr int kSub = 2;
constexpr int kI8MaxStages = 6;

template <int BN>
struct I8Cfg {
  static constexpr int BLOCK = (kWRows + BN) * kKB;
  static constexpr int STAGE = kSub * BLOCK;
  static constexpr int NS = BN == 16 ? 6 : BN == 64 ? 4 : 3;
  static constexpr int BOX = BN == 16 ? 16 : 64;   // token rows per TMA box
  static constexpr int COLS = 2 * BN < 32 ? 32 : 2 * BN;
  static_assert(NS >= kI8Producers && NS <= kI8MaxStages, "producer parity and barrier arrays");
};

struct alignas(16) I8Tail {
  uint64_t full[kI8MaxStages];
  uint64_t empty[kI8MaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint64_t never;
  uint32_t tmem_base;
  int abort_flag;
  int tiles;
  int live;
  int last_issue[kI8Producers][kI8MaxStages];
  alignas(16) float a_scale[128];
  int ebase[kMaxLocalExperts + 1];
  int etile[kMaxLocalExperts + 1];  // token tiles before expert e
};

struct I8Args {
  const float* a_scale;
  const float* w_scale;
  const float* bias;          // or null
  const int32_t* expert_base; // or null: one matrix
  void* out;
  int64_t M;                  // token rows
  int N, E, nkb, S;
  int dtype;                  // output
  int zero_tail;
  // every bounded wait gives up after wait_ns; inject: the MMA warp first waits on a barrier that
  // nothing arrives on (tests of the failure path only)
  unsigned long long wait_ns;
  int inject;
};

template <int BN>
constexpr size_t i8_smem_bytes() {
  return static_cast<size_t>(I8Cfg<BN>::NS) * I8Cfg<BN>::STAGE + sizeof(I8Tail) + 1024;
}
static_assert(i8_smem_bytes<16>() <= 227 * 1024 && i8_smem_bytes<64>() <= 227 * 1024 &&
                  i8_smem_bytes<128>() <= 227 * 1024,
              "shared memory per CTA");

// D[tmem] (+)= A[smem] * B[smem]^T, s8 x s8 -> s32.
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: D s32, A and B signed 8-bit, both K-major.
__device__ __forceinline__ uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

struct I8Tile {
  int e, n0;         // expert, first weight row (channel)
  int64_t row0;      // first token row
  int rows, cols;    // tokens in the tile, and the MMA's N (a multiple of 16)
};

// Tile order: expert, weight tile, token tile (fastest), so CTAs that run side by side share
// weight tiles. The tokens of an expert are cut into equal tiles of at most BN.
template <int BN>
__device__ __forceinline__ I8Tile decode_tile(int tile, int NT, const I8Tail* t, int E) {
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
  I8Tile r;
  r.e = lo;
  r.n0 = n * kWRows;
  r.row0 = t->ebase[lo] + static_cast<int64_t>(m) * per;
  r.rows = max(0, min(per, count - m * per));
  r.cols = max(16, (r.rows + 15) / 16 * 16);
  return r;
}

// The bases as a running maximum (by one warp): where one steps back, the rows before the largest so
// far stay with the experts that have them. So no row is written twice, and no spread of the rows has
// more tiles than the host's bound, which is the grid of a split.
__device__ __forceinline__ void ascending_bases(int* base, int E, bool grouped) {
  const int lane = threadIdx.x & 31;
  if (!grouped) return;
  int carry = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    int most = max(carry, e <= E ? base[e] : 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, most, o);
      if (lane >= o) most = max(most, up);
    }
    if (e <= E) base[e] = most;
    carry = __shfl_sync(0xffffffffu, most, 31);
  }
  __syncwarp();
}

// Set by a product whose bounded wait ran out, until take_int8_status takes it to g_int8_taken.
__device__ int32_t g_int8_status;
__device__ int32_t g_int8_taken;

// Reads and clears in one step: a product on another stream may set the word at any time.
__global__ void k_take_int8_status() { g_int8_taken = atomicExch(&g_int8_status, 0); }

__device__ __forceinline__ void i8_abort(I8Tail* t) {
  *reinterpret_cast<volatile int*>(&t->abort_flag) = 1;
  atomicOr(&g_int8_status, FMOE_STATUS_TIMEOUT_INT8);
}

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
  if (dtype == FMOE_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else if (dtype == FMOE_DTYPE_F16)
    static_cast<__half*>(out)[i] = __float2half_rn(v);
  else
    static_cast<float*>(out)[i] = v;
}

// Zeroes output rows [from, to) by 16-byte stores, single 16-bit words at the ends; thread `tid` of
// `threads`. Rows of experts that live elsewhere can be most of the output: with 4096 of 32768 rows
// live, a product of depth 1024 to 4096 bf16 channels takes 73 us, with element stores it took 78.
__device__ __forceinline__ void zero_rows_out(const I8Args& a, int64_t from, int64_t to, int64_t tid,
                                              int64_t threads) {
  const int64_t row = static_cast<int64_t>(a.N) * (a.dtype == FMOE_DTYPE_F32 ? 4 : 2);
  const int64_t bytes = (to - from) * row;
  if (bytes <= 0) return;
  uint8_t* p = static_cast<uint8_t*>(a.out) + from * row;
  int64_t head = (16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15u)) & 15;
  if (head > bytes) head = bytes;
  const int64_t wide = (bytes - head) / 16;
  for (int64_t i = tid; i < wide; i += threads)
    reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0u, 0u, 0u, 0u);
  const int64_t rest = bytes - head - wide * 16;  // like head an even number below 16
  if (tid < head / 2) reinterpret_cast<uint16_t*>(p)[tid] = 0;
  if (tid < rest / 2) reinterpret_cast<uint16_t*>(p + head + wide * 16)[tid] = 0;
}

// The epilogue of one warp: its 32 channels (one per lane) of the tile's columns c0, c0 + 16, ... in
// steps of c_step, from the accumulator at taddr; out is the element of the tile's first token at
// this warp's first channel. `live` channels of the 32 exist.
// PAIRS (16-bit outputs at 4-byte boundaries): neighbouring lanes exchange halves of their tokens,
// so a lane stores two channels at once and a warp two tokens' 64 bytes. Single 16-bit stores with
// the type decided per element took 100 us for 8192 x 7168 outputs, whatever K.
template <typename O, bool PAIRS>
__device__ __forceinline__ void store_columns(uint32_t taddr, int c0, int c_step, int cols, int rows,
                                              const float* a_scale, float ws, float bias, O* out,
                                              int N, int live) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1;
  O* mine = out + (PAIRS ? lane & ~1 : lane);
  const bool writes = lane < live;  // N is even with PAIRS, so both channels of a pair exist
  for (int c = c0; c < cols; c += c_step) {
    __syncwarp();  // the tensor memory is read by the whole warp, which the stores below divide
    float v[16];
    tmem_ld_32x32b_x16(taddr + c, v);
    tmem_ld_wait16(v);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 s = *reinterpret_cast<const float4*>(a_scale + c + i);
      v[i] = fmaf(static_cast<float>(__float_as_int(v[i])) * s.x, ws, bias);
      v[i + 1] = fmaf(static_cast<float>(__float_as_int(v[i + 1])) * s.y, ws, bias);
      v[i + 2] = fmaf(static_cast<float>(__float_as_int(v[i + 2])) * s.z, ws, bias);
      v[i + 3] = fmaf(static_cast<float>(__float_as_int(v[i + 3])) * s.w, ws, bias);
    }
    if constexpr (PAIRS) {
      // even lanes take tokens c .. c + 7, odd lanes c + 8 .. c + 15
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 8], 1);
        w[i] = odd ? pack2(static_cast<O*>(nullptr), other, v[i + 8])
                   : pack2(static_cast<O*>(nullptr), v[i], other);
      }
      if (writes) {
        O* p = mine + static_cast<int64_t>(c + (odd ? 8 : 0)) * N;
        const int left = rows - c - (odd ? 8 : 0);
        if (left >= 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i, p += N) *reinterpret_cast<uint32_t*>(p) = w[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i, p += N)
            if (i < left) *reinterpret_cast<uint32_t*>(p) = w[i];
        }
      }
    } else if (writes) {
      O* p = mine + static_cast<int64_t>(c) * N;
      const int left = rows - c;
      if (left >= 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i, p += N) from_f32(v[i], p);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, p += N)
          if (i < left) from_f32(v[i], p);
      }
    }
  }
  __syncwarp();
}

// The same for the call's output type.
__device__ __forceinline__ void store_columns(const I8Args& a, uint32_t taddr, int c0, int c_step,
                                              const I8Tile& u, int n0, const float* a_scale,
                                              float ws, float bias) {
  const int64_t at = u.row0 * a.N + n0;
  const int live = a.N - n0;
  const bool pairs = (a.N & 1) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0;
  if (a.dtype == FMOE_DTYPE_F32) {
    store_columns<float, false>(taddr, c0, c_step, u.cols, u.rows, a_scale, ws, bias,
                                static_cast<float*>(a.out) + at, a.N, live);
  } else if (a.dtype == FMOE_DTYPE_BF16) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
    if (pairs)
      store_columns<__nv_bfloat16, true>(taddr, c0, c_step, u.cols, u.rows, a_scale, ws, bias, o,
                                         a.N, live);
    else
      store_columns<__nv_bfloat16, false>(taddr, c0, c_step, u.cols, u.rows, a_scale, ws, bias, o,
                                          a.N, live);
  } else {
    __half* o = static_cast<__half*>(a.out) + at;
    if (pairs)
      store_columns<__half, true>(taddr, c0, c_step, u.cols, u.rows, a_scale, ws, bias, o, a.N,
                                  live);
    else
      store_columns<__half, false>(taddr, c0, c_step, u.cols, u.rows, a_scale, ws, bias, o, a.N,
                                   live);
  }
}

// Tokens of one of S shares of a tile: whole groups of 16, so a group has one receiver.
__device__ __forceinline__ int split_share(int rows, int S) {
  return ((rows + S - 1) / S + 15) / 16 * 16;
}

// The address in CTA `rank`'s shared memory of what this CTA has at p.
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}

// The end of a tile whose K range was split over S CTAs of the cluster, ranks rank0 + r * rank_step.
// Every CTA sends each token's 128 int32 partial sums to the CTA that finishes that token (share
// number token / per, per = tokens of a share, a multiple of 16): [sender][token of the share][128] in the receiver's
// stages, which are free once all of the tile's MMAs are done (a cluster barrier before). After
// another barrier each CTA adds its senders' sums (exact, so the split changes no result) and stores
// them. Sent rather than fetched: reads of the others' shared memory, one after the other, took
// 11 us for 256 tokens.
__device__ __forceinline__ void send_partials(uint32_t taddr, int g, const I8Tile& u, int per,
                                              uint8_t* part, int mine, int rank0, int rank_step,
                                              int channel) {
  // to the last token, not the last column: the columns, which pairs round up to 32, can hold a group
  // beyond the S shares, of a receiver that does not exist
  for (int c = g * 16; c < u.rows; c += kI8EpiCols) {
    __syncwarp();
    float v[16];
    tmem_ld_32x32b_x16(taddr + c, v);
    tmem_ld_wait16(v);
    const int share = c / per;  // of all 16 columns
    const uint32_t to = at_rank(part + ((mine * per + c - share * per) * kWRows + channel) * 4,
                                rank0 + share * rank_step);
    const int left = u.rows - c;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + i * kWRows * 4), "f"(v[i])
                     : "memory");
  }
}

__device__ __forceinline__ void finish_split(const I8Args& a, const I8Tile& u, int n0, int per,
                                             const uint8_t* part, int S, int mine) {
  const bool pairs = (a.N & 1) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3u) == 0;
  const int first = mine * per;
  const int tokens = min(per, u.rows - first);
  const float* wsp = a.w_scale + static_cast<int64_t>(u.e) * a.N;
  // a thread keeps its four channels: the block is a multiple of the 32 groups of a token
  const int c4 = (threadIdx.x % (kWRows / 4)) * 4;
  const int ch = n0 + c4;
  const int live = a.N - ch < 4 ? a.N - ch : 4;
  if (live <= 0) return;
  float ws[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ws[j] = j < live ? __ldcg(wsp + ch + j) : 0.0f;
    bias[j] = j < live && a.bias ? __ldcg(a.bias + ch + j) : 0.0f;
  }
  for (int t = threadIdx.x / (kWRows / 4); t < tokens; t += kI8Threads / (kWRows / 4)) {
    int sum[4] = {0, 0, 0, 0};
    for (int r = 0; r < S; ++r) {
      const int4 v = *reinterpret_cast<const int4*>(part + ((r * per + t) * kWRows + c4) * 4);
      sum[0] += v.x;
      sum[1] += v.y;
      sum[2] += v.z;
      sum[3] += v.w;
    }
    const int64_t row = u.row0 + first + t;
    const float as = __ldcg(a.a_scale + row);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(static_cast<float>(sum[j]) * as, ws[j], bias[j]);
    const int64_t at = row * a.N + ch;
    if (pairs && live == 4 && a.dtype != FMOE_DTYPE_F32) {
      uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at);
      if (a.dtype == FMOE_DTYPE_BF16) {
        o[0] = pack2(static_cast<__nv_bfloat16*>(nullptr), y[0], y[1]);
        o[1] = pack2(static_cast<__nv_bfloat16*>(nullptr), y[2], y[3]);
      } else {
        o[0] = pack2(static_cast<__half*>(nullptr), y[0], y[1]);
        o[1] = pack2(static_cast<__half*>(nullptr), y[2], y[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < live) store_out(a.out, a.dtype, at + j, y[j]);
    }
  }
}

// SPLIT: the cluster's S CTAs share one tile, each with a range of K; their int32 partial tiles
// are added through distributed shared memory (exact, so the split changes no result).
template <int BN, bool SPLIT>
__global__ void __launch_bounds__(kI8Threads, 1)
    k_int8_mm(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
              const I8Args args) {
  using C = I8Cfg<BN>;
  constexpr int NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  I8Tail* tail = reinterpret_cast<I8Tail*>(smem + NS * C::STAGE);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = args.E;
  const int NT = (args.N + kWRows - 1) / kWRows;
  const int S = SPLIT ? args.S : 1;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tail->tfull[b], 1);
      mbar_init(&tail->tempty[b], kI8EpiWarps * 32);
    }
    mbar_init(&tail->drain, 1);
    mbar_init(&tail->never, 1);
    tail->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, C::COLS);
    tmem_relinquish();
  }
  // everything this kernel reads may have been written by the previous grid
  pdl_begin_in_order();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    int64_t b = args.expert_base ? __ldcg(args.expert_base + e) : (e == 0 ? 0 : args.M);
    tail->ebase[e] = static_cast<int>(b < 0 ? 0 : b > args.M ? args.M : b);
  }
  __syncthreads();
  if (warp == 0) {
    ascending_bases(tail->ebase, E, args.expert_base != nullptr);
    // token tiles per expert and their running sum
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int mt = 0;
      if (e < E) {
        const int count = max(0, tail->ebase[e + 1] - tail->ebase[e]);
        mt = (count + BN - 1) / BN;
      }
      int incl = mt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (e < E) tail->etile[e] = carry + incl - mt;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      tail->etile[E] = carry;
      tail->tiles = carry * NT;
      tail->live = tail->ebase[E];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  const int tiles = tail->tiles;
  const int rank = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = SPLIT ? blockIdx.x / S : blockIdx.x;
  const int step = SPLIT ? gridDim.x / S : gridDim.x;  // SPLIT: at most one tile per cluster
  const int kb0 = rank * args.nkb / S, kb1 = (rank + 1) * args.nkb / S;

  if (warp == 0 || warp == 2 || warp == 3) {
    // ---------------------------------------------------------------- TMA producers
    const int pw = warp == 0 ? 0 : warp - 1;
    if (lane == 0) {
      const uint64_t pol_first = policy_evict_first();
      const uint64_t pol_last = policy_evict_last();
      for (int s = 0; s < NS; ++s) tail->last_issue[pw][s] = -1;
      int it = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        const I8Tile u = decode_tile<BN>(tile, NT, tail, E);
        const int boxes = (u.cols + C::BOX - 1) / C::BOX;
        const uint32_t block_bytes = (kWRows + boxes * C::BOX) * kKB;
        // a weight tile that several token tiles read stays in L2; one that is read once goes first
        const uint64_t pol_w =
            tail->etile[u.e + 1] - tail->etile[u.e] > 1 ? pol_last : pol_first;
        const int wrow = u.e * args.N + u.n0;
        for (int kb = kb0; kb < kb1; kb += kSub, ++it) {
          if (it % kI8Producers != pw) continue;
          const int s = it % NS, r = it / NS;
          // This producer issued iteration it - kI8Producers after that stage's release, and the
          // MMA warp releases in order, so with NS >= kI8Producers the barrier is at most one
          // phase behind and the parity wait is unambiguous.
          if (r > 0 && !parked_wait(&tail->empty[s], (r & 1) ^ 1, abort_flag, args.wait_ns)) {
            i8_abort(tail);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::STAGE;
          const int blocks = min(kSub, kb1 - kb);
          mbar_arrive_expect_tx(&tail->full[s], blocks * block_bytes);
          for (int j = 0; j < blocks; ++j, st += C::BLOCK) {
            const int k = (kb + j) * kKB;
            tma_load_2d(st, &tm_w, &tail->full[s], k, wrow, pol_w);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(st + (kWRows + b * C::BOX) * kKB, &tm_a, &tail->full[s], k,
                          static_cast<int>(u.row0) + b * C::BOX, pol_last);
          }
          tail->last_issue[pw][s] = r;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      int it = 0, n = 0;
      bool ok = args.inject == 0 || parked_wait(&tail->never, 0, abort_flag, args.wait_ns);
      for (int tile = first; tile < tiles && ok; tile += step, ++n) {
        const I8Tile u = decode_tile<BN>(tile, NT, tail, E);
        const uint32_t idesc = idesc_i8(kWRows, u.cols);
        const int b = n & 1, rb = n >> 1;
        const uint32_t d = tmem + b * BN;
        if (rb > 0 && !parked_wait(&tail->tempty[b], (rb & 1) ^ 1, abort_flag, args.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t more = 0;  // the tile's first MMA overwrites
        for (int kb = kb0; kb < kb1; kb += kSub, ++it) {
          const int s = it % NS, r = it / NS;
          if (!parked_wait(&tail->full[s], r & 1, abort_flag, args.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t st = smem_u32(smem + s * C::STAGE);
          for (int left = min(kSub, kb1 - kb); left > 0; --left, st += C::BLOCK) {
            const uint64_t w_desc = smem_desc_k128(st);
            const uint64_t a_desc = smem_desc_k128(st + kWRows * kKB);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma_i8(d, w_desc + 2 * j, a_desc + 2 * j, idesc, more);
              more = 1u;
            }
          }
          mma_commit(&tail->empty[s]);
        }
        if (ok) mma_commit(&tail->tfull[b]);
      }
      if (!ok) i8_abort(tail);
      mma_commit(&tail->drain);
      (void)mbar_wait(&tail->drain, 0);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const int q = warp & 3;              // TMEM lane quarter of this warp
    const int g = (warp - kI8Epi0) >> 2; // which 16 of kI8EpiCols columns
    const int etid = threadIdx.x - kI8Epi0 * 32;
    if (args.zero_tail) {  // rows of no expert
      const int64_t tid = static_cast<int64_t>(blockIdx.x) * (kI8EpiWarps * 32) + etid;
      const int64_t threads = static_cast<int64_t>(gridDim.x) * (kI8EpiWarps * 32);
      zero_rows_out(args, 0, tail->ebase[0], tid, threads);
      zero_rows_out(args, tail->live, args.M, tid, threads);
    }
    int n = 0;
    bool ok = true;
    for (int tile = first; tile < tiles; tile += step, ++n) {
      const I8Tile u = decode_tile<BN>(tile, NT, tail, E);
      const int b = n & 1, rb = n >> 1;
      const int ch = u.n0 + q * 32 + lane;
      const bool live = ch < args.N;
      const float ws = live ? __ldcg(args.w_scale + static_cast<int64_t>(u.e) * args.N + ch) : 0.0f;
      const float bias = live && args.bias ? __ldcg(args.bias + ch) : 0.0f;
      named_bar_sync(1, kI8EpiWarps * 32);  // the previous tile's a_scale is no longer read
      if (etid < u.rows) tail->a_scale[etid] = __ldcg(args.a_scale + u.row0 + etid);
      named_bar_sync(1, kI8EpiWarps * 32);
      // after a wait that ran out, the warp still takes part in the barriers of later tiles
      if (ok) ok = __all_sync(0xffffffffu, parked_wait(&tail->tfull[b], rb & 1, abort_flag, args.wait_ns));
      if (!ok) {
        if (lane == 0) i8_abort(tail);
        continue;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * BN;
      if constexpr (!SPLIT)
        store_columns(args, taddr, g * 16, kI8EpiCols, u, u.n0 + q * 32, tail->a_scale, ws, bias);
      tc_fence_before();
      mbar_arrive(&tail->tempty[b]);
    }
  }

  tc_fence_before();
  __syncthreads();
  // Never leave a bulk copy in flight into shared memory that is about to be released: after an
  // abort, wait for each stage's latest issued round (without one the MMA warp has seen them all).
  if (threadIdx.x == 0 && *abort_flag) {
    for (int s = 0; s < NS; ++s) {
      int r = -1;
      for (int p = 0; p < kI8Producers; ++p) r = max(r, tail->last_issue[p][s]);
      if (r >= 0) (void)mbar_wait(&tail->full[s], r & 1);
    }
  }
  if constexpr (SPLIT) {
    const I8Tile u = first < tiles ? decode_tile<BN>(first, NT, tail, E) : I8Tile{};
    const int per = split_share(u.rows, S);
    cluster_arrive();  // every CTA's MMAs are done, their stages free
    cluster_wait();
    tc_fence_after();
    if (warp >= kI8Epi0 && u.rows > 0)
      send_partials(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), (warp - kI8Epi0) >> 2, u,
                    per, smem, rank, 0, 1, (warp & 3) * 32 + lane);
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    if (u.rows > 0) finish_split(args, u, u.n0, per, smem, S, rank);
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// ------------------------------------------------------------------ a few tokens
// Up to four tokens: the product is a stream of the weights, which the tensor memory copies take
// from DRAM at about 45 bytes a nanosecond per SM, with a cluster's barriers on top; plain loads on
// the CUDA cores keep every SM busy and need no set-up. A warp has four weight rows and every `split`-th
// part of K; a lane multiplies 16 bytes of each with the tokens' (in shared memory) by dp4a, sixteen
// such loads in flight. Two rows per warp, blocks of 64 threads and asking for the weights' lines
// ahead (into L2, before the wait for the previous kernel) were no faster.
constexpr int kGemvTokens = 4;
constexpr int kGemvRows = 4;          // weight rows per warp
constexpr int kGemvThreads = 256;
constexpr int kGemvSmem = 46 * 1024;  // tokens in shared memory, beside part, without an opt-in

template <int M>
__global__ void __launch_bounds__(kGemvThreads)
    k_int8_gemv(const uint4* a, const uint4* w, const I8Args args, int kv, int split) {
  extern __shared__ uint4 tokens[];   // [M][kv]
  __shared__ int part[8][kGemvRows * M];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / split, slice = warp - group * split;  // row group of the block, K part
  const int n0 = (blockIdx.x * (8 / split) + group) * kGemvRows;
  const int k0 = slice * kv / split, k1 = (slice + 1) * kv / split;
  const uint4* row[kGemvRows];
#pragma unroll
  for (int r = 0; r < kGemvRows; ++r)  // rows behind the last are the last, and are not stored
    row[r] = w + static_cast<int64_t>(min(n0 + r, args.N - 1)) * kv;
  pdl_begin_in_order();
  for (int i = threadIdx.x; i < M * kv; i += kGemvThreads) tokens[i] = __ldcg(a + i);
  __syncthreads();
  int acc[kGemvRows][M] = {};
#pragma unroll 4
  for (int k = k0 + lane; k < k1; k += 32) {
    uint4 q[kGemvRows];
#pragma unroll
    for (int r = 0; r < kGemvRows; ++r) q[r] = __ldcg(row[r] + k);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 t = tokens[m * kv + k];
#pragma unroll
      for (int r = 0; r < kGemvRows; ++r) {
        int s = acc[r][m];
        s = __dp4a(static_cast<int>(q[r].x), static_cast<int>(t.x), s);
        s = __dp4a(static_cast<int>(q[r].y), static_cast<int>(t.y), s);
        s = __dp4a(static_cast<int>(q[r].z), static_cast<int>(t.z), s);
        acc[r][m] = __dp4a(static_cast<int>(q[r].w), static_cast<int>(t.w), s);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kGemvRows; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
      if (lane == 0) part[warp][r * M + m] = sum;
    }
  __syncthreads();
  // a thread per row group, row and token
  const int i = threadIdx.x;
  if (i >= (8 / split) * kGemvRows * M) return;
  const int grp = i / (kGemvRows * M), rm = i % (kGemvRows * M);
  const int n = (blockIdx.x * (8 / split) + grp) * kGemvRows + rm / M, m = rm % M;
  if (n >= args.N) return;
  int sum = 0;
  for (int s = 0; s < split; ++s) sum += part[grp * split + s][rm];
  const float y = fmaf(static_cast<float>(sum) * __ldcg(args.a_scale + m), __ldcg(args.w_scale + n),
                       args.bias ? __ldcg(args.bias + n) : 0.0f);
  store_out(args.out, args.dtype, static_cast<int64_t>(m) * args.N + n, y);
}

// ------------------------------------------------------------------ CTA pairs
// For many tokens: two CTAs share a tile of 256 weight rows x up to 256 tokens. One MMA
// (cta_group::2, M = 256) reads both CTAs' shared memory: each holds its own 128 weight rows and
// half of the tokens, so a K block costs an SM 32 KB of shared-memory fill instead of 48 for the same
// 128 x 256 outputs. 8192 x 4096 x 7168 takes 162 us (3.0 POP/s), with one CTA per tile 192. Without
// the loads and stores its MMAs take 111 us on what shared memory happens to hold; real operands
// draw more power and lower the clock.
//
// Both CTAs load into their own stages and count on the leader's (rank 0's) barrier; the leader
// issues the MMAs and commits to the barriers of both. Each CTA stores its own weight rows' outputs.
constexpr int kPairTokens = 256;
constexpr int kPairBlock = (kWRows + kPairTokens / 2) * kKB;  // 32 KB
constexpr int kPairStage = kSub * kPairBlock;
constexpr int kPairStages = 3;
constexpr int kPairBox = 32;                                  // token rows per TMA box

struct alignas(16) PairTail {
  uint64_t full[kPairStages];   // the leader's are used: one arrival and both CTAs' bytes
  uint64_t empty[kPairStages];
  uint64_t tfull[2];
  uint64_t tempty[2];           // the leader's: every epilogue warp of both CTAs
  uint64_t drain;
  uint64_t never;
  uint32_t tmem_base;
  int abort_flag;
  int tiles;
  int live;
  int gave_up;                  // set in every CTA of the cluster after a leader's abort
  int last_round[kPairStages];  // the latest round of copies that this CTA issued into the stage,
  int last_bytes[kPairStages];  // -1 for none, and its bytes
  alignas(16) float a_scale[kPairTokens];
  int ebase[kMaxLocalExperts + 1];
  int etile[kMaxLocalExperts + 1];
};
constexpr size_t kPairSmem = static_cast<size_t>(kPairStages) * kPairStage + sizeof(PairTail) + 1024;
static_assert((kPairTokens + 4 * 15) * kWRows * 4 <= kPairStages * kPairStage,
              "four shares of a tile's partial sums fit the stages");
static_assert(kPairSmem <= 227 * 1024, "pair shared memory");
static_assert(kPairStages == kI8Producers, "a stage has one producer: parity, last_round");

// Loads a box into this CTA's shared memory, its bytes counted on a barrier of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const void* tmap, uint32_t bar, int32_t c0,
                                              int32_t c1, uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "l"(hint)
      : "memory");
}

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on the barrier at `bar`'s place in both CTAs of the pair when the issued MMAs have
// finished.
__device__ __forceinline__ void commit_pair(uint64_t* bar, int lead) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3 << lead))
      : "memory");
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Tiles of 256 weight rows, otherwise as decode_tile: expert, weight tile, token tile (fastest);
// the tokens of a tile are cut in two halves of a multiple of 16.
__device__ __forceinline__ I8Tile decode_pair(int tile, int NT, const PairTail* t, int E) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
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
  const int per = ((count + mt - 1) / mt + 31) / 32 * 32;  // at most 256
  I8Tile r;
  r.e = lo;
  r.n0 = n * 2 * kWRows;
  r.row0 = t->ebase[lo] + static_cast<int64_t>(m) * per;
  r.rows = max(0, min(per, count - m * per));
  r.cols = max(32, (r.rows + 31) / 32 * 32);
  return r;
}

__device__ __forceinline__ void pair_abort(PairTail* t) {
  *reinterpret_cast<volatile int*>(&t->abort_flag) = 1;
  atomicOr(&g_int8_status, FMOE_STATUS_TIMEOUT_INT8);
}

// After an abort, by the leader once no role of either CTA issues any more: waits (bounded) until the
// copies issued into every stage have landed, in both CTAs. A round needs both CTAs' copies and the
// next needs both CTAs' stages, so a CTA is at most one round ahead of the other; the half of a
// round that was never issued is taken off what the barrier expects.
__device__ __forceinline__ void pair_drain(PairTail* t, int peer) {
  for (int s = 0; s < kPairStages; ++s) {
    const int mine = t->last_round[s], other = ld_dsmem_s32(&t->last_round[s], peer);
    const int r = max(mine, other);
    if (r < 0) continue;
    if (mine < r) {
      mbar_arrive_expect_tx(&t->full[s], ld_dsmem_s32(&t->last_bytes[s], peer));
    } else if (other < r) {
      asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(
                       smem_u32(&t->full[s])),
                   "r"(t->last_bytes[s])
                   : "memory");
    }
    (void)mbar_wait(&t->full[s], r & 1);
  }
}

// SPLIT: the S pairs of a cluster share one tile, each with a range of K.
template <bool SPLIT>
__global__ void __launch_bounds__(kI8Threads, 1)
    k_int8_pair(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                const I8Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  PairTail* tail = reinterpret_cast<PairTail*>(smem + kPairStages * kPairStage);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = args.E;
  const int NT = (args.N + 2 * kWRows - 1) / (2 * kWRows);
  const int S = SPLIT ? args.S : 1;
  const int cta = static_cast<int>(cluster_ctarank());
  const int rank = cta & 1, lead = cta & ~1;  // in the pair; the pair's leader in the cluster

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tail->tfull[b], 1);
      mbar_init(&tail->tempty[b], 2 * kI8EpiWarps);
    }
    mbar_init(&tail->drain, 1);
    mbar_init(&tail->never, 1);
    tail->abort_flag = 0;
    tail->gave_up = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tail->tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  pdl_begin_in_order();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    int64_t b = args.expert_base ? __ldcg(args.expert_base + e) : (e == 0 ? 0 : args.M);
    tail->ebase[e] = static_cast<int>(b < 0 ? 0 : b > args.M ? args.M : b);
  }
  __syncthreads();
  if (warp == 0) {
    ascending_bases(tail->ebase, E, args.expert_base != nullptr);
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int mt = 0;
      if (e < E) mt = (max(0, tail->ebase[e + 1] - tail->ebase[e]) + kPairTokens - 1) / kPairTokens;
      int incl = mt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (e < E) tail->etile[e] = carry + incl - mt;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      tail->etile[E] = carry;
      tail->tiles = carry * NT;
      tail->live = tail->ebase[E];
    }
  }
  tc_fence_before();
  __syncthreads();
  // both CTAs' barriers are initialised and both have their tensor memory
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  const int tiles = tail->tiles;
  // SPLIT: at most one tile per cluster
  const int first = SPLIT ? blockIdx.x / (2 * S) : blockIdx.x >> 1;
  const int step = SPLIT ? gridDim.x / (2 * S) : gridDim.x >> 1;
  const int kb0 = (cta >> 1) * args.nkb / S, kb1 = ((cta >> 1) + 1) * args.nkb / S;

  if (warp == 0 || warp == 2 || warp == 3) {
    // ---------------------------------------------------------------- TMA producers
    const int pw = warp == 0 ? 0 : warp - 1;
    if (lane == 0) {
      const uint64_t pol_first = policy_evict_first();
      const uint64_t pol_last = policy_evict_last();
      tail->last_round[pw] = -1;
      int it = 0;
      // the injected failure also leaves rounds that one CTA of the pair alone has issued
      bool ok = args.inject == 0 || pw != 2 - rank;
      for (int tile = first; tile < tiles && ok; tile += step) {
        const I8Tile u = decode_pair(tile, NT, tail, E);
        const int half = u.cols / 2;
        const int boxes = (half + kPairBox - 1) / kPairBox;
        const uint32_t block_bytes = 2 * (kWRows + boxes * kPairBox) * kKB;
        const uint64_t pol_w =
            tail->etile[u.e + 1] - tail->etile[u.e] > 1 ? pol_last : pol_first;
        const int wrow = u.e * args.N + u.n0 + rank * kWRows;
        const int arow = static_cast<int>(u.row0) + rank * half;
        for (int kb = kb0; kb < kb1; kb += kSub, ++it) {
          if (it % kI8Producers != pw) continue;
          const int s = it % kPairStages, r = it / kPairStages;
          if (r > 0 && !parked_wait(&tail->empty[s], (r & 1) ^ 1, abort_flag, args.wait_ns)) {
            pair_abort(tail);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kPairStage;
          const int blocks = min(kSub, kb1 - kb);
          if (rank == 0) mbar_arrive_expect_tx(&tail->full[s], blocks * block_bytes);
          const uint32_t bar = at_rank(&tail->full[s], lead);
          for (int j = 0; j < blocks; ++j, st += kPairBlock) {
            const int k = (kb + j) * kKB;
            tma_load_pair(st, &tm_w, bar, k, wrow, pol_w);
            for (int b = 0; b < boxes; ++b)
              tma_load_pair(st + (kWRows + b * kPairBox) * kKB, &tm_a, bar, k, arow + b * kPairBox,
                            pol_last);
          }
          tail->last_round[s] = r;
          tail->last_bytes[s] = blocks * (block_bytes / 2);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (the leader's)
    if (rank == 0 && elect_one()) {
      int it = 0, n = 0;
      bool ok = args.inject == 0 || parked_wait(&tail->never, 0, abort_flag, args.wait_ns);
      for (int tile = first; tile < tiles && ok; tile += step, ++n) {
        const I8Tile u = decode_pair(tile, NT, tail, E);
        const uint32_t idesc = idesc_i8(2 * kWRows, u.cols);
        const int b = n & 1, rb = n >> 1;
        const uint32_t d = tmem + b * kPairTokens;
        if (rb > 0 && !parked_wait(&tail->tempty[b], (rb & 1) ^ 1, abort_flag, args.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t more = 0;
        for (int kb = kb0; kb < kb1; kb += kSub, ++it) {
          const int s = it % kPairStages, r = it / kPairStages;
          if (!parked_wait(&tail->full[s], r & 1, abort_flag, args.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t st = smem_u32(smem + s * kPairStage);
          for (int left = min(kSub, kb1 - kb); left > 0; --left, st += kPairBlock) {
            const uint64_t w_desc = smem_desc_k128(st);
            const uint64_t a_desc = smem_desc_k128(st + kWRows * kKB);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma_i8_pair(d, w_desc + 2 * j, a_desc + 2 * j, idesc, more);
              more = 1u;
            }
          }
          commit_pair(&tail->empty[s], lead);
        }
        if (ok) commit_pair(&tail->tfull[b], lead);
      }
      if (!ok) pair_abort(tail);
      commit_pair(&tail->drain, lead);
    }
    if (lane == 0) (void)mbar_wait(&tail->drain, 0);
  } else {
    // ---------------------------------------------------------------- epilogue
    const int q = warp & 3;
    const int g = (warp - kI8Epi0) >> 2;
    const int etid = threadIdx.x - kI8Epi0 * 32;
    const uint32_t tempty[2] = {at_rank(&tail->tempty[0], lead), at_rank(&tail->tempty[1], lead)};
    if (args.zero_tail) {  // rows of no expert
      const int64_t tid = static_cast<int64_t>(blockIdx.x) * (kI8EpiWarps * 32) + etid;
      const int64_t threads = static_cast<int64_t>(gridDim.x) * (kI8EpiWarps * 32);
      zero_rows_out(args, 0, tail->ebase[0], tid, threads);
      zero_rows_out(args, tail->live, args.M, tid, threads);
    }
    int n = 0;
    bool ok = true;
    for (int tile = first; tile < tiles; tile += step, ++n) {
      const I8Tile u = decode_pair(tile, NT, tail, E);
      const int b = n & 1, rb = n >> 1;
      const int ch = u.n0 + rank * kWRows + q * 32 + lane;
      const bool live = ch < args.N;
      const float ws = live ? __ldcg(args.w_scale + static_cast<int64_t>(u.e) * args.N + ch) : 0.0f;
      const float bias = live && args.bias ? __ldcg(args.bias + ch) : 0.0f;
      named_bar_sync(1, kI8EpiWarps * 32);  // the previous tile's a_scale is no longer read
      if (etid < u.rows) tail->a_scale[etid] = __ldcg(args.a_scale + u.row0 + etid);
      named_bar_sync(1, kI8EpiWarps * 32);
      // after a wait that ran out, the warp still takes part in the barriers of later tiles
      if (ok) ok = __all_sync(0xffffffffu, parked_wait(&tail->tfull[b], rb & 1, abort_flag, args.wait_ns));
      if (!ok) {
        if (lane == 0) pair_abort(tail);
        continue;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * kPairTokens;
      if constexpr (!SPLIT)
        store_columns(args, taddr, g * 16, kI8EpiCols, u, u.n0 + rank * kWRows + q * 32,
                      tail->a_scale, ws, bias);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(tempty[b]);
    }
  }

  tc_fence_before();
  __syncthreads();
  // Never leave a bulk copy in flight into shared memory that is about to be released. Without an
  // abort of the leader its MMAs have waited for all of them.
  if (threadIdx.x == 0 && rank == 0 && *abort_flag)
    for (int c = 0; c < 2 * S; ++c)
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at_rank(&tail->gave_up, c)), "r"(1)
                   : "memory");
  cluster_arrive();  // every pair's MMAs are done, their stages free
  cluster_wait();
  tc_fence_after();
  if (*reinterpret_cast<volatile int*>(&tail->gave_up)) {
    if (threadIdx.x == 0 && rank == 0) pair_drain(tail, cta + 1);
    cluster_arrive();
    cluster_wait();
  }
  if constexpr (SPLIT) {
    const I8Tile u = first < tiles ? decode_pair(first, NT, tail, E) : I8Tile{};
    const int per = split_share(u.rows, S);
    if (warp >= kI8Epi0 && u.rows > 0)
      send_partials(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), (warp - kI8Epi0) >> 2, u,
                    per, smem, cta >> 1, rank, 2, (warp & 3) * 32 + lane);
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    if (u.rows > 0) finish_split(args, u, u.n0 + rank * kWRows, per, smem, S, cta >> 1);
    // the pair gives its tensor memory back together
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

template <int BN, bool SPLIT>
cudaError_t launch_mm(const CUtensorMap& tm_a, const CUtensorMap& tm_w, const I8Args& a, int grid,
                      cudaStream_t s) {
  const size_t smem = i8_smem_bytes<BN>();
  if constexpr (SPLIT)
    return launch_pdl_cluster(k_int8_mm<BN, true>, dim3(grid), dim3(kI8Threads), smem, s, a.S, tm_a,
                              tm_w, a);
  else
    return launch_pdl(k_int8_mm<BN, false>, dim3(grid), dim3(kI8Threads), smem, s, tm_a, tm_w, a);
}

// How many clusters of `size` CTAs, one CTA per SM, run at a time on the current device: fewer than
// SMs / size, by the sizes of its SM groups (33 of 4, 22 of 6, 15 of 8 where 148 SMs are in use).
// Asked once per device and size.
int max_clusters(int size, int dev) {
  static std::atomic<int> known[64][9];
  int n = known[dev][size].load(std::memory_order_acquire);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size * 64);
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = kPairSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, k_int8_pair<true>, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 1;
  }
  known[dev][size].store(n, std::memory_order_release);
  return n;
}

struct I8Plan {
  int bn, S;  // bn 256: CTA pairs
};

// The tile width and K split with the shortest estimated time in cycles: rounds of tiles over the
// SMs times the K blocks of a tile, a K block costing the slower of its round in the MMA warp (640
// cycles, however few the tokens) and its fill of shared memory (about 75 bytes a cycle); then the last
// tile's stores, the exchange of partial tiles and the cluster's barriers where K is split, and a
// pair's own set-up. An expert is taken to have up to twice its even share: with the even share alone
// the worst choice was 30% off.
// The constants are of a loop that issued its MMAs for lane 0. Under elect.sync a round takes about a
// third less, so 640 is too long: it hides the widths' differences, and splits look better than they
// are. Against every width and split on the present kernels: 113 products of 5 to 8192 tokens 3.6%
// from the fastest on average, 30% at worst (2048 x 512 x 7168: 16.4 us, with 64-token tiles 12.6; 256 x
// 4096 x 7168: 17.1, 14.5), 30 of experts (8 to 8192 rows) 1.1% and 10%; within 1% for two in three.
I8Plan i8_plan(int64_t M, int N, int E, int nkb, bool grouped, int sms, int dev) {
  const int64_t used = M < E ? M : E;
  int64_t per = (M + used - 1) / used;
  if (grouped) per = 2 * per < M ? 2 * per : M;
  I8Plan best{256, 1};
  double best_cost = 1e30;
  for (const int bn : {16, 64, 128, 256}) {
    const int ctas = bn == 256 ? 2 : 1;
    const int64_t NT = (N + ctas * kWRows - 1) / (ctas * kWRows);
    const int64_t mt = (per + bn - 1) / bn;
    const int64_t tiles = mt * used * NT;
    const int64_t most = (grouped ? M / bn + used : mt) * NT;  // no spread has more tiles
    const int64_t cols = ((per + mt - 1) / mt + 15) / 16 * 16;
    const double fill = (kWRows + cols / ctas) * kKB / 75.0;
    const double kb = fill > 640.0 ? fill : 640.0;
    for (int S = 1; S <= 4; ++S) {
      if (S > 1 && (nkb < 2 * S || most > max_clusters(S * ctas, dev))) break;
      const int64_t waves = S > 1 ? 1 : (tiles + sms / ctas - 1) / (sms / ctas);
      const double cost = waves * ((nkb + S - 1) / S) * kb + cols * 50.0 +
                          (ctas > 1 ? 2300.0 : 0.0) + (S > 1 ? cols * 50.0 + 5400.0 : 0.0);
      if (cost < best_cost) {
        best_cost = cost;
        best = I8Plan{bn, S};
      }
    }
  }
  return best;
}

I8Args i8_args(const Int8Product& p, int S) {
  I8Args a{};
  a.a_scale = p.a_scale;
  a.w_scale = p.w_scale;
  a.bias = p.bias;
  a.expert_base = p.expert_base;
  a.out = p.out;
  a.M = p.M;
  a.N = p.N;
  a.E = p.E;
  a.nkb = (p.K + kKB - 1) / kKB;
  a.S = S;
  a.dtype = p.out_dtype;
  a.zero_tail = p.zero_tail;
  a.wait_ns = p.wait_ns != 0 ? p.wait_ns : FMOE_WAIT_NS;
  a.inject = p.wait_ns != 0;
  return a;
}

bool i8_maps(const Int8Product& p, int box, CUtensorMap* tm_a, CUtensorMap* tm_w) {
  return tensor_map_u8(tm_a, p.a, p.K, p.M, p.K, kKB, box) &&
         tensor_map_u8(tm_w, p.w, p.K, static_cast<uint64_t>(p.E) * p.N, p.K, kKB, kWRows);
}

// The most tiles of bn tokens that any spread of the rows over the experts has, per weight tile.
int64_t most_token_tiles(const Int8Product& p, int bn) {
  const int64_t used = p.M < p.E ? p.M : p.E;
  return p.expert_base ? p.M / bn + used : (p.M + bn - 1) / bn;
}

template <int BN>
cudaError_t run_mm(const Int8Product& p, int S, int sms, cudaStream_t s) {
  CUtensorMap tm_a, tm_w;
  if (!i8_maps(p, I8Cfg<BN>::BOX, &tm_a, &tm_w)) return cudaErrorInvalidValue;
  const I8Args a = i8_args(p, S);
  int64_t most = most_token_tiles(p, BN) * ((p.N + kWRows - 1) / kWRows);
  if (S > 1) return launch_mm<BN, true>(tm_a, tm_w, a, static_cast<int>(most * S), s);
  if (most > sms) most = sms;
  return launch_mm<BN, false>(tm_a, tm_w, a, static_cast<int>(most), s);
}

template <bool SPLIT>
cudaError_t launch_pair(const Int8Product& p, int S, int sms, cudaStream_t s) {
  CUtensorMap tm_a, tm_w;
  if (!i8_maps(p, kPairBox, &tm_a, &tm_w)) return cudaErrorInvalidValue;
  const int64_t tiles = most_token_tiles(p, kPairTokens) * ((p.N + 2 * kWRows - 1) / (2 * kWRows));
  const int64_t clusters = SPLIT || tiles < sms / 2 ? tiles : sms / 2;
  return launch_pdl_cluster(k_int8_pair<SPLIT>, dim3(static_cast<unsigned>(2 * S * clusters)),
                            dim3(kI8Threads), kPairSmem, s, 2 * S, tm_a, tm_w, i8_args(p, S));
}

// K is split until there are sixteen warps per SM, or a warp has less than four steps.
template <int M>
cudaError_t launch_gemv(const Int8Product& p, int sms, cudaStream_t s) {
  const int kv = p.K / 16;
  int split = 1;
  while (split < 8 && static_cast<int64_t>((p.N + kGemvRows - 1) / kGemvRows) * split < 16 * sms &&
         kv / (2 * split) >= 128)
    split *= 2;
  const int rows = 8 / split * kGemvRows;
  return launch_pdl(k_int8_gemv<M>, dim3((p.N + rows - 1) / rows), dim3(kGemvThreads),
                    static_cast<size_t>(M) * p.K, s, static_cast<const uint4*>(p.a),
                    static_cast<const uint4*>(p.w), i8_args(p, 1), kv, split);
}

// The shared-memory opt-in of every kernel, once per device (idempotent).
cudaError_t configure(int dev) {
  static std::atomic<bool> done[64];
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const auto set = [](const void* f, size_t bytes) {
    return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(bytes));
  };
  cudaError_t e = set(reinterpret_cast<const void*>(k_int8_pair<false>), kPairSmem);
  if (e == cudaSuccess) e = set(reinterpret_cast<const void*>(k_int8_pair<true>), kPairSmem);
#define SET(BN, SPLIT) \
  if (e == cudaSuccess) \
    e = set(reinterpret_cast<const void*>(k_int8_mm<BN, SPLIT>), i8_smem_bytes<BN>());
  SET(16, false) SET(16, true) SET(64, false) SET(64, true) SET(128, false) SET(128, true)
#undef SET
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
  return e;
}

}  // namespace

cudaError_t launch_quantize_int8(const void* x, int dtype, int64_t rows, int64_t K, void* q,
                                 float* scale, int sms, cudaStream_t s) {
  const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0 &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  if (dtype == FMOE_DTYPE_BF16)
    return vec ? quantize_rows<__nv_bfloat16, true>(x, rows, K, q, scale, sms, s)
               : quantize_rows<__nv_bfloat16, false>(x, rows, K, q, scale, sms, s);
  return vec ? quantize_rows<__half, true>(x, rows, K, q, scale, sms, s)
             : quantize_rows<__half, false>(x, rows, K, q, scale, sms, s);
}

cudaError_t launch_int8_product(const Int8Product& p, int sms, cudaStream_t s) {
  // The tensor cores take 10.4 us for 1 to 4 tokens x 4096 x 7168, this way 1, 2 and 4 tokens take 8.0,
  // 9.2 and 9.0 (2048 x 2048: 5.6 against 2.8, 3.3 and 3.2). More channels are enough tiles for every
  // SM: 9472 x 7168 takes 14.6 and 14.2, 17.3 and 15.3, 16384 x 7168 takes 20.9, and 20.6 and 22.3 for one
  // token and two. With short rows the set-up counts again: 9472 x 1024 takes 5.0 against 2.8, 2.9 and 4.0.
  if (p.wait_ns == 0 && p.tile_tokens == 0 && !p.expert_base && p.M <= kGemvTokens &&
      p.M * p.K <= kGemvSmem && (p.M <= 2 || p.N <= 64 * sms)) {
    switch (p.M) {
      case 1:
        return launch_gemv<1>(p, sms, s);
      case 2:
        return launch_gemv<2>(p, sms, s);
      case 3:
        return launch_gemv<3>(p, sms, s);
      default:
        return launch_gemv<4>(p, sms, s);
    }
  }
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  const cudaError_t e = configure(dev);
  if (e != cudaSuccess) return e;
  const I8Plan plan = p.tile_tokens != 0
                          ? I8Plan{p.tile_tokens, p.split}
                          : i8_plan(p.M, p.N, p.E, (p.K + kKB - 1) / kKB, p.expert_base != nullptr,
                                    sms, dev);
  switch (plan.bn) {
    case 16:
      return run_mm<16>(p, plan.S, sms, s);
    case 64:
      return run_mm<64>(p, plan.S, sms, s);
    case 128:
      return run_mm<128>(p, plan.S, sms, s);
    default:
      return plan.S > 1 ? launch_pair<true>(p, plan.S, sms, s)
                        : launch_pair<false>(p, 1, sms, s);
  }
}

cudaError_t take_int8_status(int32_t* status, cudaStream_t s) {
  static std::mutex one_at_a_time;  // g_int8_taken is one call's until it has been copied out
  const std::lock_guard<std::mutex> hold(one_at_a_time);
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_int8_taken);
  if (e != cudaSuccess) return e;
  k_take_int8_status<<<1, 1, 0, s>>>();
  e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, sizeof(int32_t), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e;
}

}  // namespace fmoe
