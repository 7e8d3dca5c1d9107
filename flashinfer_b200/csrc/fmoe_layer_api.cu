// fmoe_layer_api.cu -- argument checks and launches of the operators around the experts
// (include/fmoe.h): tokens sorted by expert and back, int8 and int4 products, norms, balance loss.
#include <initializer_list>

#include "fmoe_internal.h"

namespace fmoe {
namespace {

bool at(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

size_t elem(int dtype) { return dtype == FMOE_DTYPE_F32 ? 4 : 2; }

bool float_type(int dtype) {
  return dtype == FMOE_DTYPE_F32 || dtype == FMOE_DTYPE_BF16 || dtype == FMOE_DTYPE_F16;
}

struct Span {
  const void* p;
  uint64_t bytes;
};

// Whether an output shares a byte with an input or with another output.
bool overlap(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  const auto hit = [](const Span& a, const Span& b) {
    if (!a.p || !b.p || a.bytes == 0 || b.bytes == 0) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x < y + b.bytes && y < x + a.bytes;
  };
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    for (const Span& i : ins)
      if (hit(*o, i)) return true;
    for (auto p = outs.begin(); p != o; ++p)
      if (hit(*o, *p)) return true;
  }
  return false;
}

int done(cudaError_t e) { return e == cudaSuccess ? FMOE_OK : FMOE_ERR_CUDA; }

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

int order_size(int32_t T, int32_t K, int32_t E, int32_t align, int64_t* rows, size_t* scratch) {
  if (T < 0 || K < 1 || E < 1 || E > kMaxOrderExperts || align < 1 || align > 1024)
    return FMOE_ERR_SHAPE;
  const int64_t picks = static_cast<int64_t>(T) * K;
  const int64_t n = picks + (picks < E ? picks : E) * static_cast<int64_t>(align - 1);
  if (n > INT32_MAX - 1024) return FMOE_ERR_SHAPE;
  *rows = n;
  *scratch = order_scratch_bytes(picks, E);
  return FMOE_OK;
}

int check_order(const FmoeTokenOrder* o, TokenOrder* out) {
  if (!o) return FMOE_ERR_NULL;
  int64_t least = 0;
  size_t scratch = 0;
  const int rc = order_size(o->num_tokens, o->top_k, o->num_local_experts, 1, &least, &scratch);
  if (rc) return rc;
  if (o->num_rows < least || o->num_rows > INT32_MAX - 1024) return FMOE_ERR_SHAPE;
  if (!o->expert_base || (o->num_rows > 0 && !o->row_pick) || (o->num_tokens > 0 && !o->pick_row))
    return FMOE_ERR_NULL;
  if (!at(o->expert_base, 4) || !at(o->row_pick, 4) || !at(o->pick_row, 4)) return FMOE_ERR_ALIGN;
  *out = TokenOrder{o->expert_base, o->row_pick, o->pick_row, o->num_tokens,
                    o->top_k,       o->num_local_experts, o->num_rows};
  return FMOE_OK;
}

// Blocks of 256 threads along every row must fit one grid dimension.
bool grid_fits(int64_t rows, int64_t units) { return rows * (units / 256 + 1) < INT32_MAX - 4096; }

// One-shot failure-path injection of fmoe_debug_arm_int8_timeout for this host thread's next product.
thread_local unsigned long long g_int8_wait_ns = 0;
// One-shot choice of fmoe_debug_arm_int8_plan for this host thread's next product.
thread_local int g_int8_tile_tokens = 0, g_int8_split = 0;
// The same two for the products with 4-bit weights.
thread_local unsigned long long g_int4_wait_ns = 0;
thread_local int g_int4_tile_tokens = 0, g_int4_split = 0;

int int8_product(const Int8Product& call, void* stream) {
  Int8Product p = call;
  p.wait_ns = g_int8_wait_ns;
  p.tile_tokens = g_int8_tile_tokens;
  p.split = g_int8_split;
  g_int8_wait_ns = 0;
  g_int8_tile_tokens = g_int8_split = 0;
  if (p.M < 0 || p.M > INT32_MAX - 1024 || p.N < 1 || p.K < 16 || p.K % 16 != 0 || p.K > 131056 ||
      p.E < 1 || p.E > kMaxLocalExperts ||
      static_cast<int64_t>(p.E) * p.N > INT32_MAX - 1024)
    return FMOE_ERR_SHAPE;
  if (!float_type(p.out_dtype)) return FMOE_ERR_DTYPE;
  if (p.M == 0) return FMOE_OK;
  // every part of a split needs a K block, every tile a block of the grid
  if (p.tile_tokens != 0 &&
      ((p.K + 127) / 128 < p.split ||
       (p.M / p.tile_tokens + p.E) * ((p.N + 127) / 128) * 8 > INT32_MAX))
    return FMOE_ERR_SHAPE;
  for (const void* q : {p.a, p.w, static_cast<const void*>(p.a_scale),
                        static_cast<const void*>(p.w_scale), static_cast<const void*>(p.out)})
    if (!q) return FMOE_ERR_NULL;
  if (!at(p.a, 16) || !at(p.w, 16) || !at(p.a_scale, 4) || !at(p.w_scale, 4) || !at(p.bias, 4) ||
      !at(p.expert_base, 4) || !at(p.out, elem(p.out_dtype)))
    return FMOE_ERR_ALIGN;
  const uint64_t EN = static_cast<uint64_t>(p.E) * p.N;
  if (overlap({{p.out, static_cast<uint64_t>(p.M) * p.N * elem(p.out_dtype)}},
              {{p.a, static_cast<uint64_t>(p.M) * p.K},
               {p.w, EN * p.K},
               {p.a_scale, static_cast<uint64_t>(p.M) * 4},
               {p.w_scale, EN * 4},
               {p.bias, static_cast<uint64_t>(p.N) * 4},
               {p.expert_base, static_cast<uint64_t>(p.E + 1) * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_int8_product(p, sms, as_stream(stream)));
}

size_t norm_workspace(int64_t T, int H) {
  return static_cast<size_t>(3) * (T < kMaxNormBlocks ? T : kMaxNormBlocks) * H * 4;
}

// What the forward and the backward pass have in common.
int check_norm(const FmoeBlockNormArgs* a, BlockNorm* p) {
  if (!a) return FMOE_ERR_NULL;
  if (a->num_tokens < 0 || a->num_tokens > INT32_MAX - 1024 || a->hidden_size < 1 ||
      a->hidden_size > 16384 || a->gate_kind < FMOE_GATE_NONE || a->gate_kind > FMOE_GATE_FULL)
    return FMOE_ERR_SHAPE;
  if (!float_type(a->dtype)) return FMOE_ERR_DTYPE;
  const auto param = [&](const void* q, int dtype) {
    return !q || dtype == a->dtype || dtype == FMOE_DTYPE_F32;
  };
  if (!param(a->post_weight, a->post_weight_dtype) || !param(a->gate, a->gate_dtype) ||
      !param(a->pre_weight, a->pre_weight_dtype))
    return FMOE_ERR_DTYPE;
  if (a->num_tokens > 0) {
    if (!a->residual || (a->gate_kind != FMOE_GATE_NONE && !a->gate)) return FMOE_ERR_NULL;
    // without a block output there is nothing to normalise or to gate
    if (!a->branch && (a->post_weight || a->gate_kind != FMOE_GATE_NONE)) return FMOE_ERR_NULL;
  }
  *p = BlockNorm{};
  p->dtype = a->dtype;
  p->T = a->num_tokens;
  p->H = a->hidden_size;
  p->f = a->branch;
  p->x = a->residual;
  p->wp = a->post_weight;
  p->g = a->gate;
  p->wq = a->pre_weight;
  p->wp_dtype = a->post_weight_dtype;
  p->g_dtype = a->gate_dtype;
  p->wq_dtype = a->pre_weight_dtype;
  p->gate = a->gate_kind;
  p->s = a->residual_scale;
  p->eps = a->eps;
  p->stats = a->stats;
  const size_t e = elem(a->dtype);
  if (!at(a->branch, e) || !at(a->residual, e) || !at(a->stats, 4) ||
      (a->post_weight && !at(a->post_weight, elem(a->post_weight_dtype))) ||
      (a->gate && !at(a->gate, elem(a->gate_dtype))) ||
      (a->pre_weight && !at(a->pre_weight, elem(a->pre_weight_dtype))))
    return FMOE_ERR_ALIGN;
  return FMOE_OK;
}

uint64_t gate_count(const FmoeBlockNormArgs* a) {
  const uint64_t T = a->num_tokens, H = a->hidden_size;
  return a->gate_kind == FMOE_GATE_TOKEN ? T : a->gate_kind == FMOE_GATE_CHANNEL ? H
         : a->gate_kind == FMOE_GATE_FULL ? T * H : 0;
}

bool int4_group(int k, int group) {
  if (k < 32 || k % 32 != 0 || k > 131072 || group > INT32_MAX - 131072) return false;
  return group == 32 || group == 64 || (group > 0 && group % 128 == 0);
}

// Weights in 4 bits, given or wanted: the checks of both directions.
int check_int4_weights(const Int4Weights& p) {
  if (p.rows < 0 || p.rows > INT32_MAX - 1024) return FMOE_ERR_SHAPE;
  if (!float_type(p.dtype) || !float_type(p.scale_dtype)) return FMOE_ERR_DTYPE;
  if (p.rows == 0) return FMOE_OK;
  if (!p.w || !p.packed || !p.scale) return FMOE_ERR_NULL;
  if (!at(p.w, 16) || !at(p.packed, 16) || !at(p.scale, elem(p.scale_dtype))) return FMOE_ERR_ALIGN;
  return FMOE_OK;
}

size_t layer_norm_workspace(int64_t T, int H) {
  return static_cast<size_t>(2) * (T < kMaxLnBlocks ? T : kMaxLnBlocks) * H * 4;
}

// What the layer norm's forward and backward pass have in common.
int check_layer_norm(const FmoeLayerNormArgs* a, LayerNorm* p) {
  if (!a) return FMOE_ERR_NULL;
  if (a->num_tokens < 0 || a->num_tokens > INT32_MAX - 1024 || a->hidden_size < 1 ||
      a->hidden_size > 16384)
    return FMOE_ERR_SHAPE;
  if (!float_type(a->dtype)) return FMOE_ERR_DTYPE;
  const auto param = [&](const void* q, int dtype) {
    return !q || dtype == a->dtype || dtype == FMOE_DTYPE_F32;
  };
  if (!param(a->weight, a->weight_dtype) || !param(a->bias, a->bias_dtype)) return FMOE_ERR_DTYPE;
  if (a->num_tokens > 0 && !a->residual) return FMOE_ERR_NULL;
  const size_t e = elem(a->dtype);
  if (!at(a->branch, e) || !at(a->residual, e) || !at(a->stats, 8) ||
      (a->weight && !at(a->weight, elem(a->weight_dtype))) ||
      (a->bias && !at(a->bias, elem(a->bias_dtype))))
    return FMOE_ERR_ALIGN;
  *p = LayerNorm{};
  p->dtype = a->dtype;
  p->T = a->num_tokens;
  p->H = a->hidden_size;
  p->f = a->branch;
  p->x = a->residual;
  p->w = a->weight;
  p->b = a->bias;
  p->w_dtype = a->weight_dtype;
  p->b_dtype = a->bias_dtype;
  p->eps = a->eps;
  p->stats = a->stats;
  return FMOE_OK;
}

size_t balance_workspace(int64_t T, int E, int S) {
  const int64_t most = (T + 7) / 8;
  return static_cast<size_t>((most < kMaxBalanceBlocks ? most : kMaxBalanceBlocks) + S) * E * 8;
}

int check_balance(const FmoeBalanceArgs* a, Balance* p) {
  if (!a) return FMOE_ERR_NULL;
  if (a->num_tokens < 0 || a->num_tokens > INT32_MAX - 1024 || a->num_experts < 1 ||
      a->num_experts > kMaxBalanceExperts || a->top_k < 1 || a->num_sequences < 1 ||
      a->num_sequences > kMaxBalanceSequences || (!a->sequence_base && a->num_sequences != 1) ||
      (a->scoring != FMOE_SCORING_SOFTMAX && a->scoring != FMOE_SCORING_SIGMOID))
    return FMOE_ERR_SHAPE;
  if (!float_type(a->dtype)) return FMOE_ERR_DTYPE;
  if (!at(a->logits, elem(a->dtype)) || !at(a->topk_ids, 4) || !at(a->sequence_base, 4) ||
      !at(a->loss, 4) || !at(a->counts, 4) || !at(a->factor, 4) || !at(a->grad_loss, 4) ||
      !at(a->grad_logits, elem(a->dtype)) || !at(a->workspace, 4))
    return FMOE_ERR_ALIGN;
  *p = Balance{};
  p->logits = a->logits;
  p->dtype = a->dtype;
  p->ids = a->topk_ids;
  p->base = a->sequence_base;
  p->T = a->num_tokens;
  p->E = a->num_experts;
  p->K = a->top_k;
  p->S = a->num_sequences;
  p->sigmoid = a->scoring == FMOE_SCORING_SIGMOID;
  p->loss = a->loss;
  p->counts = a->counts;
  p->factor = a->factor;
  p->workspace = a->workspace;
  p->grad_loss = a->grad_loss;
  p->grad_logits = a->grad_logits;
  return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" {

int fmoe_sort_size(int32_t T, int32_t K, int32_t E, int32_t align, int64_t* num_rows,
                   size_t* scratch_bytes) {
  if (!num_rows || !scratch_bytes) return FMOE_ERR_NULL;
  return order_size(T, K, E, align, num_rows, scratch_bytes);
}

int fmoe_sort_by_expert(const int32_t* topk_ids, int32_t local_expert_offset, int32_t align,
                        const FmoeTokenOrder* order, void* scratch, size_t scratch_bytes,
                        void* stream) {
  TokenOrder o;
  int rc = check_order(order, &o);
  if (rc) return rc;
  int64_t rows = 0;
  size_t need = 0;
  rc = order_size(o.T, o.K, o.E, align, &rows, &need);
  if (rc) return rc;
  if (o.R < rows) return FMOE_ERR_SHAPE;
  if (local_expert_offset < 0) return FMOE_ERR_OFFSET;
  if (o.T > 0 && !topk_ids) return FMOE_ERR_NULL;
  if (!at(topk_ids, 4) || !at(scratch, 4)) return FMOE_ERR_ALIGN;
  if (need > 0 && (!scratch || scratch_bytes < need)) return FMOE_ERR_WORKSPACE;
  const uint64_t picks = static_cast<uint64_t>(o.T) * o.K;
  if (overlap({{o.expert_base, static_cast<uint64_t>(o.E + 1) * 4},
               {o.row_pick, static_cast<uint64_t>(o.R) * 4},
               {o.pick_row, picks * 4},
               {scratch, need}},
              {{topk_ids, picks * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_order(topk_ids, o, local_expert_offset, align, order->expert_base,
                           order->row_pick, order->pick_row, static_cast<int32_t*>(scratch),
                           as_stream(stream)));
}

int fmoe_sort_rows(const void* x, int64_t row_bytes, const FmoeTokenOrder* order, void* rows,
                   int32_t zero_tail, void* stream) {
  TokenOrder o;
  int rc = check_order(order, &o);
  if (rc) return rc;
  if (row_bytes < 1 || row_bytes > INT32_MAX || !grid_fits(o.T, row_bytes)) return FMOE_ERR_SHAPE;
  if (o.T == 0 && !(zero_tail && o.R > 0)) return FMOE_OK;
  if ((o.T > 0 && !x) || !rows) return FMOE_ERR_NULL;
  if (overlap({{rows, static_cast<uint64_t>(o.R) * row_bytes}},
              {{x, static_cast<uint64_t>(o.T) * row_bytes}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_sort_rows(x, rows, o, row_bytes, zero_tail, sms, as_stream(stream)));
}

int fmoe_unsort_rows(const void* rows, int32_t dtype, int64_t H, const FmoeTokenOrder* order,
                     const float* weights, void* y, void* stream) {
  TokenOrder o;
  int rc = check_order(order, &o);
  if (rc) return rc;
  if (!float_type(dtype)) return FMOE_ERR_DTYPE;
  if (H < 1 || H > (INT32_MAX >> 2) || !grid_fits(o.T, H)) return FMOE_ERR_SHAPE;
  if (o.T == 0) return FMOE_OK;
  if (!rows || !y) return FMOE_ERR_NULL;
  const size_t e = elem(dtype);
  if (!at(rows, e) || !at(y, e) || !at(weights, 4)) return FMOE_ERR_ALIGN;
  if (overlap({{y, static_cast<uint64_t>(o.T) * H * e}},
              {{rows, static_cast<uint64_t>(o.R) * H * e},
               {weights, static_cast<uint64_t>(o.T) * o.K * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_unsort_rows(rows, weights, y, dtype, o, H, as_stream(stream)));
}

int fmoe_unsort_rows_backward(const void* grad_y, const void* rows, int32_t dtype, int64_t H,
                              const FmoeTokenOrder* order, const float* weights, void* grad_rows,
                              float* grad_weights, void* stream) {
  TokenOrder o;
  int rc = check_order(order, &o);
  if (rc) return rc;
  if (!float_type(dtype)) return FMOE_ERR_DTYPE;
  if (H < 1 || H > (INT32_MAX >> 2) || !grid_fits(o.T, H)) return FMOE_ERR_SHAPE;
  const size_t e = elem(dtype);
  if (o.T == 0) {
    // no tokens: no row has a pick
    const size_t bytes = static_cast<size_t>(o.R) * H * e;
    if (!grad_rows || bytes == 0) return FMOE_OK;
    if (!at(grad_rows, e)) return FMOE_ERR_ALIGN;
    return done(cudaMemsetAsync(grad_rows, 0, bytes, as_stream(stream)));
  }
  if (!grad_rows && !grad_weights) return FMOE_OK;
  if (!grad_y || (grad_weights && !rows)) return FMOE_ERR_NULL;
  if (!at(grad_y, e) || !at(rows, e) || !at(grad_rows, e) || !at(weights, 4) ||
      !at(grad_weights, 4))
    return FMOE_ERR_ALIGN;
  const uint64_t picks = static_cast<uint64_t>(o.T) * o.K;
  if (overlap({{grad_rows, static_cast<uint64_t>(o.R) * H * e}, {grad_weights, picks * 4}},
              {{grad_y, static_cast<uint64_t>(o.T) * H * e},
               {rows, static_cast<uint64_t>(o.R) * H * e},
               {weights, picks * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_unsort_back(grad_y, rows, weights, grad_rows, grad_weights, dtype, o, H, sms,
                                 as_stream(stream)));
}

int fmoe_quantize_int8(const void* x, int32_t dtype, int64_t R, int64_t K, void* q, float* scale,
                       void* stream) {
  if (R < 0 || R > INT32_MAX - 1024 || K < 1 || K > INT32_MAX - 65536) return FMOE_ERR_SHAPE;
  if (dtype != FMOE_DTYPE_BF16 && dtype != FMOE_DTYPE_F16) return FMOE_ERR_DTYPE;
  if (R == 0) return FMOE_OK;
  if (!x || !q || !scale) return FMOE_ERR_NULL;
  if (!at(x, 2) || !at(scale, 4)) return FMOE_ERR_ALIGN;
  const uint64_t n = static_cast<uint64_t>(R) * K;
  if (overlap({{q, n}, {scale, static_cast<uint64_t>(R) * 4}}, {{x, 2 * n}})) return FMOE_ERR_SHAPE;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_quantize_int8(x, dtype, R, K, q, scale, sms, as_stream(stream)));
}

int fmoe_int8_matmul(const void* a, const void* b, const float* a_scale, const float* b_scale,
                     const float* bias, int64_t m, int32_t n, int32_t k, void* out,
                     int32_t out_dtype, void* stream) {
  return int8_product(
      Int8Product{a, b, a_scale, b_scale, bias, nullptr, out, m, n, k, 1, out_dtype, 0, 0, 0, 0},
      stream);
}

int fmoe_int8_expert_matmul(const void* rows, const void* weights, const float* row_scale,
                            const float* weight_scale, const int32_t* expert_base, int64_t R,
                            int32_t E, int32_t n, int32_t k, void* out, int32_t out_dtype,
                            int32_t zero_tail, void* stream) {
  if (R > 0 && !expert_base) return FMOE_ERR_NULL;
  return int8_product(Int8Product{rows, weights, row_scale, weight_scale, nullptr, expert_base, out,
                                  R, n, k, E, out_dtype, zero_tail, 0, 0, 0},
                      stream);
}

int fmoe_debug_arm_int8_timeout(uint64_t wait_ns) {
  if (wait_ns < 100000ull || wait_ns > 2000000000ull) return FMOE_ERR_SHAPE;
  g_int8_wait_ns = wait_ns;
  return FMOE_OK;
}

int fmoe_debug_arm_int8_plan(int32_t tile_tokens, int32_t split) {
  if ((tile_tokens != 16 && tile_tokens != 64 && tile_tokens != 128 && tile_tokens != 256) ||
      split < 1 || split > 4)
    return FMOE_ERR_SHAPE;
  g_int8_tile_tokens = tile_tokens;
  g_int8_split = split;
  return FMOE_OK;
}

int fmoe_int8_status(int32_t* status, void* stream) {
  if (!status) return FMOE_ERR_NULL;
  return done(take_int8_status(status, as_stream(stream)));
}

int fmoe_block_norm_workspace_size(int64_t T, int32_t H, size_t* bytes) {
  if (!bytes) return FMOE_ERR_NULL;
  if (T < 0 || T > INT32_MAX - 1024 || H < 1 || H > 16384) return FMOE_ERR_SHAPE;
  *bytes = norm_workspace(T, H);
  return FMOE_OK;
}

int fmoe_block_norm(const FmoeBlockNormArgs* a, void* stream) {
  BlockNorm p;
  int rc = check_norm(a, &p);
  if (rc) return rc;
  if (a->normed && a->normed_q) return FMOE_ERR_SHAPE;
  if (a->normed_q && a->hidden_size % kBlock != 0) return FMOE_ERR_SHAPE;
  if (p.T == 0) return FMOE_OK;
  if ((a->pre_weight != nullptr) != (a->normed != nullptr || a->normed_q != nullptr) ||
      (a->normed_q != nullptr) != (a->normed_scale != nullptr))
    return FMOE_ERR_NULL;
  const size_t e = elem(a->dtype);
  if (!at(a->hidden, e) || !at(a->normed, e) || !at(a->normed_scale, 4)) return FMOE_ERR_ALIGN;
  if (a->normed_q) {
    for (const void* q : {a->branch, a->residual, a->post_weight, a->gate, a->pre_weight,
                          static_cast<const void*>(a->hidden),
                          static_cast<const void*>(a->normed_q)})
      if (!at(q, 16)) return FMOE_ERR_ALIGN;
  }
  const uint64_t n = static_cast<uint64_t>(p.T) * p.H, row = n * e;
  const Span params[] = {{a->post_weight, a->post_weight ? p.H * elem(a->post_weight_dtype) : 0},
                         {a->gate, a->gate ? gate_count(a) * elem(a->gate_dtype) : 0},
                         {a->pre_weight, a->pre_weight ? p.H * elem(a->pre_weight_dtype) : 0}};
  // hidden may be the residual itself: every element is read by the thread that writes it
  const Span residual{a->hidden == a->residual ? nullptr : a->residual, row};
  if (overlap({{a->hidden, row}, {a->normed, row}, {a->normed_q, n},
               {a->normed_scale, n / kBlock * 4}, {a->stats, static_cast<uint64_t>(p.T) * 8}},
              {{a->branch, row}, residual, params[0], params[1], params[2]}))
    return FMOE_ERR_SHAPE;
  if (!a->hidden && !a->pre_weight && !a->stats) return FMOE_OK;
  p.h = a->hidden;
  p.y = a->normed;
  p.q = a->normed_q;
  p.q_scale = a->normed_scale;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_block_norm(p, sms, as_stream(stream)));
}

int fmoe_block_norm_backward(const FmoeBlockNormArgs* a, void* stream) {
  BlockNorm p;
  int rc = check_norm(a, &p);
  if (rc) return rc;
  const size_t e = elem(a->dtype);
  if ((a->grad_branch && !a->branch) || (a->grad_post_weight && !a->post_weight) ||
      (a->grad_gate && a->gate_kind == FMOE_GATE_NONE) || (a->grad_pre_weight && !a->pre_weight))
    if (p.T > 0) return FMOE_ERR_NULL;
  const bool sums = a->grad_post_weight || a->grad_pre_weight ||
                    (a->grad_gate && a->gate_kind == FMOE_GATE_CHANNEL);
  if (!at(a->grad_hidden, e) || !at(a->grad_normed, e) || !at(a->grad_branch, e) ||
      !at(a->grad_residual, e) || !at(a->workspace, 4) ||
      (a->grad_post_weight && !at(a->grad_post_weight, elem(a->post_weight_dtype))) ||
      (a->grad_gate && !at(a->grad_gate, elem(a->gate_dtype))) ||
      (a->grad_pre_weight && !at(a->grad_pre_weight, elem(a->pre_weight_dtype))))
    return FMOE_ERR_ALIGN;
  cudaStream_t s = as_stream(stream);
  if (p.T == 0) {
    // no tokens: the sums over tokens are zero
    const Span z[] = {{a->grad_post_weight, p.H * elem(a->post_weight_dtype)},
                      {a->gate_kind == FMOE_GATE_CHANNEL ? a->grad_gate : nullptr,
                       p.H * elem(a->gate_dtype)},
                      {a->grad_pre_weight, p.H * elem(a->pre_weight_dtype)}};
    for (const Span& w : z)
      if (w.p && cudaMemsetAsync(const_cast<void*>(w.p), 0, w.bytes, s) != cudaSuccess)
        return FMOE_ERR_CUDA;
    return FMOE_OK;
  }
  if (!a->stats || (a->grad_normed && !a->pre_weight)) return FMOE_ERR_NULL;
  const size_t need = norm_workspace(p.T, p.H);
  if (sums && (!a->workspace || a->workspace_bytes < need)) return FMOE_ERR_WORKSPACE;
  const uint64_t row = static_cast<uint64_t>(p.T) * p.H * e;
  const Span params[] = {{a->post_weight, a->post_weight ? p.H * elem(a->post_weight_dtype) : 0},
                         {a->gate, a->gate ? gate_count(a) * elem(a->gate_dtype) : 0},
                         {a->pre_weight, a->pre_weight ? p.H * elem(a->pre_weight_dtype) : 0}};
  if (overlap({{a->grad_branch, row},
               {a->grad_residual, row},
               {a->grad_post_weight, params[0].bytes},
               {a->grad_gate, params[1].bytes},
               {a->grad_pre_weight, params[2].bytes},
               {a->workspace, sums ? need : 0}},
              {{a->branch, row}, {a->residual, row}, params[0], params[1], params[2],
               {a->grad_hidden, row}, {a->grad_normed, row},
               {a->stats, static_cast<uint64_t>(p.T) * 8}}))
    return FMOE_ERR_SHAPE;
  p.back = true;
  p.da = a->grad_hidden;
  p.dy = a->grad_normed;
  p.df = a->grad_branch;
  p.dx = a->grad_residual;
  p.dwp = a->grad_post_weight;
  p.dg = a->grad_gate;
  p.dwq = a->grad_pre_weight;
  p.part = static_cast<float*>(a->workspace);
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_block_norm(p, sms, s));
}

int fmoe_quantize_int4(const void* w, int32_t dtype, int64_t rows, int32_t k, int32_t group,
                       void* packed, void* scale, void* zero, void* stream) {
  if (!int4_group(k, group)) return FMOE_ERR_SHAPE;
  const Int4Weights p{const_cast<void*>(w), dtype, rows, k, group, (k + group - 1) / group,
                      zero == nullptr, static_cast<uint8_t*>(packed), scale, dtype,
                      static_cast<uint8_t*>(zero)};
  int rc = check_int4_weights(p);
  if (rc || p.rows == 0) return rc;
  const uint64_t n = static_cast<uint64_t>(p.rows) * p.K, g = static_cast<uint64_t>(p.rows) * p.groups;
  if (overlap({{p.packed, n / 2}, {p.scale, g * elem(dtype)}, {p.zero, g}}, {{w, n * elem(dtype)}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_quantize_int4(p, sms, as_stream(stream)));
}

int fmoe_dequantize_int4(const void* packed, const void* scale, int32_t scale_dtype,
                         const void* zero, int64_t rows, int32_t k, int32_t group, void* w,
                         int32_t dtype, void* stream) {
  if (!int4_group(k, group)) return FMOE_ERR_SHAPE;
  const Int4Weights p{w, dtype, rows, k, group, (k + group - 1) / group, zero == nullptr,
                      static_cast<uint8_t*>(const_cast<void*>(packed)), const_cast<void*>(scale),
                      scale_dtype, static_cast<uint8_t*>(const_cast<void*>(zero))};
  int rc = check_int4_weights(p);
  if (rc || p.rows == 0) return rc;
  const uint64_t n = static_cast<uint64_t>(p.rows) * p.K, g = static_cast<uint64_t>(p.rows) * p.groups;
  if (overlap({{w, n * elem(dtype)}}, {{packed, n / 2}, {scale, g * elem(scale_dtype)}, {zero, g}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_dequantize_int4(p, sms, as_stream(stream)));
}

int fmoe_int4_workspace_size(int64_t m, int32_t n, int32_t k, int32_t E, size_t* bytes) {
  if (!bytes) return FMOE_ERR_NULL;
  if (m < 0 || m > INT32_MAX - 1024 || n < 1 || k < 32 || k % 32 != 0 || k > 131072 || E < 1 ||
      E > kMaxLocalExperts)
    return FMOE_ERR_SHAPE;
  // whether the rows have bases is not known here: the larger of the two plans
  size_t most = 0;
  for (const bool grouped : {false, true}) {
    if (!grouped && E > 1) continue;
    const Int4Plan p = int4_plan(m, n, k, E, grouped);
    const size_t need = p.S > 1 ? static_cast<size_t>(p.S) * m * n * 4 : 0;
    if (need > most) most = need;
  }
  *bytes = most;
  return FMOE_OK;
}

int fmoe_int4_matmul(const FmoeInt4Args* a, void* stream) {
  const unsigned long long wait_ns = g_int4_wait_ns;
  const int tile_tokens = g_int4_tile_tokens, split = g_int4_split;
  g_int4_wait_ns = 0;
  g_int4_tile_tokens = g_int4_split = 0;
  if (!a) return FMOE_ERR_NULL;
  if (a->num_rows < 0 || a->num_rows > INT32_MAX - 1024 || a->n < 1 || !int4_group(a->k, a->group) ||
      a->num_experts < 1 || a->num_experts > kMaxLocalExperts ||
      static_cast<int64_t>(a->num_experts) * a->n > INT32_MAX - 1024)
    return FMOE_ERR_SHAPE;
  if (!a->expert_base && a->num_experts != 1) return FMOE_ERR_NULL;
  if (a->expert_base && a->bias) return FMOE_ERR_SHAPE;
  if ((a->dtype != FMOE_DTYPE_BF16 && a->dtype != FMOE_DTYPE_F16) ||
      (a->scale_dtype != a->dtype && a->scale_dtype != FMOE_DTYPE_F32))
    return FMOE_ERR_DTYPE;
  if (a->num_rows == 0) return FMOE_OK;
  for (const void* q : {a->x, a->weight, a->scale, static_cast<const void*>(a->out)})
    if (!q) return FMOE_ERR_NULL;
  if (!at(a->x, 16) || !at(a->weight, 16) || !at(a->scale, elem(a->scale_dtype)) || !at(a->bias, 4) ||
      !at(a->expert_base, 4) || !at(a->out, 2) || !at(a->workspace, 16))
    return FMOE_ERR_ALIGN;
  // the tiles of every spread of the rows are counted in 32 bits
  if ((a->num_rows / 64 + a->num_experts) * ((a->n + 127ll) / 128) * 8 > INT32_MAX) return FMOE_ERR_SHAPE;
  size_t need = 0;
  int rc = fmoe_int4_workspace_size(a->num_rows, a->n, a->k, a->num_experts, &need);
  if (rc) return rc;
  if (tile_tokens != 0) {
    if ((a->k + 63) / 64 < split) return FMOE_ERR_SHAPE;
    need = split > 1 ? static_cast<size_t>(split) * a->num_rows * a->n * 4 : 0;
  }
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return FMOE_ERR_WORKSPACE;
  const uint64_t M = a->num_rows, EN = static_cast<uint64_t>(a->num_experts) * a->n;
  const uint64_t g = EN * ((a->k + a->group - 1) / a->group);
  if (overlap({{a->out, M * a->n * 2}, {a->workspace, need}},
              {{a->x, M * a->k * 2},
               {a->weight, EN * a->k / 2},
               {a->scale, g * elem(a->scale_dtype)},
               {a->zero, g},
               {a->bias, static_cast<uint64_t>(a->n) * 4},
               {a->expert_base, static_cast<uint64_t>(a->num_experts + 1) * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  const Int4Product p{a->x, a->dtype, static_cast<const uint8_t*>(a->weight), a->scale, a->scale_dtype,
                      static_cast<const uint8_t*>(a->zero), a->bias, a->expert_base, a->out,
                      a->num_rows, a->n, a->k, a->num_experts, a->group, a->zero_tail,
                      static_cast<float*>(a->workspace), wait_ns, tile_tokens, split};
  return done(launch_int4_product(p, sms, as_stream(stream)));
}

int fmoe_int4_status(int32_t* status, void* stream) {
  if (!status) return FMOE_ERR_NULL;
  return done(take_int4_status(status, as_stream(stream)));
}

int fmoe_debug_arm_int4_timeout(uint64_t wait_ns) {
  if (wait_ns < 100000ull || wait_ns > 2000000000ull) return FMOE_ERR_SHAPE;
  g_int4_wait_ns = wait_ns;
  return FMOE_OK;
}

int fmoe_debug_arm_int4_plan(int32_t tile_tokens, int32_t split) {
  if ((tile_tokens != 64 && tile_tokens != 128 && tile_tokens != 256) || split < 1 || split > 8)
    return FMOE_ERR_SHAPE;
  g_int4_tile_tokens = tile_tokens;
  g_int4_split = split;
  return FMOE_OK;
}

int fmoe_layer_norm_workspace_size(int64_t T, int32_t H, size_t* bytes) {
  if (!bytes) return FMOE_ERR_NULL;
  if (T < 0 || T > INT32_MAX - 1024 || H < 1 || H > 16384) return FMOE_ERR_SHAPE;
  *bytes = layer_norm_workspace(T, H);
  return FMOE_OK;
}

int fmoe_layer_norm(const FmoeLayerNormArgs* a, void* stream) {
  LayerNorm p;
  int rc = check_layer_norm(a, &p);
  if (rc) return rc;
  if ((a->normed && a->normed_q) || (a->normed_q && a->hidden_size % kBlock != 0))
    return FMOE_ERR_SHAPE;
  if (p.T == 0) return FMOE_OK;
  if ((a->normed_q != nullptr) != (a->normed_scale != nullptr)) return FMOE_ERR_NULL;
  const size_t e = elem(a->dtype);
  if (!at(a->hidden, e) || !at(a->normed, e) || !at(a->normed_scale, 4)) return FMOE_ERR_ALIGN;
  if (a->normed_q) {
    for (const void* q : {a->branch, a->residual, a->weight, a->bias,
                          static_cast<const void*>(a->hidden), static_cast<const void*>(a->normed_q)})
      if (!at(q, 16)) return FMOE_ERR_ALIGN;
  }
  const uint64_t n = static_cast<uint64_t>(p.T) * p.H, row = n * e;
  // hidden may be the residual itself: an element is used by the thread alone that writes it, after it was read.
  // (Rows off the 16-byte boundaries share 16 bytes with their neighbours: a thread may read a neighbour's elements
  // while that row's block rewrites them, and puts zeros in their place before their first use.)
  const Span residual{a->hidden == a->residual ? nullptr : a->residual, row};
  if (overlap({{a->hidden, row}, {a->normed, row}, {a->normed_q, n}, {a->normed_scale, n / kBlock * 4},
               {a->stats, static_cast<uint64_t>(p.T) * 8}},
              {{a->branch, row}, residual,
               {a->weight, a->weight ? p.H * elem(a->weight_dtype) : 0},
               {a->bias, a->bias ? p.H * elem(a->bias_dtype) : 0}}))
    return FMOE_ERR_SHAPE;
  if (!a->hidden && !a->normed && !a->normed_q && !a->stats) return FMOE_OK;
  p.h = a->hidden;
  p.y = a->normed;
  p.q = a->normed_q;
  p.q_scale = a->normed_scale;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_layer_norm(p, sms, as_stream(stream)));
}

int fmoe_layer_norm_backward(const FmoeLayerNormArgs* a, void* stream) {
  LayerNorm p;
  int rc = check_layer_norm(a, &p);
  if (rc) return rc;
  const size_t e = elem(a->dtype);
  const size_t we = elem(a->weight_dtype), be = elem(a->bias_dtype);
  const bool sums = a->grad_weight || a->grad_bias;
  if ((a->grad_weight && !a->weight) || (a->grad_bias && !a->bias)) return FMOE_ERR_NULL;
  // the shares of the sums go through the workspace in pairs and fours
  if (!at(a->grad_hidden, e) || !at(a->grad_normed, e) || !at(a->grad_input, e) ||
      !at(a->workspace, sums ? 16 : 4) || (a->grad_weight && !at(a->grad_weight, we)) ||
      (a->grad_bias && !at(a->grad_bias, be)))
    return FMOE_ERR_ALIGN;
  cudaStream_t s = as_stream(stream);
  if (p.T == 0) {  // no tokens: the sums over tokens are zero
    if ((a->grad_weight && cudaMemsetAsync(a->grad_weight, 0, p.H * we, s) != cudaSuccess) ||
        (a->grad_bias && cudaMemsetAsync(a->grad_bias, 0, p.H * be, s) != cudaSuccess))
      return FMOE_ERR_CUDA;
    return FMOE_OK;
  }
  if (!a->grad_input && !sums) return FMOE_OK;
  if (!a->stats) return FMOE_ERR_NULL;
  const size_t need = layer_norm_workspace(p.T, p.H);
  if (sums && (!a->workspace || a->workspace_bytes < need)) return FMOE_ERR_WORKSPACE;
  const uint64_t row = static_cast<uint64_t>(p.T) * p.H * e;
  if (overlap({{a->grad_input, row},
               {a->grad_weight, p.H * we},
               {a->grad_bias, p.H * be},
               {a->workspace, sums ? need : 0}},
              {{a->branch, row}, {a->residual, row}, {a->weight, a->weight ? p.H * we : 0},
               {a->grad_hidden, row}, {a->grad_normed, row},
               {a->stats, static_cast<uint64_t>(p.T) * 8}}))
    return FMOE_ERR_SHAPE;
  p.back = true;
  p.dh = a->grad_hidden;
  p.dy = a->grad_normed;
  p.dx = a->grad_input;
  p.dw = a->grad_weight;
  p.db = a->grad_bias;
  p.part = static_cast<float*>(a->workspace);
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_layer_norm(p, sms, s));
}

int fmoe_balance_workspace_size(int64_t T, int32_t E, int32_t S, size_t* bytes) {
  if (!bytes) return FMOE_ERR_NULL;
  if (T < 0 || T > INT32_MAX - 1024 || E < 1 || E > kMaxBalanceExperts || S < 1 ||
      S > kMaxBalanceSequences)
    return FMOE_ERR_SHAPE;
  *bytes = balance_workspace(T, E, S);
  return FMOE_OK;
}

int fmoe_balance_loss(const FmoeBalanceArgs* a, void* stream) {
  Balance p;
  int rc = check_balance(a, &p);
  if (rc) return rc;
  if (static_cast<int64_t>(p.T) * p.K > INT32_MAX) return FMOE_ERR_SHAPE;  // the counts are int32
  if (!p.counts || (p.loss && !p.factor) || (p.T > 0 && (!p.ids || (p.loss && !p.logits))))
    return FMOE_ERR_NULL;
  const size_t need = balance_workspace(p.T, p.E, p.S);
  if (!p.workspace || a->workspace_bytes < need) return FMOE_ERR_WORKSPACE;
  const uint64_t T = p.T, S = p.S;
  if (overlap({{p.loss, 4}, {p.counts, S * p.E * 4}, {p.factor, S * 4}, {p.workspace, need}},
              {{p.logits, T * p.E * elem(p.dtype)}, {p.ids, T * p.K * 4}, {p.base, (S + 1) * 4}}))
    return FMOE_ERR_SHAPE;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_balance(p, sms, as_stream(stream)));
}

int fmoe_balance_loss_backward(const FmoeBalanceArgs* a, void* stream) {
  Balance p;
  int rc = check_balance(a, &p);
  if (rc) return rc;
  if (p.T == 0) return FMOE_OK;
  if (!p.logits || !p.counts || !p.factor || !p.grad_loss || !p.grad_logits) return FMOE_ERR_NULL;
  const uint64_t S = p.S, rows = static_cast<uint64_t>(p.T) * p.E * elem(p.dtype);
  if (overlap({{p.grad_logits, rows}}, {{p.logits, rows}, {p.base, (S + 1) * 4},
                                        {p.counts, S * p.E * 4}, {p.factor, S * 4}, {p.grad_loss, 4}}))
    return FMOE_ERR_SHAPE;
  p.back = true;
  int sms = 0;
  rc = device_sms(&sms);
  if (rc) return rc;
  return done(launch_balance(p, sms, as_stream(stream)));
}

}  // extern "C"
