// Host side of the cache operators in include/busfill.h (rope_axes, kv4_*,
// attn_kv4): argument checks, the choice of the kernel and its launch shape.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "busfill.h"
#include "kv4_attn.cuh"
#include "kv4_cache.cuh"
#include "kv4_prompt.cuh"
#include "kv4_weights.cuh"

using namespace busfill;
using namespace busfill::kv4;

namespace {

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool is16bit(int dtype) { return dtype == BUSFILL_TYPE_F16 || dtype == BUSFILL_TYPE_BF16; }

int check_cache(const busfill_kv4* c) {
  if (!c || !c->pages || !c->table || !c->kv_len) return BUSFILL_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return BUSFILL_ERR_SHAPE;
  if (c->batch < 1 || c->batch > BUSFILL_KV4_MAX_BATCH || c->heads < 1 || c->heads > 65535 || c->num_pages < 1 ||
      c->table_cols < 1 || c->table_cols > (1 << 24))
    return BUSFILL_ERR_SHAPE;
  if (!aligned(c->pages, 16) || !aligned(c->table, 4) || !aligned(c->kv_len, 4)) return BUSFILL_ERR_ALIGNMENT;
  return BUSFILL_OK;
}

View view_of(const busfill_kv4* c) {
  return View{c->pages, c->table, c->kv_len, c->num_pages, c->table_cols, c->batch, c->heads};
}

// f(std::integral_constant<int, D>) for the cache's head dimension
template <typename Fn>
int by_dim(int d, Fn f) {
  if (d == 64) return f(std::integral_constant<int, 64>());
  if (d == 128) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 256>());
}

// Raise a kernel's dynamic shared memory limit, once per device.
template <typename Kernel>
bool raise_smem(Kernel kernel, int bytes, int dev, std::once_flag (&once)[64], cudaError_t (&err)[64]) {
  std::call_once(once[dev & 63], [&] {
    err[dev & 63] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
  return err[dev & 63] == cudaSuccess;
}

// The tcgen05 kernel takes a call whose widest sequence has this many query
// rows per key/value head, if the call has kPromptTotal rows in all. Us of
// attn_kernel / prompt_kernel, 8 sequences of 4096 tokens and 8 heads of 128:
// 32 rows 49 / 57, 40 rows 58 / 57, 96 rows 105 / 57; heads of 64: 48 rows
// 41 / 47, 64 rows 47 / 47, 96 rows 59 / 47; 4 heads of 256: 32 rows 64 / 67,
// 40 rows 72 / 68. One sequence, 8 heads of 128: 48 rows (384 in all) 25 / 39
// at 4096 tokens; 64 (512) 70 / 76 at 32000; 128 (1024) 33 / 40 and 121 / 76.
constexpr int prompt_rows(int head_dim) { return head_dim == 64 ? 57 : 37; }
constexpr long long kPromptTotal = 640;

// Query rows from which the weights' second pass goes to tcgen05. Us of
// weights_kernel / weights_prompt_kernel, 8 sequences of 4096 tokens, 8 heads
// of 128: 24 rows 27 / 35, 32 rows 35 / 36, 40 rows 42 / 37, 96 rows 88 / 38;
// heads of 64: 32 rows 24 / 33, 48 rows 31 / 32, 64 rows 43 / 34; one sequence
// of 512: 16 rows 13 / 15, 32 rows 16 / 15, 64 rows 26 / 15.
constexpr int kWeightsRows = 33;

constexpr long long kMaxGrid = 2147483647;

// Query rows of the widest sequence and head from which two row tiles share a
// warp's pass over the pages, heads of 64 only. Us with one / two, 32 sequences
// of 1024 tokens, 8 heads of 64: 8 rows 25 / 29, 24 rows 32 / 35, 32 rows
// 38 / 35, 48 rows 46 / 43. Wider heads have no registers for it (8 sequences
// of 4096, heads of 128: 32 rows 49 / 68).
constexpr int kTwoTileRows = 25;

// The kernels of a call: busfill_attn_kv4_kernel_for.
enum { kFewRows = 0, kFewRowsTwoTiles = 1, kManyRows = 2, kWeightsManyRows = 4 };
int choose(long long all_rows, int rows, int head_dim) {
  const int weights = rows >= kWeightsRows ? kWeightsManyRows : 0;
  if (rows >= prompt_rows(head_dim) && all_rows >= kPromptTotal) return kManyRows | weights;
  return (head_dim == 64 && rows >= kTwoTileRows ? kFewRowsTwoTiles : kFewRows) | weights;
}

// Workspace of the attention calls on a stream: a counter per CTA, a word
// between a call's two kernels, then the largest kernel's partial results.
constexpr size_t kCounterBytes = 4096;
constexpr int kMaxCtas = kCounterBytes / 4 - 1;
// What calls that do not take prompt_kernel need of it (2.4 MB), and all calls (39 MB).
size_t few_rows_bytes(int sms) {
  size_t f = part_floats<64, 2>();
  f = std::max(f, part_floats<128, 1>());
  f = std::max(f, part_floats<256, 1>());
  f = std::max(f, (size_t)2 * wsum::Geo<128>::kTokens);
  return kCounterBytes + (size_t)sms * f * sizeof(float);
}
size_t workspace_bytes(int sms) {
  size_t f = (size_t)2 * prompt::Geo<64>::kPartFloats;
  f = std::max(f, (size_t)2 * prompt::Geo<128>::kPartFloats);
  f = std::max(f, (size_t)2 * prompt::Geo<256>::kPartFloats);
  return std::max(few_rows_bytes(sms), kCounterBytes + (size_t)sms * f * sizeof(float));
}

template <int D, int NT>
int launch_attn(const AttnParams& p, const host::Context& ctx, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t err[64];
  using G = Geo<D, NT>;
  if (!raise_smem(attn_kernel<D, NT>, G::kBytes, ctx.dev, once, err)) return BUSFILL_ERR_LAUNCH;
  void* args[] = {const_cast<AttnParams*>(&p)};
  return host::launch(reinterpret_cast<const void*>(attn_kernel<D, NT>), dim3(ctx.sms), dim3(G::kWarps * 32),
                      G::kBytes, s, args);
}

template <int D>
int launch_prompt(const AttnParams& p, const host::Context& ctx, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t err[64];
  constexpr int bytes = prompt::Geo<D>::kAlloc;
  if (!raise_smem(prompt_kernel<D>, bytes, ctx.dev, once, err)) return BUSFILL_ERR_LAUNCH;
  void* args[] = {const_cast<AttnParams*>(&p)};
  return host::launch(reinterpret_cast<const void*>(prompt_kernel<D>), dim3(ctx.sms), dim3(prompt::kThreads), bytes, s,
                      args);
}

template <int D>
int launch_weights(const AttnParams& p, const host::Context& ctx, cudaStream_t s, bool many) {
  void* args[] = {const_cast<AttnParams*>(&p)};
  static std::once_flag once[64], few_once[64];
  static cudaError_t err[64], few_err[64];
  if (!many) {
    using G = WeightsGeo<D>;
    if (!raise_smem(weights_kernel<D>, G::kBytes, ctx.dev, few_once, few_err)) return BUSFILL_ERR_LAUNCH;
    return host::launch((const void*)weights_kernel<D>, dim3(ctx.sms), dim3(G::kWarps * 32), G::kBytes, s, args);
  }
  constexpr int bytes = wsum::Geo<D>::kAlloc;
  if (!raise_smem(weights_prompt_kernel<D>, bytes, ctx.dev, once, err)) return BUSFILL_ERR_LAUNCH;
  return host::launch((const void*)weights_prompt_kernel<D>, dim3(ctx.sms), dim3(wsum::kThreads), bytes, s, args);
}

}  // namespace

extern "C" {

int busfill_kv4_page_bytes(int head_dim) {
  return head_dim == 64 || head_dim == 128 || head_dim == 256 ? 72 * head_dim : BUSFILL_ERR_SHAPE;
}

int busfill_rope_axes(const busfill_rope* r, void* stream) {
  if (!r || !r->cos || !r->sin || !r->axis) return BUSFILL_ERR_INVALID_ARG;
  // a step of no tokens has nothing to point at
  if (r->tokens != 0 && (!r->q || !r->q_out || !r->positions || (r->k_heads > 0 && (!r->k || !r->k_out))))
    return BUSFILL_ERR_INVALID_ARG;
  if (!is16bit(r->dtype)) return BUSFILL_ERR_INVALID_ARG;
  if (r->tokens < 0 || r->q_heads < 1 || r->k_heads < 0 || r->q_heads > 65535 || r->k_heads > 65535 ||
      r->head_dim < 2 || r->head_dim > 512 || r->rot < 2 || (r->rot & 1) || r->rot > r->head_dim || r->axes < 1 ||
      r->axes > 4 || r->max_pos < 1)
    return BUSFILL_ERR_SHAPE;
  const int half = r->rot / 2;
  static_assert(kMaxFreqs == 256, "rot <= 512");
  RopeParams p{};
  for (int i = 0; i < half; ++i) {
    if (r->axis[i] >= r->axes) return BUSFILL_ERR_INVALID_ARG;
    p.axis[i] = r->axis[i];
  }
  const void* ptrs[] = {r->q, r->q_out, r->k_heads ? r->k : r->q, r->k_heads ? r->k_out : r->q_out};
  const int64_t strides[] = {r->q_token, r->q_head, r->q_out_token, r->q_out_head,
                             r->k_heads ? r->k_token : 0, r->k_heads ? r->k_head : 0,
                             r->k_heads ? r->k_out_token : 0, r->k_heads ? r->k_out_head : 0};
  // 16-byte pieces where every row starts on 16 bytes and the pieces come out even
  bool vec = r->adjacent ? r->rot % 8 == 0 : half % 8 == 0;
  vec = vec && (r->head_dim - r->rot) % 8 == 0;
  for (const void* q : ptrs) {
    if (!aligned(q, 2)) return BUSFILL_ERR_ALIGNMENT;
    vec = vec && aligned(q, 16);
  }
  if (!aligned(r->positions, 4) || !aligned(r->cos, 4) || !aligned(r->sin, 4)) return BUSFILL_ERR_ALIGNMENT;
  for (int64_t st : strides) vec = vec && st % 8 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  host::Context ctx;
  const int st = host::context(s, &ctx);
  if (st != BUSFILL_OK || r->tokens == 0) return st;
  p.q = r->q, p.k = r->k, p.q_out = r->q_out, p.k_out = r->k_out;
  p.positions = r->positions, p.cos = r->cos, p.sin = r->sin;
  p.q_token = r->q_token, p.q_head = r->q_head, p.k_token = r->k_token, p.k_head = r->k_head;
  p.qo_token = r->q_out_token, p.qo_head = r->q_out_head, p.ko_token = r->k_out_token, p.ko_head = r->k_out_head;
  p.tokens = r->tokens, p.q_heads = r->q_heads, p.k_heads = r->k_heads, p.dim = r->head_dim, p.half = half;
  p.max_pos = r->max_pos;
  p.sign = r->inverse ? -1.0f : 1.0f;
  p.error = ctx.error;
  const int pairs = vec ? (r->adjacent ? 4 : 8) : 1;
  const int pieces = half / pairs + (r->head_dim - r->rot) / (vec ? 8 : 1);
  const int heads = r->q_heads + r->k_heads;
  // Heads of one thread: as many as leave an SM 256 threads. Us with 1 / 2 / 4 /
  // 8, 64 + 8 heads of 128, event times of about 8 us more than the kernel's:
  // 32 tokens 8 / 10 / 10 / 12, 256 tokens 14 / 10 / 12 / 14, 512 tokens
  // 21 / 16 / 12 / 14, 1024 tokens 33 / 25 / 18 / 16, 8192 tokens 217 / 145 /
  // 94 / 80.
  int per = 8;
  while (per > 1 && (long long)r->tokens * pieces * ((heads + per - 1) / per) < (long long)ctx.sms * 256) per /= 2;
  p.heads_per_thread = per;
  p.groups = (heads + per - 1) / per;
  const long long blocks = ((long long)r->tokens * pieces * p.groups + 255) / 256;
  if (blocks > kMaxGrid) return BUSFILL_ERR_SHAPE;
  const bool h = r->dtype == BUSFILL_TYPE_F16, adj = r->adjacent != 0;
  const void* kern;
#define ROPE_KERNEL(T) \
  (adj ? (vec ? (const void*)rope_kernel<T, true, true> : (const void*)rope_kernel<T, true, false>) \
       : (vec ? (const void*)rope_kernel<T, false, true> : (const void*)rope_kernel<T, false, false>))
  kern = h ? ROPE_KERNEL(__half) : ROPE_KERNEL(__nv_bfloat16);
#undef ROPE_KERNEL
  void* args[] = {&p};
  return host::launch(kern, dim3((unsigned)blocks), dim3(256), 0, s, args);
}

int busfill_kv4_append(const busfill_kv4* cache, const busfill_kv4_rows* r, void* stream) {
  int st = check_cache(cache);
  if (st != BUSFILL_OK) return st;
  if (!r || (r->tokens != 0 && (!r->k || !r->v)) || !is16bit(r->dtype)) return BUSFILL_ERR_INVALID_ARG;
  if (r->tokens < 0 || (!r->q_start && r->tokens != cache->batch)) return BUSFILL_ERR_SHAPE;
  if (!aligned(r->k, 2) || !aligned(r->v, 2) || !aligned(r->q_start, 4)) return BUSFILL_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  host::Context ctx;
  st = host::context(s, &ctx);
  if (st != BUSFILL_OK || r->tokens == 0) return st;
  AppendParams p{};
  p.c = view_of(cache);
  p.k = r->k, p.v = r->v, p.q_start = r->q_start;
  p.k_token = r->k_token, p.k_head = r->k_head, p.v_token = r->v_token, p.v_head = r->v_head;
  p.tokens = r->tokens;
  p.vec = aligned(r->k, 16) && aligned(r->v, 16) && (r->k_token | r->k_head | r->v_token | r->v_head) % 8 == 0;
  p.error = ctx.error;
  // Four groups a lane where one would make more than 128 warps an SM. Us with
  // one / four (event times, some 8 us more than the kernel's), 8 heads of 128:
  // 512 tokens 8 / 10, 2048 tokens 14 / 14, 4096 tokens 21 / 18, 8192 tokens
  // 33 / 29; 4 heads of 64: 4096 tokens 10 / 12.
  const int groups = (2 * cache->heads * (cache->head_dim / 8) + 31) / 32;
  const bool four = (long long)p.tokens * groups >= (long long)ctx.sms * 128;
  p.chunks = four ? (groups + 3) / 4 : groups;
  const long long blocks = ((long long)p.tokens * p.chunks + 7) / 8;
  if (blocks > kMaxGrid / 8) return BUSFILL_ERR_SHAPE;   // the kernel counts warps in an int
  void* args[] = {&p};
  return by_dim(cache->head_dim, [&](auto d) {
    const void* kern = r->dtype == BUSFILL_TYPE_F16
                           ? (four ? (const void*)append_kernel<d(), __half, 4> : (const void*)append_kernel<d(), __half, 1>)
                           : (four ? (const void*)append_kernel<d(), __nv_bfloat16, 4>
                                   : (const void*)append_kernel<d(), __nv_bfloat16, 1>);
    return host::launch(kern, dim3((unsigned)blocks), dim3(256), 0, s, args);
  });
}

int busfill_kv4_read(const busfill_kv4* cache, const int32_t* q_start, int tokens, uint16_t* k, uint16_t* v,
                     void* stream) {
  int st = check_cache(cache);
  if (st != BUSFILL_OK) return st;
  if (tokens != 0 && (!k || !v)) return BUSFILL_ERR_INVALID_ARG;
  if (tokens < 0 || (!q_start && tokens != cache->batch)) return BUSFILL_ERR_SHAPE;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(q_start, 4)) return BUSFILL_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  host::Context ctx;
  st = host::context(s, &ctx);
  if (st != BUSFILL_OK || tokens == 0) return st;
  ReadParams p{view_of(cache), q_start, tokens, (2 * cache->heads + 7) / 8,
               reinterpret_cast<__half*>(k), reinterpret_cast<__half*>(v), ctx.error};
  const long long blocks = ((long long)tokens * p.chunks + 7) / 8;
  if (blocks > kMaxGrid / 8) return BUSFILL_ERR_SHAPE;
  void* args[] = {&p};
  return by_dim(cache->head_dim, [&](auto d) {
    return host::launch((const void*)read_kernel<d()>, dim3((unsigned)blocks), dim3(256), 0, s, args);
  });
}

int busfill_attn_kv4(const busfill_kv4* cache, const busfill_attn* a, void* stream) {
  int st = check_cache(cache);
  if (st != BUSFILL_OK) return st;
  if (!a || (a->tokens != 0 && (!a->q || !a->out || (a->weights && !a->lse))) || !is16bit(a->dtype) || a->window < 0 ||
      (a->window > 0 && !a->causal) || !(a->scale == a->scale))
    return BUSFILL_ERR_INVALID_ARG;
  if (a->tokens < 0 || a->q_heads < 1 || a->q_heads % cache->heads != 0 || a->max_q < 1 ||
      (!a->q_start && a->tokens != cache->batch) ||
      (long long)a->max_q * (a->q_heads / cache->heads) > (1 << 30) ||
      (a->weights && a->weights_cols < (int64_t)64 * cache->table_cols))
    return BUSFILL_ERR_SHAPE;
  if (!aligned(a->q, 16) || !aligned(a->out, 16) || (a->q_token | a->q_head | a->out_token | a->out_head) % 8 != 0 ||
      !aligned(a->lse, 4) || !aligned(a->weights, 4) || !aligned(a->q_start, 4))
    return BUSFILL_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  host::Context ctx;
  st = host::context(s, &ctx);
  if (st != BUSFILL_OK || a->tokens == 0) return st;
  const int max_q = a->q_start ? a->max_q : 1, rows = max_q * (a->q_heads / cache->heads);
  const int kernels = choose((long long)a->tokens * a->q_heads, rows, cache->head_dim);
  void* work = nullptr;
  const size_t bytes = workspace_bytes(ctx.sms);
  st = host::workspace(ctx, s, bytes, kernels & kManyRows ? bytes : few_rows_bytes(ctx.sms), kCounterBytes, &work);
  if (st != BUSFILL_OK) return st;
  AttnParams p{};
  p.c = view_of(cache);
  p.q = a->q, p.out = a->out, p.lse = a->lse, p.weights = a->weights, p.q_start = a->q_start;
  p.q_token = a->q_token, p.q_head = a->q_head, p.o_token = a->out_token, p.o_head = a->out_head;
  p.weights_cols = a->weights_cols;
  p.scale_log2 = a->scale * kLog2e;
  p.tokens = a->tokens, p.q_heads = a->q_heads, p.group = a->q_heads / cache->heads;
  p.by_group = divide_by((unsigned)p.group);
  p.max_q = max_q;
  // a window as long as the table can hold is none (and stays clear of the end of int)
  p.causal = a->causal != 0, p.window = a->window < (int64_t)kPage * cache->table_cols ? a->window : 0, p.bf16 = a->dtype == BUSFILL_TYPE_BF16;
  p.wide_out = aligned(a->out, 32) && (a->out_token | a->out_head) % 16 == 0;
  p.counters = static_cast<unsigned*>(work);
  p.refused = p.counters + kMaxCtas;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + kCounterBytes);
  p.error = ctx.error;
  if (ctx.sms > kMaxCtas) return BUSFILL_ERR_UNSUPPORTED_DEVICE;
  st = by_dim(cache->head_dim, [&](auto d) {
    if (kernels & kManyRows) return launch_prompt<d()>(p, ctx, s);
    if constexpr (d() == 64) {
      if (kernels & kFewRowsTwoTiles) return launch_attn<d(), 2>(p, ctx, s);
    }
    return launch_attn<d(), 1>(p, ctx, s);
  });
  if (st != BUSFILL_OK || !a->weights) return st;
  const bool many = (kernels & kWeightsManyRows) != 0;
  return by_dim(cache->head_dim, [&](auto d) { return launch_weights<d()>(p, ctx, s, many); });
}

int busfill_attn_kv4_kernel_for(int tokens, int q_heads, int heads, int head_dim, int max_q) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || tokens < 0 || heads < 1 || heads > 65535 ||
      q_heads < 1 || q_heads % heads != 0 || max_q < 1 || (long long)max_q * (q_heads / heads) > (1 << 30))
    return BUSFILL_ERR_SHAPE;
  return choose((long long)tokens * q_heads, max_q * (q_heads / heads), head_dim);
}

int busfill_kv4_evict(const busfill_kv4* cache, const busfill_kv4_eviction* e, void* stream) {
  int st = check_cache(cache);
  if (st != BUSFILL_OK) return st;
  if (!e || !e->weights || !e->weights_out || !e->index || !e->kv_len_out || !e->out_table ||
      e->kv_len_out == cache->kv_len)
    return BUSFILL_ERR_INVALID_ARG;
  const bool in_place = e->out_table == cache->table;
  if (e->keep < 1 || e->recent < 0 || e->recent > e->keep || e->weights_cols < (int64_t)64 * cache->table_cols ||
      e->out_cols < 1 || e->out_cols > (1 << 24) || (int64_t)64 * e->out_cols < e->keep ||
      (in_place && e->out_cols != cache->table_cols))
    return BUSFILL_ERR_SHAPE;
  if (!aligned(e->weights, 4) || !aligned(e->weights_out, 4) || !aligned(e->index, 4) || !aligned(e->kv_len_out, 4) ||
      !aligned(e->out_table, 4))
    return BUSFILL_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  host::Context ctx;
  st = host::context(s, &ctx);
  if (st != BUSFILL_OK) return st;
  EvictParams p{view_of(cache), e->weights, e->weights_out, e->weights_cols, e->index, e->kv_len_out,
                e->out_table,   e->out_cols, e->keep,       e->recent,       in_place, ctx.error};
  const int rows = cache->batch * cache->heads;
  void* args[] = {&p};
  static std::once_flag once[64];
  static cudaError_t err[64];
  if (!raise_smem(evict_select_kernel, kSelectBytes, ctx.dev, once, err)) return BUSFILL_ERR_LAUNCH;
  st = host::launch((const void*)evict_select_kernel, dim3(rows), dim3(kSelectThreads), kSelectBytes, s, args);
  if (st != BUSFILL_OK) return st;
  return by_dim(cache->head_dim, [&](auto d) {
    int per = 1;
    void* margs[] = {&p, &per};
    if (in_place)
      return host::launch((const void*)evict_move_kernel<d(), true>, dim3((unsigned)rows),
                          dim3(MoveGeo<d(), true>::kThreads), 0, s, margs);
    // Eight CTAs an SM, as far as there are tokens (select and move of 64 rows
    // of 32000 weights, keep 8000: two an SM 102 us, four 80, eight 80, 32 80).
    using G = MoveGeo<d(), false>;
    per = std::max(1, std::min((e->keep + G::kTokens - 1) / G::kTokens, (ctx.sms * 8 + rows - 1) / rows));
    return host::launch((const void*)evict_move_kernel<d(), false>, dim3((unsigned)(rows * per)), dim3(G::kThreads), 0,
                        s, margs);
  });
}

}  // extern "C"
