// The memory-bound operators around the cache: rotary positions, quantizing
// new tokens into the cache, reading tokens back, and eviction.
#pragma once

#include "kv4_format.cuh"

namespace busfill {
namespace kv4 {

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
constexpr int kMaxFreqs = 256;

struct RopeParams {
  const void *q, *k;
  void *q_out, *k_out;
  const int* positions;
  const float *cos, *sin;
  long long q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head;
  int tokens, q_heads, k_heads, dim, half, max_pos;
  int heads_per_thread, groups;   // groups of heads_per_thread heads
  float sign;                     // -1: turn back
  unsigned* error;
  uint8_t axis[kMaxFreqs];
};

// One thread owns a piece of the channels of one token and turns it in
// heads_per_thread heads, so that the angles are read once for these.
// VEC: a piece is 8 channel pairs in two 16-byte vectors (HALVES), or 4 pairs
// in one; else one pair. Behind the rotated pieces come copied ones.
// Bound by memory: 8190 tokens of 72 heads of 128 59 us, 305 MB at 5.2 TB/s.
template <typename T, bool ADJ, bool VEC>
__global__ void rope_kernel(const __grid_constant__ RopeParams p) {
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  constexpr int kPairs = VEC ? (ADJ ? 4 : 8) : 1;
  constexpr int kCopy = VEC ? 8 : 1;
  const int turned = p.half / kPairs;
  const int pieces = turned + (p.dim - 2 * p.half) / kCopy;
  const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long rest = id / pieces;
  const int piece = (int)(id - rest * pieces);
  const int token = (int)(rest / p.groups), group = (int)(rest - (long long)token * p.groups);
  if (token >= p.tokens) return;
  float c[kPairs], s[kPairs];
  if (piece < turned) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int f = piece * kPairs + i;
      const int pos = p.positions[(size_t)p.axis[f] * p.tokens + token];
      if ((unsigned)pos < (unsigned)p.max_pos) {
        c[i] = __ldg(p.cos + (size_t)pos * p.half + f);
        s[i] = p.sign * __ldg(p.sin + (size_t)pos * p.half + f);
      } else {
        c[i] = s[i] = __int_as_float(0x7fc00000);
        atomicOr(p.error, kErrIndex);
      }
    }
  }
  const int h0 = group * p.heads_per_thread, h1 = min(h0 + p.heads_per_thread, p.q_heads + p.k_heads);
  auto source = [&](int h) {
    return h < p.q_heads ? static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head
                         : static_cast<const T*>(p.k) + token * p.k_token + (h - p.q_heads) * p.k_head;
  };
  auto target = [&](int h) {
    return h < p.q_heads ? static_cast<T*>(p.q_out) + token * p.qo_token + h * p.qo_head
                         : static_cast<T*>(p.k_out) + token * p.ko_token + (h - p.q_heads) * p.ko_head;
  };
  const int at = piece < turned ? piece * kPairs : 2 * p.half + (piece - turned) * kCopy;
  if constexpr (VEC) {
    // kBatch heads' loads in flight
    constexpr int kBatch = 4;
    for (int h = h0; h < h1; h += kBatch) {
      uint4 u[kBatch], v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (h + k >= h1) break;
        const T* x = source(h + k);
        u[k] = *reinterpret_cast<const uint4*>(x + (ADJ && piece < turned ? 2 * at : at));
        if (!ADJ && piece < turned) v[k] = *reinterpret_cast<const uint4*>(x + p.half + at);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (h + k >= h1) break;
        T* y = target(h + k);
        if (piece < turned) {
          T* a = reinterpret_cast<T*>(&u[k]);   // halves: x0 in a, x1 in b; adjacent: pairs in a
          T* b = reinterpret_cast<T*>(&v[k]);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            T& e0 = ADJ ? a[2 * i] : a[i];
            T& e1 = ADJ ? a[2 * i + 1] : b[i];
            const float x0 = to_float(e0), x1 = to_float(e1);
            from_float(e0, x0 * c[i] - x1 * s[i]);
            from_float(e1, x1 * c[i] + x0 * s[i]);
          }
          *reinterpret_cast<uint4*>(y + (ADJ ? 2 * at : at)) = u[k];
          if (!ADJ) *reinterpret_cast<uint4*>(y + p.half + at) = v[k];
        } else {
          *reinterpret_cast<uint4*>(y + at) = u[k];
        }
      }
    }
  } else {
    for (int h = h0; h < h1; ++h) {
      const T* x = source(h);
      T* y = target(h);
      if (piece < turned) {
        const int i0 = ADJ ? 2 * at : at, i1 = ADJ ? 2 * at + 1 : p.half + at;
        const float x0 = to_float(x[i0]), x1 = to_float(x[i1]);
        from_float(y[i0], x0 * c[0] - x1 * s[0]);
        from_float(y[i1], x1 * c[0] + x0 * s[0]);
      } else {
        y[at] = x[at];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendParams {
  View c;
  const void *k, *v;
  const int* q_start;
  long long k_token, k_head, v_token, v_head;
  int tokens;
  int chunks;      // warps of a token
  int vec;         // 16-byte loads
  unsigned* error;
};

__device__ __forceinline__ __half2 pair_of(__half, uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ __nv_bfloat162 pair_of(__nv_bfloat16, uint32_t u) {
  return *reinterpret_cast<__nv_bfloat162*>(&u);
}
__device__ __forceinline__ float2 to_floats(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 to_floats(__nv_bfloat162 x) { return __bfloat1622float2(x); }

// Quantizes the 8 channels of one lane (16-bit pairs u), whose block's other
// 24 are on the lanes j ^ 1, j ^ 2, j ^ 3 (j = lane % 4 is the place in the
// block). Returns the code word in key order and the block's scale. Pairs are
// worked on together where there are instructions for it (an append of 7814
// tokens, 8 heads of 128: 36 us element by element, 24 in pairs).
template <typename T>
__device__ __forceinline__ uint32_t quantize8(const uint32_t* u, int j, __half& scale) {
  using Pair = decltype(pair_of(T(), 0u));
  Pair x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair y = pair_of(T(), u[i]);
    x[i] = pair_of(T(), u[i] & __heq2_mask(y, y));   // NaN counts as 0
  }
  // the block's largest x and largest -x
  const Pair hi = __hmax2(__hmax2(x[0], x[1]), __hmax2(x[2], x[3]));
  const Pair lo = __hmin2(__hmin2(x[0], x[1]), __hmin2(x[2], x[3]));
  Pair both;
  both.x = __hmax(hi.x, hi.y);
  both.y = __hneg(__hmin(lo.x, lo.y));
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&both), m);
    both = __hmax2(both, pair_of(T(), other));
  }
  const float2 pn = to_floats(both);
  float top = pn.x > pn.y ? pn.x : -pn.y;
  if (__any_sync(0xffffffffu, pn.x == pn.y && pn.x != 0.0f)) {
    // +top and -top: the first one's sign
    int at = 64;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float2 y = to_floats(x[i >> 1]);
      const float z = i & 1 ? y.y : y.x;
      if (fabsf(z) == pn.x) at = 2 * (8 * j + i) + (z < 0.0f);
    }
#pragma unroll
    for (int m = 1; m <= 2; m <<= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, m));
    if (pn.x == pn.y) top = at & 1 ? -pn.x : pn.x;
  }
  top = fminf(fmaxf(top, -65504.0f), 65504.0f);
  // 7 significant bits, to nearest even
  unsigned b = __float_as_uint(top * -0.125f);
  b = (b + 0xFFFFu + ((b >> 17) & 1u)) & ~0x1FFFFu;
  scale = __float2half_rn(fminf(fmaxf(__uint_as_float(b), -kMaxScale), kMaxScale));
  const float d = __half2float(scale);
  // floor(x / d + 8.5), exactly, as the whole number nearest to x / d + 8 with
  // ties up: x has at most 11 significant bits and d 7, so x / d + 8.5 is a
  // whole number or at least 2^-14 away from one. The product with the
  // reciprocal is off by less than 2^-19; 2^-16 more lifts the ties over their
  // boundary and nothing else. 2^23 added and taken away rounds to whole.
  const float inv = d == 0.0f ? 0.0f : copysignf(__frcp_rn(fabsf(d)), d);
  float even[4], odd[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = to_floats(x[i]);
    even[i] = y.x, odd[i] = y.y;
    fma_f32x2(even[i], odd[i], inv, 8.0f + 0x1p-16f);
    even[i] = fminf(fmaxf(even[i], 0.0f), 15.0f);
    odd[i] = fminf(fmaxf(odd[i], 0.0f), 15.0f);
    add_f32x2(even[i], odd[i], 0x1p23f, 0x1p23f);
    add_f32x2(even[i], odd[i], -0x1p23f, -0x1p23f);
  }
  // four codes of a half word, in fp32 (below 2^16), then as bits under 2^23
  const float e = fmaf(fmaf(fmaf(even[3], 16.0f, even[2]), 16.0f, even[1]), 16.0f, even[0]) + 0x1p23f;
  const float o = fmaf(fmaf(fmaf(odd[3], 16.0f, odd[2]), 16.0f, odd[1]), 16.0f, odd[0]) + 0x1p23f;
  return prmt(__float_as_uint(e), __float_as_uint(o), 0x5410u);
}

// One lane takes 8 channels of a key or value row (word j of block b), GROUPS
// times. Its elements are on their way before the token's place in the cache
// is looked up, a chain of four small loads that would otherwise set the time.
// Bound: 2 D bytes read and 9/16 D written a row, 41 MB and 6.3 us for 7814
// tokens and 8 heads of 128; measured 24.5 us (33 before the loads came first):
// 17.8 M warp instructions, 285 for each two rows, keep the issue slots 75 %
// busy, with the math pipes next (DRAM 15 %).
template <int D, typename T, int GROUPS>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  using F = Fmt<D>;
  constexpr int kItems = D / 8;
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int warp = (int)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int token = warp / p.chunks;
  if (token >= p.tokens) return;
  const int item0 = (warp - token * p.chunks) * (32 * GROUPS) + lane;
  alignas(16) uint32_t e[GROUPS][4];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int item = item0 + 32 * g, row = item / kItems, piece = item - row * kItems;   // row: 2 * head + (value)
    const int head = row >> 1;
    if (head < p.c.heads) {
      const T* src = row & 1 ? static_cast<const T*>(p.v) + token * p.v_token + head * p.v_head
                             : static_cast<const T*>(p.k) + token * p.k_token + head * p.k_head;
      if (p.vec) {
        *reinterpret_cast<uint4*>(e[g]) = __ldg(reinterpret_cast<const uint4*>(src + piece * 8));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(e[g])[i] = src[piece * 8 + i];
      }
    } else {
      *reinterpret_cast<uint4*>(e[g]) = make_uint4(0, 0, 0, 0);
    }
  }
  const int b = sequence_of(p.q_start, p.c.batch, token, lane);
  if (b < 0) return;
  bool bad = false;
  int first, n;
  rows_of(p.q_start, b, p.tokens, first, n, bad);
  const int len = cached(p.c, b, bad);
  const int i = token - first;
  const int slot = len - n + i;
  const bool inside = i < n;
  if (i < 0 || (inside && slot < 0)) bad = true;   // i < 0: the starts do not rise
  int page = 0;
  if (!bad && inside) page = page_of(p.c, p.c.table, p.c.table_cols, b, slot / kPage, bad);
  if (bad) {   // an index out of range: nothing is written
    if (lane == 0) atomicOr(p.error, kErrIndex);
    return;
  }
  if (!inside) return;
  const int t = slot & (kPage - 1), sw = value_swizzle<D>(t);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int item = item0 + 32 * g, row = item / kItems, piece = item - row * kItems;
    const int head = row >> 1, blk = piece >> 2, j = piece & 3;
    __half d;
    const uint32_t w = quantize8<T>(e[g], j, d);
    if (head >= p.c.heads) continue;
    uint8_t* pg = p.c.pages + ((size_t)page * p.c.heads + head) * F::kPageBytes;
    if (!(row & 1)) {
      *reinterpret_cast<uint32_t*>(pg + t * F::kRow + (j * F::kBlocks + blk) * 4) = w;
      if (j == 0) *reinterpret_cast<__half*>(pg + F::kKeyScale + (t * F::kBlocks + blk) * 2) = d;
    } else {
      // the low half of the key-order word is the value word 2j, the high half 2j + 1
      uint8_t* r = pg + F::kValue + t * F::kRow;
      *reinterpret_cast<uint16_t*>(r + (((2 * j) ^ sw) * F::kBlocks + blk) * 2) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(r + (((2 * j + 1) ^ sw) * F::kBlocks + blk) * 2) = (uint16_t)(w >> 16);
      if (j == 0) *reinterpret_cast<__half*>(pg + F::kValueScale + (blk * kPage + tile_perm(t)) * 2) = d;
    }
  }
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct ReadParams {
  View c;
  const int* q_start;
  int tokens;
  int chunks;      // warps of a token: ceil(2 * heads / 8)
  __half *k, *v;
  unsigned* error;
};

// A group of 4 lanes takes a key or value row of one token and head: lane j
// reads words j of all blocks with one load and writes 16 bytes of each.
// Bound by the writes: 64000 tokens, 8 heads of 128: 60 us, 336 MB at 5.6 TB/s.
template <int D>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
  using F = Fmt<D>;
  constexpr int NB = F::kBlocks;
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int warp = (int)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int token = warp / p.chunks;
  if (token >= p.tokens) return;
  const int b = sequence_of(p.q_start, p.c.batch, token, lane);
  if (b < 0) return;
  bool bad = false;
  int first, n;
  rows_of(p.q_start, b, p.tokens, first, n, bad);
  const int len = cached(p.c, b, bad);
  const int i = token - first;
  const int slot = len - n + i;
  const bool inside = i < n;
  if (i < 0 || (inside && slot < 0)) bad = true;   // i < 0: the starts do not rise
  int page = 0;
  if (!bad && inside) page = page_of(p.c, p.c.table, p.c.table_cols, b, slot / kPage, bad);
  if (bad) {
    if (lane == 0) atomicOr(p.error, kErrIndex);
    return;
  }
  if (!inside) return;
  const int row = (warp - token * p.chunks) * 8 + (lane >> 2), j = lane & 3;
  const int head = row >> 1, isv = row & 1;
  if (head >= p.c.heads) return;
  const int t = slot & (kPage - 1);
  const uint8_t* pg = p.c.pages + ((size_t)page * p.c.heads + head) * F::kPageBytes;
  uint32_t x[NB];
  __half d[NB];
  if (!isv) {
    load_words<NB>(pg + t * F::kRow + j * 4 * NB, x);
    alignas(16) uint32_t sc[NB / 2];
    load_words<NB / 2>(pg + F::kKeyScale + t * 2 * NB, sc);
#pragma unroll
    for (int k = 0; k < NB; ++k) d[k] = reinterpret_cast<const __half*>(sc)[k];
  } else {
    uint32_t y[NB];   // value words 2j and 2j + 1 of all blocks
    load_words<NB>(pg + F::kValue + t * F::kRow + ((2 * j) ^ value_swizzle<D>(t)) * 2 * NB, y);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      x[k] = prmt(y[k / 2], y[NB / 2 + k / 2], k & 1 ? 0x7632u : 0x5410u);
      d[k] = reinterpret_cast<const __half*>(pg + F::kValueScale)[k * kPage + tile_perm(t)];
    }
  }
  __half* out = (isv ? p.v : p.k) + ((size_t)token * p.c.heads + head) * D + 8 * j;
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const __half2 d2 = __half2half2(d[k]);
    *reinterpret_cast<uint4*>(out + 32 * k) = dequant_key8(x[k], d2, minus_72(d2));
  }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
struct EvictParams {
  View c;
  const float* weights;
  float* weights_out;
  long long weights_cols;
  int* index;
  int* kv_len_out;
  const int* out_table;
  int out_cols, keep, recent;
  int in_place;
  unsigned* error;
};

// Order of the weights as unsigned numbers: larger weight, larger key; -0
// counts as 0, NaN as the least.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w + 0.0f);   // -0 + 0 = 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectKeys = 40960;   // weights that are held in shared memory at a time
constexpr int kSelectRows = kSelectKeys / 32;   // of 32 weights; a mask of ties and one of those that stay for each
constexpr int kSelectBytes = kSelectKeys * 4 + 2 * kSelectRows * 4;
static_assert(2 * kSelectRows >= 2048, "the histogram lies where the masks do");

// Inclusive sum over the lanes.
__device__ __forceinline__ unsigned warp_sum(unsigned x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, m);
    if (lane >= m) x += y;
  }
  return x;
}
// Exclusive sum of x over the CTA's 32 warps of threads.
__device__ __forceinline__ unsigned block_sum(unsigned x, unsigned* sums) {
  static_assert(kSelectThreads == 1024, "a lane per warp");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned run = warp_sum(x);
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  const unsigned y = sums[lane];
  return __shfl_sync(0xffffffffu, warp_sum(y) - y, warp) + run - x;
}

// Which tokens stay: one CTA per sequence and head. The (keep - recent)-th
// largest key is found digit by digit (11, 11 and 10 bits, a shared histogram
// each: wide digits spread weights of like size over many counters); then one
// ordered pass writes the kept slots, every warp a run of them, 32 at a time:
// ballots count and place them, so neighbouring lanes write neighbouring
// entries (a run per thread scattered its stores: 8 us of 31 for 64 rows of
// 32000). Among the tokens with exactly that key the lower slots win. The
// weights sit in shared memory; of longer sequences the histograms read them
// from global memory and the ordered pass goes part by part. 64 rows of 32000:
// 29 us (load 4, three digits 8, ordered pass 11), 8 rows of 1100: 8 us.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
  extern __shared__ unsigned select_smem[];
  float* held = reinterpret_cast<float*>(select_smem);
  unsigned* hist = select_smem + kSelectKeys;
  __shared__ unsigned sums[32], part_ties[32], part_stays[32];
  __shared__ unsigned pick[2];   // digit, keys still to find
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  const int b = blockIdx.x / p.c.heads, h = blockIdx.x - b * p.c.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bool bad = false;
  const int len = cached(p.c, b, bad);
  if (bad && tid == 0) atomicOr(p.error, kErrIndex);
  const int keep = min(len, p.keep), recent = min(p.recent, keep);
  const int old = len - recent, need = keep - recent;
  const size_t row = (size_t)b * p.c.heads + h;
  const float* w = p.weights + row * p.weights_cols;
  float* wo = p.weights_out + row * p.weights_cols;
  int* index = p.index + row * p.keep;
  const bool fits = len <= kSelectKeys;
  if (fits) {
#pragma unroll 8
    for (int i = tid; i < len; i += kSelectThreads) held[i] = w[i];
  }
  const float* keys = fits ? held : w;

  unsigned edge = 0, mask = 0, left = (unsigned)need;
  if (need > 0 && need < old) {
    for (int shift = 21;; shift = shift > 10 ? 10 : 0) {
      const int bins = shift ? 2048 : 1024;
      hist[tid] = hist[tid + 1024] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < old; i += kSelectThreads) {
        const unsigned key = weight_key(keys[i]);
        if ((key & mask) == edge) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      // the digit where the count from above reaches `left`: two digits a thread
      const int top = bins - 1 - 2 * tid;
      const unsigned n0 = top > 0 ? hist[top] : 0, n1 = top > 0 ? hist[top - 1] : 0;
      const unsigned above = block_sum(n0 + n1, sums);
      if (above < left && above + n0 + n1 >= left) {
        const bool second = above + n0 < left;
        pick[0] = (unsigned)(second ? top - 1 : top);
        pick[1] = left - above - (second ? n0 : 0);
      }
      __syncthreads();
      edge |= pick[0] << shift;
      mask |= (unsigned)(bins - 1) << shift;
      left = pick[1];
      if (shift == 0) break;
    }
  }
  // `left` tokens of key == edge and all of key > edge stay (need == old:
  // everything stays; need == 0: nothing); what is written has been read
  if (need == 0) edge = 0xffffffffu;   // no key is as large
  const int sure = need >= old ? 0 : old;   // from here on all stay
  unsigned* masks = hist;
  unsigned at = 0, ties = 0;   // kept, and ties met, in earlier parts
  for (int base = 0; base < len; base += kSelectKeys) {
    const int n = min(kSelectKeys, len - base);
    __syncthreads();
    if (!fits)
      for (int i = tid; i < n; i += kSelectThreads) held[i] = w[base + i];
    __syncthreads();
    const int run = (n + kSelectThreads - 1) / kSelectThreads * 32, i0 = min(n, warp * run), i1 = min(n, i0 + run);
    unsigned mine = 0, stays = 0;   // of the warp's run: ties, kept above them
#pragma unroll 4
    for (int i = i0; i < i1; i += 32) {
      const unsigned key = i + lane < i1 ? weight_key(held[i + lane]) : 0;
      const bool out = i + lane >= i1, last = base + i + lane >= sure;
      const unsigned tie = __ballot_sync(0xffffffffu, !out && !last && key == edge),
                     stay = __ballot_sync(0xffffffffu, !out && (last || key > edge));
      if (lane == 0) masks[i / 32] = tie, masks[kSelectRows + i / 32] = stay;
      mine += __popc(tie);
      stays += __popc(stay);
    }
    if (lane == 0) part_ties[warp] = mine, part_stays[warp] = stays;
    __syncthreads();
    // a lane per warp: ties before its run, those that stay (rank < left), where its run goes
    const unsigned its = part_ties[lane], ties_to = ties + warp_sum(its), ties_from = ties_to - its;
    const unsigned kept = part_stays[lane] + (ties_from < left ? min(its, left - ties_from) : 0);
    const unsigned kept_to = at + warp_sum(kept);
    unsigned rank = __shfl_sync(0xffffffffu, ties_from, warp);
    unsigned to = __shfl_sync(0xffffffffu, kept_to - kept, warp);
    ties = __shfl_sync(0xffffffffu, ties_to, 31);
    at = __shfl_sync(0xffffffffu, kept_to, 31);
    const unsigned below = (1u << lane) - 1;
#pragma unroll 4
    for (int i = i0; i < i1; i += 32) {
      const unsigned tied = masks[i / 32], above = masks[kSelectRows + i / 32], me = 1u << lane;
      const bool stay = (above & me) || ((tied & me) && rank + __popc(tied & below) < left);
      const unsigned staying = tied ? __ballot_sync(0xffffffffu, stay) : above;
      if (stay) {
        const unsigned x = to + __popc(staying & below);
        index[x] = base + i + lane;
        wo[x] = held[i + lane];
      }
      rank += __popc(tied);
      to += __popc(staying);
    }
  }
  for (int i = keep + tid; i < p.keep; i += kSelectThreads) index[i] = -1;
  __syncthreads();
  for (long long i = keep + tid; i < p.weights_cols; i += kSelectThreads) wo[i] = 0.0f;
  if (h == 0 && tid == 0) p.kv_len_out[b] = keep;
}

template <int D>
struct Piece {};   // what one of a token's 8 lanes moves: D/16 bytes
template <> struct Piece<64> { using type = uint32_t; };
template <> struct Piece<128> { using type = uint2; };
template <> struct Piece<256> { using type = uint4; };

template <int D>
struct MovedToken {
  typename Piece<D>::type k, v, ks;
  __half vs;
};

// Lane c of a token's 8 reads (writes) its share of slot t of a page.
template <int D>
__device__ __forceinline__ void read_token(const uint8_t* pg, int t, int c, MovedToken<D>& m) {
  using F = Fmt<D>;
  using P = typename Piece<D>::type;
  m.k = reinterpret_cast<const P*>(pg + t * F::kRow)[c];
  m.v = reinterpret_cast<const P*>(pg + F::kValue + t * F::kRow)[c ^ value_swizzle<D>(t)];
  if (c == 0) m.ks = reinterpret_cast<const P*>(pg + F::kKeyScale)[t];
  if (c < F::kBlocks) m.vs = reinterpret_cast<const __half*>(pg + F::kValueScale)[c * kPage + tile_perm(t)];
}
template <int D>
__device__ __forceinline__ void write_token(uint8_t* pg, int t, int c, const MovedToken<D>& m) {
  using F = Fmt<D>;
  using P = typename Piece<D>::type;
  reinterpret_cast<P*>(pg + t * F::kRow)[c] = m.k;
  reinterpret_cast<P*>(pg + F::kValue + t * F::kRow)[c ^ value_swizzle<D>(t)] = m.v;
  if (c == 0) reinterpret_cast<P*>(pg + F::kKeyScale)[t] = m.ks;
  if (c < F::kBlocks) reinterpret_cast<__half*>(pg + F::kValueScale)[c * kPage + tile_perm(t)] = m.vs;
}

// Moves the kept tokens, a group of 8 lanes to a token and ROWS tokens a lane
// at a time. To other pages: many small CTAs. In place: one large CTA per
// sequence and head goes through them in order: token i comes from a slot
// >= i, so once a round has been read, nothing that is still to be read lies
// below what the round writes. 64 rows of 8000 kept tokens, heads of 128: 40 us
// for 147 MB in gathered pieces of 8 to 64 bytes.
template <int D, bool IN_PLACE>
struct MoveGeo {
  static constexpr int kThreads = IN_PLACE ? 1024 : 256;
  static constexpr int kRows = IN_PLACE ? 4 : 2;
  static constexpr int kTokens = kThreads / 8 * kRows;   // of a CTA in a round
};

template <int D, bool IN_PLACE>
__global__ void __launch_bounds__(MoveGeo<D, IN_PLACE>::kThreads)
    evict_move_kernel(const EvictParams p, int ctas_per_row) {
  using F = Fmt<D>;
  using G = MoveGeo<D, IN_PLACE>;
  constexpr int R = G::kRows, kGroups = G::kThreads / 8;
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  const int row = blockIdx.x / ctas_per_row, part = blockIdx.x - row * ctas_per_row;
  const int b = row / p.c.heads, h = row - b * p.c.heads;
  bool bad = false;
  const int len = cached(p.c, b, bad);
  const int keep = min(len, p.keep);
  if (IN_PLACE && keep == len) return;
  const int* index = p.index + (size_t)row * p.keep;
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3;
  const size_t page_stride = (size_t)p.c.heads * F::kPageBytes;
  uint8_t* base = p.c.pages + (size_t)h * F::kPageBytes;
  for (int i0 = part * G::kTokens; i0 < keep; i0 += ctas_per_row * G::kTokens) {
    MovedToken<D> m[R];
    int from[R], to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = i0 + r * kGroups + g;
      from[r] = i < keep ? index[i] : 0;
      to[r] = i < keep ? p.out_table[(size_t)b * p.out_cols + i / kPage] : 0;
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (i0 + r * kGroups + g < keep) {
        const int pg = page_of(p.c, p.c.table, p.c.table_cols, b, from[r] / kPage, bad);
        read_token<D>(base + pg * page_stride, from[r] & (kPage - 1), c, m[r]);
      }
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = i0 + r * kGroups + g;
      if (i < keep) {
        if ((unsigned)to[r] < (unsigned)p.c.num_pages)
          write_token<D>(base + to[r] * page_stride, i & (kPage - 1), c, m[r]);
        else
          bad = true;
      }
    }
    if (IN_PLACE) __syncthreads();
  }
  if (bad) atomicOr(p.error, kErrIndex);
}

}  // namespace kv4
}  // namespace busfill
