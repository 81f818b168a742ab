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
  int chunks;      // warps of a token: ceil(2 * heads * D / 8 / 32)
  int vec;         // 16-byte loads
  unsigned* error;
};

// Quantizes the 8 channels x of one lane, whose block's other 24 are on the
// lanes j ^ 1, j ^ 2, j ^ 3 (j = lane % 4 is the place in the block). Returns
// the code word in key order and the block's scale.
__device__ __forceinline__ uint32_t quantize8(float* x, int j, __half& scale) {
  float top = 0.0f;
  int at = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -65504.0f), 65504.0f) : 0.0f;
    if (fabsf(x[i]) > fabsf(top)) {
      top = x[i];
      at = 8 * j + i;
    }
  }
  // the block's value of largest magnitude, the first of equals
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, top, m);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, m);
    if (fabsf(t2) > fabsf(top) || (fabsf(t2) == fabsf(top) && a2 < at)) {
      top = t2;
      at = a2;
    }
  }
  // 7 significant bits, to nearest even
  unsigned u = __float_as_uint(top * -0.125f);
  u = (u + 0xFFFFu + ((u >> 17) & 1u)) & ~0x1FFFFu;
  scale = __float2half_rn(fminf(fmaxf(__uint_as_float(u), -kMaxScale), kMaxScale));
  const float d = __half2float(scale);
  // floor(x / d + 8.5), exactly: x has at most 11 significant bits and d 7, so
  // x / d + 8.5 is a whole number or at least 2^-14 away from one. The product
  // with the reciprocal is off by less than 2^-19; 2^-16 more lifts the ties
  // over their boundary and nothing else. (The IEEE division instead: 39 us
  // for 16000 tokens x 8 heads of 128, against 15.)
  const float inv = copysignf(__frcp_rn(fabsf(d)), d);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int q = __float2int_rd(fmaf(x[i], inv, 8.5f + 0x1p-16f));
    q = d == 0.0f ? 8 : min(max(q, 0), 15);
    w |= (uint32_t)q << (4 * ((i >> 1) + 4 * (i & 1)));
  }
  return w;
}

// One lane takes 8 channels of one key or value row: word j of block b.
template <int D, typename T>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  using F = Fmt<D>;
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
  if (inside && slot < 0) bad = true;
  int page = 0;
  if (inside && slot >= 0) page = page_of(p.c, p.c.table, p.c.table_cols, b, slot / kPage, bad);
  if (bad) {   // an index out of range: nothing is written
    if (lane == 0) atomicOr(p.error, kErrIndex);
    return;
  }
  if (!inside) return;
  constexpr int kItems = D / 8;
  const int item = (warp - token * p.chunks) * 32 + lane;
  const int row = item / kItems, piece = item - row * kItems;   // row: 2 * head + (value)
  const int head = row >> 1, isv = row & 1;
  const bool live = head < p.c.heads;
  const int blk = piece >> 2, j = piece & 3;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (live) {
    const T* src = isv ? static_cast<const T*>(p.v) + token * p.v_token + head * p.v_head
                       : static_cast<const T*>(p.k) + token * p.k_token + head * p.k_head;
    load8(src + piece * 8, p.vec, x);
  }
  __half d;
  const uint32_t w = quantize8(x, j, d);
  if (!live) return;
  const int t = slot & (kPage - 1);
  uint8_t* pg = p.c.pages + ((size_t)page * p.c.heads + head) * F::kPageBytes;
  if (!isv) {
    *reinterpret_cast<uint32_t*>(pg + t * F::kRow + (j * F::kBlocks + blk) * 4) = w;
    if (j == 0) *reinterpret_cast<__half*>(pg + F::kKeyScale + (t * F::kBlocks + blk) * 2) = d;
  } else {
    // the low half of the key-order word is the value word 2j, the high half 2j + 1
    const int sw = value_swizzle<D>(t);
    uint8_t* r = pg + F::kValue + t * F::kRow;
    *reinterpret_cast<uint16_t*>(r + (((2 * j) ^ sw) * F::kBlocks + blk) * 2) = (uint16_t)w;
    *reinterpret_cast<uint16_t*>(r + (((2 * j + 1) ^ sw) * F::kBlocks + blk) * 2) = (uint16_t)(w >> 16);
    if (j == 0) *reinterpret_cast<__half*>(pg + F::kValueScale + (blk * kPage + tile_perm(t)) * 2) = d;
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
  if (inside && slot < 0) bad = true;
  int page = 0;
  if (inside && slot >= 0) page = page_of(p.c, p.c.table, p.c.table_cols, b, slot / kPage, bad);
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

// Which tokens stay: one CTA per sequence and head. The (keep - recent)-th
// largest key is found digit by digit (8 bits a pass over the weights, a
// shared histogram), then one more pass writes the kept slots in order; among
// the tokens with exactly that key the lower slots win.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
  __shared__ unsigned hist[256];
  __shared__ unsigned sums[32], totals[2];
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

  unsigned edge = 0, mask = 0, left = (unsigned)need;
  if (need > 0 && need < old) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += kSelectThreads) {
        const unsigned key = weight_key(w[i]);
        if ((key & mask) == edge) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {   // the digit where the count from above reaches `left`
        unsigned mine = 0;
        for (int k = 0; k < 8; ++k) mine += hist[255 - (8 * lane + k)];
        unsigned run = mine;
        for (int m = 1; m < 32; m <<= 1) {
          const unsigned y = __shfl_up_sync(0xffffffffu, run, m);
          if (lane >= m) run += y;
        }
        unsigned above = run - mine;
        if (above < left && run >= left) {
          for (int k = 0; k < 8; ++k) {
            const unsigned n = hist[255 - (8 * lane + k)];
            if (above + n >= left) {
              pick[0] = 255u - (8 * lane + k);
              pick[1] = left - above;
              break;
            }
            above += n;
          }
        }
      }
      __syncthreads();
      edge |= pick[0] << shift;
      mask |= 255u << shift;
      left = pick[1];
      __syncthreads();
    }
  }
  // ordered pass: `left` tokens of key == edge and all of key > edge stay
  // (need == old: everything stays; need == 0: nothing)
  unsigned at = 0, ties = 0;
  const bool all = need >= old;
  for (int i0 = 0; i0 < len; i0 += kSelectThreads) {
    const int i = i0 + tid;
    float x = 0.0f;
    bool above = false, tie = false;
    if (i < len) {
      x = w[i];
      if (i >= old || all) {
        above = true;
      } else if (need > 0) {
        const unsigned key = weight_key(x);
        above = key > edge;
        tie = key == edge;
      }
    }
    // rank of the ties first, then of the kept
    unsigned bal = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) sums[warp] = __popc(bal);
    __syncthreads();
    if (warp == 0) {
      const unsigned mine = sums[lane];
      unsigned run = mine;
      for (int m = 1; m < 32; m <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, run, m);
        if (lane >= m) run += y;
      }
      sums[lane] = run - mine;
      if (lane == 31) totals[0] = run;
    }
    __syncthreads();
    const unsigned rank = ties + sums[warp] + __popc(bal & ((1u << lane) - 1));
    const bool stay = above || (tie && rank < left);
    ties += totals[0];
    __syncthreads();
    bal = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) sums[warp] = __popc(bal);
    __syncthreads();
    if (warp == 0) {
      const unsigned mine = sums[lane];
      unsigned run = mine;
      for (int m = 1; m < 32; m <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, run, m);
        if (lane >= m) run += y;
      }
      sums[lane] = run - mine;
      if (lane == 31) totals[1] = run;
    }
    __syncthreads();
    // kept tokens move down: what is written here has been read by now
    if (stay) {
      const unsigned to = at + sums[warp] + __popc(bal & ((1u << lane) - 1));
      index[to] = i;
      wo[to] = x;
    }
    at += totals[1];
    __syncthreads();
  }
  for (int i = keep + tid; i < p.keep; i += kSelectThreads) index[i] = -1;
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

// Moves the kept tokens. To other pages: every group of 8 lanes takes kept
// tokens of its own. In place: one CTA per sequence and head goes through
// them in order, kMoveRows groups at a time: token i comes from a slot >= i,
// so once a round has been read, nothing that is still to be read lies below
// what the round writes.
constexpr int kMoveThreads = 512;
constexpr int kMoveRows = 4;   // tokens a lane holds in one round

template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p, int ctas_per_row) {
  using F = Fmt<D>;
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  const int row = blockIdx.x / ctas_per_row, part = blockIdx.x - row * ctas_per_row;
  const int b = row / p.c.heads, h = row - b * p.c.heads;
  bool bad = false;
  const int len = cached(p.c, b, bad);
  const int keep = min(len, p.keep);
  if (p.in_place && keep == len) return;
  const int* index = p.index + (size_t)row * p.keep;
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3;
  constexpr int kGroups = kMoveThreads / 8;
  const size_t page_stride = (size_t)p.c.heads * F::kPageBytes;
  uint8_t* base = p.c.pages + (size_t)h * F::kPageBytes;
  for (int i0 = part * kGroups * kMoveRows; i0 < keep; i0 += ctas_per_row * kGroups * kMoveRows) {
    MovedToken<D> m[kMoveRows];
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
      const int i = i0 + r * kGroups + g;
      if (i < keep) {
        const int from = index[i];
        const int pg = page_of(p.c, p.c.table, p.c.table_cols, b, from / kPage, bad);
        read_token<D>(base + pg * page_stride, from & (kPage - 1), c, m[r]);
      }
    }
    if (p.in_place) __syncthreads();
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
      const int i = i0 + r * kGroups + g;
      if (i < keep) {
        const int to = p.out_table[(size_t)b * p.out_cols + i / kPage];
        if ((unsigned)to < (unsigned)p.c.num_pages)
          write_token<D>(base + to * page_stride, i & (kPage - 1), c, m[r]);
        else
          bad = true;
      }
    }
    if (p.in_place) __syncthreads();
  }
  if (bad) atomicOr(p.error, kErrIndex);
}

}  // namespace kv4
}  // namespace busfill
