// Attention over the 4-bit cache for few query rows per sequence and head
// (single tokens, speculated tokens).
//
//   out[r] = sum_s p[r,s] v[s],  p = softmax_s(scale * q[r] . k[s])
//
// Bound: every cached token costs 9/8 D bytes (K and V codes and scales, once
// per key/value head) and, for G query heads a group, 4 G D flops: the bytes
// bound it while the codes can be turned into matrix operands fast enough. So
// the codes go into the matrix instructions almost as they are:
//   * A 4-bit code c under zero exponent bits is the fp16 subnormal c 2^-24
//     (or, four bits up, c 2^-20), exactly, and the tensor core multiplies
//     subnormals like any other number: one AND per two values. The factor
//     16 between the nibbles is taken from q (keys: exact in fp16, q is
//     brought to a row maximum near 2^10 by a power of two first) or from
//     the sums (values).
//   * The -8 of (c - 8) d leaves the sums: sum q (c - 8) starts its
//     accumulator at -8 sum q; sum p d (c - 8) subtracts 8 sum p d, which one
//     more matrix instruction per block (an operand of ones) adds up from
//     the same rounded products.
//   * Scales never touch the codes: the keys' multiply the finished block
//     sums in fp32, the values' multiply p, in fp32 too. p d is rounded to
//     fp16 once (the matrix operand, and the transposition between the two
//     products moves 16-bit pairs). It uses fp16's whole range: the row's
//     reference is set by the largest p d of a page, so only terms 2^-25 below
//     the largest one lose bits, whatever the size of the values.
//   * The tensor core lines a subnormal's products up as if it were 2^-14, so
//     what is added up is good to about 2^-14 of a code step: an element whose
//     sum cancels is off by up to 1e-5 of its block's largest value (the rows'
//     error against 64 bits is that of one fp16 rounding, 2.6e-4, up to 131071
//     tokens of like weight).
// The matrix instruction is m16n8k16 with the tokens (scores) or channels
// (output) as its 16 rows and the query rows as its 8 columns, so that a
// group of 8 query heads fills it.
//
// Work. A unit is one page of one (sequence, head, row group of 8 NT rows).
// Units are numbered sequence by sequence and dealt out evenly, in ranges, to
// all warps of a persistent grid: the split follows the lengths on the
// device, whatever they are. A warp streams its pages with bulk copies into a
// ring of its own and meets no other warp until its range is done. A range
// begins and ends inside an item, as a rule: the pieces of an item are joined
// first inside the CTA, then, by the CTA that comes last (a counter), from
// the workspace; always in the order of the ranges, so results repeat bit for
// bit.
//
// Measured, 64 query heads over 8 of 128: 32 sequences to 16000 tokens 86 us
// (353 MB, 4.1 TB/s; bulk copies of that size alone 64-74 us), one of 131071
// 46 us (151 MB, 3.3 TB/s), one of 300 9 us.
#pragma once

#include "kv4_format.cuh"

namespace busfill {
namespace kv4 {

constexpr int kMaxBatch = 1024;
constexpr float kLag = 4.0f;    // log2 growth of a row's maximum that is not followed
constexpr float kLift = 11.0f;  // log2 of p d at the row's reference; p d < 2^(kLift + kLag), with room in fp16
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  View c;
  const void* q;
  void* out;
  float* lse;        // [tokens][q_heads] or nullptr
  float* weights;    // [batch][heads][weights_cols] (weights kernel)
  const int* q_start;
  long long q_token, q_head, o_token, o_head, weights_cols;
  float scale_log2;  // scale * log2(e)
  int tokens, q_heads, group, max_q;
  Divisor by_group;  // division by group
  int causal, window, bf16;
  int wide_out;      // output rows start on 32 bytes
  unsigned* counters;   // one per CTA, zero between calls
  unsigned* refused;    // whether the attention kernel refused the call, for the weights' pass behind it
  float* part;          // partial results (layout of the kernel)
  unsigned* error;
};

// the bulk copy global -> shared (bytes a multiple of 16) counted on an mbarrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// d += a b
__device__ __forceinline__ void mma_16816(float* d, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// d = a b + c
__device__ __forceinline__ void mma_16816_from(float* d, const uint32_t* a, const uint32_t* b, const float* c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a sequence asks for: its rows, and the pages that some row of it sees.
struct Span {
  int first, n;     // rows of the step's tensors, max_q at most
  int len;          // cached tokens
  int past;         // cached tokens before the first row's own (negative: rows that see nothing)
  int page0, pages; // pages [page0, page0 + pages)
};
__device__ __forceinline__ Span span_of(const AttnParams& p, int b, bool& bad) {
  Span s;
  rows_of(p.q_start, b, p.tokens, s.first, s.n, bad);
  s.len = cached(p.c, b, bad);
  s.past = s.len - s.n;
  if (s.n > p.max_q) {
    bad = true;
    s.n = p.max_q;
  }
  const int lo = p.window > 0 ? max(0, min(s.past + 1 - p.window, s.len - 1)) : 0;
  s.page0 = lo / kPage;
  s.pages = s.n > 0 && s.len > 0 ? (s.len + kPage - 1) / kPage - s.page0 : 0;
  return s;
}
// slots [lo, hi) that row i of the span sees
__device__ __forceinline__ void sees(const AttnParams& p, const Span& s, int i, int& lo, int& hi) {
  hi = p.causal ? min(s.len, s.past + i + 1) : s.len;
  lo = p.window > 0 ? max(0, s.past + i + 1 - p.window) : 0;
}

// The warp's sum.
__device__ __forceinline__ long long warp_total(long long x) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}
// A sequence's units for running_sum: more than 2^30 as a number that it refuses.
__device__ __forceinline__ int counted(long long units) {
  return (int)min(units, (1ll << 30) + (1ll << 16));
}
// pre[1 .. n] (of `counted`) to its running sum, pre[0] = 0 (one warp).
// More than about 2^30 in all is refused: no work, and reported; or all of it
// is, if `refused` says so. Returns whether it was.
__device__ __forceinline__ bool running_sum(int* pre, int n, int lane, bool& bad, bool refused = false) {
  int total = 0, size = 0;
  for (int i = lane; i < n; i += 32) size += (pre[i + 1] >> 16) + 1;
  const bool over = refused || __reduce_add_sync(0xffffffffu, size) > (1 << 14) + n;
  bad = bad || over;
  if (lane == 0) pre[0] = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    int x = i0 + lane < n && !over ? pre[i0 + lane + 1] : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, m);
      if (lane >= m) x += y;
    }
    if (i0 + lane < n) pre[i0 + lane + 1] = total + x;
    total += __shfl_sync(0xffffffffu, x, 31);
  }
  return over;
}
// running_sum in an attention kernel, which also tells the weights' pass.
__device__ __forceinline__ void running_sum_first(const AttnParams& p, int* pre, int lane, bool& bad) {
  const bool over = running_sum(pre, p.c.batch, lane, bad);
  if (p.weights && blockIdx.x == 0 && lane == 0) *p.refused = over;
}

// Query operand of one row group of 8 rows, and per column pair (2j, 2j + 1)
// of the score fragments: -8 sum(q) of every block, the factor to log2
// scores, the slots seen.
template <int D>
struct QueryTile {
  uint32_t b[Fmt<D>::kBlocks][4];   // [block][2 * half + reg]
  float corr[Fmt<D>::kBlocks][4];   // as the accumulator's start: columns 2j, 2j + 1 twice
  float factor[2];
  int lo[2], hi[2];
};

template <int D>
__device__ __forceinline__ void load_queries(const AttnParams& p, const Span& s, int head, int r0, int lane,
                                             QueryTile<D>& t) {
  constexpr int NB = Fmt<D>::kBlocks;
  const int n = lane >> 2, j = lane & 3;
  const int row = r0 + n, i = p.by_group(row);
  const bool live = i < s.n;
  float x[NB][8];
  float top = 0.0f;
  const uint16_t* src = static_cast<const uint16_t*>(p.q) + (size_t)(s.first + i) * p.q_token +
                        (size_t)(head * p.group + row - i * p.group) * p.q_head + 8 * j;
  uint4 raw[NB];   // all loads before the first use: one latency, not one a block
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    raw[b] = make_uint4(0, 0, 0, 0);
    if (live) raw[b] = __ldg(reinterpret_cast<const uint4*>(src + 32 * b));
  }
  if (p.bf16) {
#pragma unroll
    for (int b = 0; b < NB; ++b) to_floats<__nv_bfloat16>(raw[b], x[b]);
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) to_floats<__half>(raw[b], x[b]);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[b][e]));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // power of two that brings the row's maximum to [2^9, 2^10); none for 0 and
  // non-finite rows
  int e = 136 - (int)(__float_as_uint(top) >> 23);
  if (top == 0.0f || !(top <= 3.4e38f)) e = 0;
  e = max(-126, min(126, e));
  // the scale's sign goes to the queries, so that the factor orders scores;
  // codes weigh 2^-24 (see above); -inf times the factor stays -inf
  const float up = copysignf(__uint_as_float((unsigned)(127 + e) << 23), p.scale_log2);
  const float factor =
      fmaxf(fabsf(p.scale_log2) * __uint_as_float((unsigned)(127 - e) << 23) * 16777216.0f, 1e-37f);
  float corr[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      const float y0 = x[b][k] * up, y1 = x[b][k + 1] * up, y2 = x[b][k + 2] * up, y3 = x[b][k + 3] * up;
      sum += (y0 + y1) + (y2 + y3);
      t.b[b][k / 2] = h2_as_u32(__floats2half2_rn(y0, y1));
      t.b[b][k / 2 + 1] = h2_as_u32(__floats2half2_rn(y2 * 0.0625f, y3 * 0.0625f));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    corr[b] = sum * (-8.0f / 16777216.0f);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int from = 4 * (2 * j + k);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      t.corr[b][k] = t.corr[b][k + 2] = __shfl_sync(0xffffffffu, corr[b], from);
      asm("" : "+f"(t.corr[b][k + 2]));   // four registers, ready to be an accumulator
    }
    t.factor[k] = __shfl_sync(0xffffffffu, factor, from);
    const int ri = p.by_group(r0 + 2 * j + k);
    t.lo[k] = 0;   // columns without a row see everything, so that they hold up no page
    t.hi[k] = s.len;
    if (ri < s.n) sees(p, s, ri, t.lo[k], t.hi[k]);
  }
}

// Scores of 16 tokens (tokens 16 mt .. of the page) for NT row tiles, times
// nothing: s[nt][0..3] are rows (token tile_perm(lane / 4), and + 8) x column
// pair. To log2 scores: * factor.
template <int D, int NT>
__device__ __forceinline__ void scores_16(const uint8_t* page, int mt, int lane, const QueryTile<D>* q, float (*s)[4]) {
  using F = Fmt<D>;
  constexpr int NB = F::kBlocks;
  const int j = lane & 3, t = 16 * mt + tile_perm(lane >> 2);
  uint32_t w0[NB], w1[NB], sc0[NB / 2], sc1[NB / 2];
  load_words<NB>(page + t * F::kRow + j * 4 * NB, w0);
  load_words<NB>(page + (t + 8) * F::kRow + j * 4 * NB, w1);
  load_words<NB / 2>(page + F::kKeyScale + t * 2 * NB, sc0);
  load_words<NB / 2>(page + F::kKeyScale + (t + 8) * 2 * NB, sc1);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t x0 = w0[b], x1 = w1[b];
    const uint32_t a0[4] = {x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u};
    const uint32_t a1[4] = {x0 >> 8 & 0x000f000fu, x1 >> 8 & 0x000f000fu, x0 >> 8 & 0x00f000f0u,
                            x1 >> 8 & 0x00f000f0u};
    const float2 d0 = __half22float2(u32_as_h2(sc0[b / 2])), d1 = __half22float2(u32_as_h2(sc1[b / 2]));
    const float e0 = b & 1 ? d0.y : d0.x, e1 = b & 1 ? d1.y : d1.x;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float acc[4];
      mma_16816_from(acc, a0, q[nt].b[b], q[nt].corr[b]);
      mma_16816(acc, a1, q[nt].b[b] + 2);
      s[nt][0] = fmaf(e0, acc[0], s[nt][0]);
      s[nt][1] = fmaf(e0, acc[1], s[nt][1]);
      s[nt][2] = fmaf(e1, acc[2], s[nt][2]);
      s[nt][3] = fmaf(e1, acc[3], s[nt][3]);
    }
  }
}

// Running output of NT row tiles: o is channels x rows. Lane (c = lane / 4,
// j = lane % 4) holds, of block b and half u, the channels 32b + 8(c/2) + 4u +
// (c%2) (regs 0, 1: rows 2j, 2j + 1; in 2^24 ths) and the same + 2 (regs 2, 3; in
// 2^20 ths); pd: sum of p d per block. m is the row's reference: the largest
// log2 of a page's greatest p and greatest |d| together, as far as that is
// followed, less kLift.
template <int D, int NT>
struct Running {
  float o[NT][Fmt<D>::kBlocks][2][4];
  float pd[NT][Fmt<D>::kBlocks][4];   // every row alike: a whole accumulator
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) m[nt][k] = -INFINITY, l[nt][k] = 0.0f;
#pragma unroll
      for (int b = 0; b < Fmt<D>::kBlocks; ++b) {
        pd[nt][b][0] = pd[nt][b][1] = pd[nt][b][2] = pd[nt][b][3] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[nt][b][e >> 2][e & 3] = 0.0f;
      }
    }
  }
};

// 2^x of it is above the largest |d| among the value scales of a page's `left`
// first tokens (what lies behind them may be anything): -14 for fp16's
// subnormals, or none.
template <int D>
__device__ __forceinline__ int above_value_scales(const uint8_t* scales, int left, int lane) {
  constexpr int NB = Fmt<D>::kBlocks;
  uint32_t w[NB];   // columns 2 NB lane .. of the blocks' 64 each
  load_words<NB>(scales + lane * 4 * NB, w);
  if (left < kPage) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int x = (2 * NB * lane + 2 * i) & (kPage - 1);
      w[i] &= (tile_perm(x) < left ? 0xffffu : 0u) | (tile_perm(x + 1) < left ? 0xffff0000u : 0u);
    }
  }
  __half2 top = __habs2(u32_as_h2(w[0]));
#pragma unroll
  for (int i = 1; i < NB; ++i) top = __hmax2(top, __habs2(u32_as_h2(w[i])));
  const unsigned bits = __reduce_max_sync(0xffffffffu, (unsigned)__half_as_ushort(__hmax(top.x, top.y)));
  return min(11, (int)(bits >> 10) - 14);
}

// One page (64 tokens, slots base .. base + 63) into the running output.
template <int D, int NT>
__device__ __forceinline__ void attend_page(const uint8_t* page, int base, int len, int lane, const QueryTile<D>* q,
                                            Running<D, NT>& run) {
  using F = Fmt<D>;
  constexpr int NB = F::kBlocks;
  const int c = lane >> 2, j = lane & 3;
  const float lift = (float)above_value_scales<D>(page + F::kValueScale, len - base, lane) - kLift;
  float s[4][NT][4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt) scores_16<D, NT>(page, mt, lane, q, s[mt]);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // the page lies inside what every row of the tile sees?
    const bool whole = base >= max(q[nt].lo[0], q[nt].lo[1]) && base + kPage <= min(q[nt].hi[0], q[nt].hi[1]);
    if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = base + 16 * mt + tile_perm(c) + 8 * (e >> 1);
          if (slot < q[nt].lo[e & 1] || slot >= q[nt].hi[e & 1]) s[mt][nt][e] = -INFINITY;
        }
    }
    float top[2] = {s[0][nt][0], s[0][nt][1]};
    top[0] = fmaxf(top[0], s[0][nt][2]);
    top[1] = fmaxf(top[1], s[0][nt][3]);
#pragma unroll
    for (int mt = 1; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], s[mt][nt][e]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], x));
      top[k] = fmaf(top[k], q[nt].factor[k], lift);
    }
    // The reference m follows only what has grown by more than kLag, as most
    // pages change some row's maximum a little.
    if (__any_sync(0xffffffffu, top[0] > run.m[nt][0] + kLag || top[1] > run.m[nt][1] + kLag)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float m = fmaxf(run.m[nt][k], top[k]);
        const float f = m == run.m[nt][k] ? 1.0f : exp2_approx(run.m[nt][k] - m);
        run.m[nt][k] = m;
        run.l[nt][k] *= f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int e = k; e < 8; e += 2) run.o[nt][b][e >> 2][e & 3] *= f;
          run.pd[nt][b][k] *= f;
          run.pd[nt][b][k + 2] *= f;
        }
      }
    }
    const float off[2] = {run.m[nt][0] == -INFINITY ? 0.0f : -run.m[nt][0],
                          run.m[nt][1] == -INFINITY ? 0.0f : -run.m[nt][1]};
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[mt][nt][e] = exp2_approx(fmaf(s[mt][nt][e], q[nt].factor[e & 1], off[e & 1]));
        run.l[nt][e & 1] += s[mt][nt][e];
      }
  }
  const uint8_t* vals = page + F::kValue;
  const uint8_t* vsc = page + F::kValueScale;
#pragma unroll
  for (int mt = 0; mt < 4; ++mt) {
    const int ta = 16 * mt + tile_perm(2 * j), tb = 16 * mt + tile_perm(2 * j + 1);
    uint32_t w[4][NB / 2];
    load_words<NB / 2>(vals + ta * F::kRow + (c ^ value_swizzle<D>(ta)) * 2 * NB, w[0]);
    load_words<NB / 2>(vals + tb * F::kRow + (c ^ value_swizzle<D>(tb)) * 2 * NB, w[1]);
    load_words<NB / 2>(vals + (ta + 8) * F::kRow + (c ^ value_swizzle<D>(ta + 8)) * 2 * NB, w[2]);
    load_words<NB / 2>(vals + (tb + 8) * F::kRow + (c ^ value_swizzle<D>(tb + 8)) * 2 * NB, w[3]);
    // slots behind the sequence hold anything, non-finite scales too
    const int left = len - base - 16 * mt;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // scales of the tokens whose scores the lane holds (column c: token tile_perm(c))
      const __half* sc = reinterpret_cast<const __half*>(vsc) + b * kPage + 16 * mt + c;
      float d0 = __half2float(sc[0]), d1 = __half2float(sc[8]);
      if (left < 16) {
        if (tile_perm(c) >= left) d0 = 0.0f;
        if (tile_perm(c) + 8 >= left) d1 = 0.0f;
      }
      const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
      const uint32_t x0 = prmt(w[0][b / 2], w[1][b / 2], sel), x1 = prmt(w[2][b / 2], w[3][b / 2], sel);
      const uint32_t a0[4] = {x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u};
      const uint32_t a1[4] = {x0 >> 8 & 0x000f000fu, x0 >> 8 & 0x00f000f0u, x1 >> 8 & 0x000f000fu,
                              x1 >> 8 & 0x00f000f0u};
      const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // rows (columns of the operand) x tokens 2j, 2j + 1 of each 8-token tile
        float x[4] = {s[mt][nt][0], s[mt][nt][1], s[mt][nt][2], s[mt][nt][3]};
        mul_f32x2(x[0], x[1], d0);
        mul_f32x2(x[2], x[3], d1);
        const uint32_t pb[2] = {transpose_8x8(h2_as_u32(__floats2half2_rn(x[0], x[1]))),
                                transpose_8x8(h2_as_u32(__floats2half2_rn(x[2], x[3])))};
        mma_16816(run.o[nt][b][0], a0, pb);
        mma_16816(run.o[nt][b][1], a1, pb);
        mma_16816(run.pd[nt][b], ones, pb);
      }
    }
  }
}

// The finished running output as plain sums: o[channel] = sum p v, and the
// row sums l over the warp.
template <int D, int NT>
__device__ __forceinline__ void settle(Running<D, NT>& run) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) run.l[nt][k] += __shfl_xor_sync(0xffffffffu, run.l[nt][k], x);
#pragma unroll
    for (int b = 0; b < Fmt<D>::kBlocks; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        run.o[nt][b][e >> 2][e & 3] =
            fmaf(run.o[nt][b][e >> 2][e & 3], e & 2 ? 1048576.0f : 16777216.0f, -8.0f * run.pd[nt][b][e & 1]);
  }
}
template <int D>
__device__ __forceinline__ int channel_of(int lane, int b, int u, int e) {
  const int c = lane >> 2;
  return 32 * b + 8 * (c >> 1) + 4 * u + (c & 1) + (e & 2);
}

template <int D>
__device__ __forceinline__ void store_out(const AttnParams& p, const Span& s, int head, int row, int ch, float x) {
  const int i = p.by_group(row);
  if (i >= s.n) return;
  const size_t at = (size_t)(s.first + i) * p.o_token + (size_t)(head * p.group + row - i * p.group) * p.o_head + ch;
  if (p.bf16)
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p.out)[at] = __float2half_rn(x);
}
// four channels, ch a multiple of 4
__device__ __forceinline__ void store_out4(const AttnParams& p, const Span& s, int head, int row, int ch,
                                           const float4& o, float f) {
  const int i = p.by_group(row);
  if (i >= s.n) return;
  const size_t at = (size_t)(s.first + i) * p.o_token + (size_t)(head * p.group + row - i * p.group) * p.o_head + ch;
  uint2 v;
  if (p.bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * f, o.y * f), b = __floats2bfloat162_rn(o.z * f, o.w * f);
    v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    v = make_uint2(h2_as_u32(__floats2half2_rn(o.x * f, o.y * f)), h2_as_u32(__floats2half2_rn(o.z * f, o.w * f)));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = v;
}
__device__ __forceinline__ void store_lse(const AttnParams& p, const Span& s, int head, int row, float m, float l) {
  const int i = p.by_group(row);
  if (!p.lse || i >= s.n) return;
  p.lse[(size_t)(s.first + i) * p.q_heads + head * p.group + row - i * p.group] =
      l > 0.0f ? (m + log2f(l)) * kLn2 : l == 0.0f ? -INFINITY : l;
}

// The rows [first, first + n) of a sequence with nothing cached: 0, lse -inf.
// One warp of every CTA comes here, and the CTAs share the rows.
template <int D>
__device__ __forceinline__ void store_empty_rows(const AttnParams& p, int first, int n, int lane) {
  constexpr int V = D / 8;   // 16-byte pieces of a row and head
  const long long step = (long long)gridDim.x * 32, me = (long long)blockIdx.x * 32 + lane;
  for (long long x = me; x < (long long)n * p.q_heads * V; x += step) {
    const long long r = x / V, i = r / p.q_heads;
    const size_t at = (size_t)(first + i) * p.o_token + (size_t)(r - i * p.q_heads) * p.o_head + 8 * (x - r * V);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) = make_uint4(0, 0, 0, 0);
  }
  if (p.lse)
    for (long long x = me; x < (long long)n * p.q_heads; x += step) p.lse[(size_t)first * p.q_heads + x] = -INFINITY;
}

// Position in the list of units.
struct Cursor {
  int b, head, rg, page;    // page: index in the sequence
  int rgs;                  // row groups of the sequence
  Span s;
};
static_assert(sizeof(Cursor) <= 64, "item slots in shared memory");

// Geometry by head dimension and row tiles: warps of a CTA (one CTA per SM)
// and pages of each warp's ring.
template <int D, int NT>
struct Geo {
  static constexpr int kWarps = D == 64 && NT == 1 ? 12 : 8;
  static constexpr int kStages = D == 64 ? 3 : D == 128 ? 2 : 1;
  static constexpr int kRows = 8 * NT;
  static constexpr int kPieceFloats = kRows * (D + 2);          // o, m, l of a piece
  static constexpr int kRingBytes = kStages * Fmt<D>::kPageBytes;
  static constexpr int kFirstOff = kWarps * kRingBytes;         // o of every warp's first piece
  static constexpr int kPreOff = kFirstOff + kWarps * kRows * D * 4;   // units before each sequence
  static constexpr int kBarOff = kPreOff + (kMaxBatch + 2) * 4;
  static constexpr int kMetaOff = kBarOff + kWarps * kStages * 8;      // m, then l, of every piece and row
  static constexpr int kItemOff = kMetaOff + 2 * 2 * kWarps * kRows * 4;   // the item of every piece
  static constexpr int kMiscOff = kItemOff + 2 * kWarps * 64;
  static constexpr int kBytes = kMiscOff + 512;
  static_assert(kPieceFloats * 4 <= kRingBytes && kPieceFloats % 4 == 0, "a piece fits the warp's ring");
  static_assert(kBytes <= 232448, "dynamic shared memory");
};
// workspace, per CTA: its two partial items
template <int D, int NT>
constexpr size_t part_floats() {
  return (size_t)2 * Geo<D, NT>::kPieceFloats;
}


// units before sequence b in pre[b]; sets the cursor to unit u < pre[batch]
template <int ROWS>
__device__ __forceinline__ void seek(const AttnParams& p, const int* pre, int u, Cursor& c, bool& bad) {
  int lo = 0, hi = p.c.batch;   // last b with pre[b] <= u; empty sequences before it share its start
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= u)
      lo = mid;
    else
      hi = mid;
  }
  c.b = lo;
  c.s = span_of(p, lo, bad);
  c.rgs = (c.s.n * p.group + ROWS - 1) / ROWS;
  int r = u - pre[lo];
  c.head = r / (c.rgs * c.s.pages);
  r -= c.head * c.rgs * c.s.pages;
  c.rg = r / c.s.pages;
  c.page = c.s.page0 + r - c.rg * c.s.pages;
}

// From any page of an item to the first of the next; true at a sequence's end.
template <int ROWS>
__device__ __forceinline__ bool next_item(const AttnParams& p, const int* pre, Cursor& c, bool& bad) {
  bool moved = false;
  if (++c.rg == c.rgs) {
    c.rg = 0;
    if (++c.head == p.c.heads) {
      c.head = 0;
      moved = true;
      do ++c.b;
      while (c.b < p.c.batch && pre[c.b + 1] == pre[c.b]);
      if (c.b < p.c.batch) {
        c.s = span_of(p, c.b, bad);
        c.rgs = (c.s.n * p.group + ROWS - 1) / ROWS;
      }
    }
  }
  c.page = c.s.page0;
  return moved;
}

// The pages of a range of units one after another, for the copies that run
// ahead: a cursor of its own; the warp's lanes hold the next 32 page numbers.
template <int D, int ROWS>
struct PageFeed {
  Cursor in;
  int held = -64, number = 0;   // lane i holds the number of page held + i

  __device__ explicit PageFeed(const Cursor& c) : in(c) {}
  __device__ __forceinline__ const uint8_t* next(const AttnParams& p, const int* pre, int lane, bool& bad) {
    if (in.page < held || in.page >= held + 32) {
      held = in.page;
      number = 0;
      if (held + lane < in.s.page0 + in.s.pages)
        number = page_of(p.c, p.c.table, p.c.table_cols, in.b, held + lane, bad);
    }
    const int pg = __shfl_sync(0xffffffffu, number, in.page - held);
    const uint8_t* src = p.c.pages + ((size_t)pg * p.c.heads + in.head) * Fmt<D>::kPageBytes;
    if (++in.page == in.s.page0 + in.s.pages && next_item<ROWS>(p, pre, in, bad)) held = -64;
    return src;
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(Geo<D, NT>::kWarps * 32, 1) attn_kernel(const __grid_constant__ AttnParams p) {
  using F = Fmt<D>;
  using G = Geo<D, NT>;
  constexpr int NB = F::kBlocks, ROWS = G::kRows, W = G::kWarps, S = G::kStages, PF = G::kPieceFloats;
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre = reinterpret_cast<int*>(smem + G::kPreOff);
  int* misc = reinterpret_cast<int*>(smem + G::kMiscOff);
  int* piece_item = misc;            // [2 * W]: first unit of the item, -1: no piece
  auto piece_cursor = [&](int i) { return reinterpret_cast<Cursor*>(smem + G::kItemOff + 64 * i); };
  float* meta_m = reinterpret_cast<float*>(smem + G::kMetaOff);
  float* meta_l = meta_m + 2 * W * ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * G::kRingBytes;
  const uint32_t ring_s = smem_u32(ring);
  const uint32_t bar0 = smem_u32(smem + G::kBarOff) + warp * S * 8;
  if (lane < S) mbar_init(bar0 + 8 * lane, 1);
  fence_mbar_init();
  if (threadIdx.x == 0) misc[126] = 0;
  __syncthreads();
  pdl_wait_prerequisites();
  pdl_launch_dependents();

  // units of every sequence, then their running sum (warp 0)
  bool bad = false;
  const int batch = p.c.batch;
  for (int b0 = 32 * warp; b0 < batch; b0 += W * 32) {
    const int b = b0 + lane;
    Span s{};
    if (b < batch) {
      s = span_of(p, b, bad);
      pre[b + 1] = counted((long long)p.c.heads * ((s.n * p.group + ROWS - 1) / ROWS) * s.pages);
      if (s.pages > 0) atomicAdd(&misc[126], p.c.heads * ((s.n * p.group + ROWS - 1) / ROWS));
    }
    for (unsigned left = __ballot_sync(0xffffffffu, s.n > 0 && s.pages == 0); left; left &= left - 1) {
      const int from = __ffs(left) - 1;
      store_empty_rows<D>(p, __shfl_sync(0xffffffffu, s.first, from), __shfl_sync(0xffffffffu, s.n, from), lane);
    }
  }
  __syncthreads();
  if (warp == 0) running_sum_first(p, pre, lane, bad);
  __syncthreads();
  const int T = pre[batch], items = misc[126];
  // CTAs that share the list: every one gets a unit; where a warp would get
  // two pages at most, no more than there are items, as a split item has to
  // be joined through the workspace (one sequence of 300 tokens, 8 heads: 8
  // CTAs of 5 pages, 9.6 us, against 40 of one page and 5 parts an item, 12.1 us then)
  const long long ctas = min((int)gridDim.x, max(min(items, T), (T + 2 * W - 1) / (2 * W)));
  if ((int)blockIdx.x >= ctas) {
    if (bad) atomicOr(p.error, kErrIndex);
    return;
  }
  const int c0 = (int)((long long)T * blockIdx.x / ctas), c1 = (int)((long long)T * (blockIdx.x + 1) / ctas);
  const int u0 = c0 + (int)((long long)(c1 - c0) * warp / W), u1 = c0 + (int)((long long)(c1 - c0) * (warp + 1) / W);

  float* my_part = p.part + (size_t)blockIdx.x * part_floats<D, NT>();
  if (lane == 0) piece_item[2 * warp] = piece_item[2 * warp + 1] = -1;
  bool ok = true;
  if (u0 < u1) {
    Cursor c;
    seek<ROWS>(p, pre, u0, c, bad);
    PageFeed<D, ROWS> feed(c);
    auto next_source = [&] { return feed.next(p, pre, lane, bad); };
    int issued = u0;
    for (int k = 0; k < S && issued < u1; ++k, ++issued) {
      const uint8_t* src = next_source();
      if (lane == 0) {
        mbar_arrive_expect_tx(bar0 + 8 * k, F::kPageBytes);
        bulk_load(ring_s + k * F::kPageBytes, src, F::kPageBytes, bar0 + 8 * k);
      }
    }
    const uint8_t* ahead = issued < u1 ? next_source() : nullptr;

    QueryTile<D> q[NT];
    Running<D, NT> run;
    int stage = 0;
    uint32_t parity = 0;
    int item0 = u0 - (c.page - c.s.page0);   // first unit of the current item
    int begun = u0;                          // first unit of the current piece
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) load_queries<D>(p, c.s, c.head, c.rg * ROWS + 8 * nt, lane, q[nt]);
    run.clear();
    for (int u = u0; u < u1; ++u) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar0 + 8 * stage, parity));
      if (!ok) break;
      attend_page<D, NT>(ring + stage * F::kPageBytes, c.page * kPage, c.s.len, lane, q, run);
      __syncwarp();
      if (ahead) {
        if (lane == 0) {
          mbar_arrive_expect_tx(bar0 + 8 * stage, F::kPageBytes);
          bulk_load(ring_s + stage * F::kPageBytes, ahead, F::kPageBytes, bar0 + 8 * stage);
        }
        ++issued;
        ahead = issued < u1 ? next_source() : nullptr;
      }
      if (++stage == S) {
        stage = 0;
        parity ^= 1;
      }
      const bool ends = c.page + 1 == c.s.page0 + c.s.pages;
      if (!ends && u + 1 < u1) {
        ++c.page;
        continue;
      }
      // a piece is done
      settle<D, NT>(run);
      if (ends && begun == item0) {   // the whole item
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float inv[2] = {run.l[nt][0] == 0.0f ? 0.0f : 1.0f / run.l[nt][0],
                                run.l[nt][1] == 0.0f ? 0.0f : 1.0f / run.l[nt][1]};
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = c.rg * ROWS + 8 * nt + 2 * (lane & 3) + (e & 1);
              store_out<D>(p, c.s, c.head, row, channel_of<D>(lane, b, e >> 2, e),
                           run.o[nt][b][e >> 2][e & 3] * inv[e & 1]);
            }
          if (lane < 4) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              store_lse(p, c.s, c.head, c.rg * ROWS + 8 * nt + 2 * lane + k, run.m[nt][k], run.l[nt][k]);
          }
        }
      } else {
        // kept for the join: the last piece in the ring (all of it has
        // landed and been read), an earlier one beside it
        const bool last = u + 1 == u1;
        float* to = reinterpret_cast<float*>(last ? ring : smem + G::kFirstOff + warp * ROWS * D * 4);
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              to[(8 * nt + 2 * (lane & 3) + (e & 1)) * D + channel_of<D>(lane, b, e >> 2, e)] =
                  run.o[nt][b][e >> 2][e & 3];
          if (lane < 4) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              meta_m[(2 * warp + last) * ROWS + 8 * nt + 2 * lane + k] = run.m[nt][k];
              meta_l[(2 * warp + last) * ROWS + 8 * nt + 2 * lane + k] = run.l[nt][k];
            }
          }
        }
        if (lane == 0) {
          piece_item[2 * warp + last] = item0;
          *piece_cursor(2 * warp + last) = c;
        }
      }
      if (u + 1 < u1) {   // the next item
        next_item<ROWS>(p, pre, c, bad);
        item0 = begun = u + 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) load_queries<D>(p, c.s, c.head, c.rg * ROWS + 8 * nt, lane, q[nt]);
        run.clear();
      }
    }
    if (!ok && lane == 0) {   // gave up: nothing may land after the CTA is gone
      atomicOr(p.error, 1u);
      for (int k = 0; k < S; ++k) mbar_wait(bar0 + 8 * k, k < stage ? parity ^ 1 : parity);
    }
  }
  __threadfence_block();
  __syncthreads();

  // Join: first the CTA's own pieces, item by item (their m and l are in
  // shared memory), then, where this CTA is the last one of an item that is
  // split between CTAs, all CTAs' parts from the workspace. A task is 32
  // 4-channel pieces of an item's rows, one per lane of a warp. An empty piece
  // has m = -inf, l = 0, o = 0; NaN scores leave m at -inf and l NaN.
  constexpr int QUADS = D / 4, TASKS = ROWS * QUADS / 32;
  auto share = [](float m, float top) { return m == -INFINITY ? 1.0f : exp2_approx(m - top); };
  int* list = piece_item + 2 * W;   // the pieces there are, in order
  int* group = list + 2 * W;        // the first in `list` of every item
  int* counts = group + 2 * W + 1;  // items, and whether this CTA joins slot 0, slot 1
  if (warp == 0) {
    const bool has = lane < 2 * W && piece_item[lane < 2 * W ? lane : 0] >= 0;
    const unsigned all = __ballot_sync(0xffffffffu, has);
    if (has) list[__popc(all & ((1u << lane) - 1))] = lane;
    __syncwarp();
    const int n = __popc(all);
    const bool heads = lane < n && (lane == 0 || piece_item[list[lane]] != piece_item[list[lane - 1]]);
    const unsigned first = __ballot_sync(0xffffffffu, heads);
    if (heads) group[__popc(first & ((1u << lane) - 1))] = lane;
    if (lane == 0) {
      group[__popc(first)] = n;
      counts[0] = __popc(first);
      counts[1] = counts[2] = 0;
    }
  }
  __syncthreads();
  const int groups = counts[0];
  for (int task = warp; task < groups * TASKS; task += W) {
    const int g = task / TASKS, x = (task - g * TASKS) * 32 + lane, row = x / QUADS, ch = 4 * (x - row * QUADS);
    const int k0 = group[g], n = group[g + 1] - k0, item0 = piece_item[list[k0]];
    const Cursor& c = *piece_cursor(list[k0]);
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
    for (int i = 0; i < n; ++i) top = fmaxf(top, meta_m[list[k0 + i] * ROWS + row]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const int id = list[k0 + i];
      const float4 v = reinterpret_cast<const float4*>(
          smem + (id & 1 ? (id >> 1) * G::kRingBytes : G::kFirstOff + (id >> 1) * ROWS * D * 4))[x];
      const float f = share(meta_m[id * ROWS + row], top);
      sum = fmaf(meta_l[id * ROWS + row], f, sum);
      o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
    }
    if (item0 >= c0 && item0 + c.s.pages <= c1) {
      store_out4(p, c.s, c.head, c.rg * ROWS + row, ch, o, sum == 0.0f ? 0.0f : 1.0f / sum);
      if (ch == 0) store_lse(p, c.s, c.head, c.rg * ROWS + row, top, sum);
    } else {
      // slot 0: the item began before this CTA's range; slot 1: it goes on behind it
      float* to = my_part + (size_t)(item0 < c0 ? 0 : 1) * PF;
      reinterpret_cast<float4*>(to)[x] = o;
      if (ch == 0) to[ROWS * D + row] = top, to[ROWS * (D + 1) + row] = sum;
    }
  }
  __syncthreads();
  // An item in slot 0 or 1 is held by the CTAs [first, last]; the one that
  // arrives last joins the parts.
  auto item_of = [&](int slot) { return piece_cursor(list[slot == 0 ? 0 : group[groups - 1]]); };
  auto holders = [&](int slot, int& first, int& last) {
    const int item0 = piece_item[list[slot == 0 ? 0 : group[groups - 1]]];
    first = (int)((((long long)item0 + 1) * ctas - 1) / T);
    last = (int)(((long long)(item0 + item_of(slot)->s.pages) * ctas - 1) / T);
    return slot == 0 ? item0 < c0 : item0 >= c0 && item0 + item_of(slot)->s.pages > c1;
  };
  if (threadIdx.x < 64 && lane == 0 && groups > 0) {
    int first, last;
    if (holders(warp, first, last)) {
      __threadfence();
      if (atom_add_acq_rel_gpu(p.counters + first, 1u) == (unsigned)(last - first)) {
        p.counters[first] = 0;
        counts[1 + warp] = 1;
      }
    }
  }
  __syncthreads();
  for (int slot = 0; slot < 2; ++slot) {
    if (!counts[1 + slot]) continue;
    int first, last;
    holders(slot, first, last);
    const int n = last - first + 1;
    const Cursor& c = *item_of(slot);
    auto theirs = [&](int i) {
      return p.part + (size_t)(first + i) * part_floats<D, NT>() + (size_t)(i == 0 ? 1 : 0) * PF;
    };
    // The parts come to shared memory (the rings are free now), as many as fit
    // at a time: asynchronous copies keep all of them in flight with a short
    // loop. The reference moves with the parts.
    constexpr int FIT = W * G::kRingBytes / (PF * 4), EACH = (TASKS + W - 1) / W;
    float top[EACH], sum[EACH];
    float4 o[EACH];
#pragma unroll
    for (int t = 0; t < EACH; ++t) top[t] = -INFINITY, sum[t] = 0.0f, o[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < n; i0 += FIT) {
      const int have = min(FIT, n - i0);
      __syncthreads();
#pragma unroll 1
      for (int k = threadIdx.x; k < have * (PF / 4); k += W * 32)
        cp_async16(smem_u32(smem) + 16 * k, theirs(i0 + k / (PF / 4)) + 4 * (k % (PF / 4)), true);
      cp_async_wait_all();
      __syncthreads();
#pragma unroll
      for (int t = 0; t < EACH; ++t) {
        const int x = (warp + t * W) * 32 + lane, row = x / QUADS;
        if (warp + t * W >= TASKS) break;
        const float* parts = reinterpret_cast<const float*>(smem);
        float next = top[t];
        for (int i = 0; i < have; ++i) next = fmaxf(next, parts[i * PF + ROWS * D + row]);
        const float old = share(top[t], next);
        sum[t] *= old;
        o[t].x *= old, o[t].y *= old, o[t].z *= old, o[t].w *= old;
        top[t] = next;
#pragma unroll 2
        for (int i = 0; i < have; ++i) {
          const float4 v = reinterpret_cast<const float4*>(parts + i * PF)[x];
          const float f = share(parts[i * PF + ROWS * D + row], next);
          sum[t] = fmaf(parts[i * PF + ROWS * (D + 1) + row], f, sum[t]);
          o[t].x = fmaf(v.x, f, o[t].x), o[t].y = fmaf(v.y, f, o[t].y), o[t].z = fmaf(v.z, f, o[t].z),
          o[t].w = fmaf(v.w, f, o[t].w);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < EACH; ++t) {
      const int x = (warp + t * W) * 32 + lane, row = x / QUADS, ch = 4 * (x - row * QUADS);
      if (warp + t * W >= TASKS) break;
      store_out4(p, c.s, c.head, c.rg * ROWS + row, ch, o[t], sum[t] == 0.0f ? 0.0f : 1.0f / sum[t]);
      if (ch == 0) store_lse(p, c.s, c.head, c.rg * ROWS + row, top[t], sum[t]);
    }
  }
  if (bad) atomicOr(p.error, kErrIndex);
}

// The weight that the call's rows give every cached token, added to the
// running sums: weights[b][h][s] += sum over the rows r of the group of
// exp(score[r,s] - lse[r]). Keys only, so half the bytes of the attention. A
// warp streams whole pages (ranges of the list of all pages, as above) and
// walks over the rows that see each, so every sum has one owner and one order.
// One sequence of 131071 tokens, 8 heads of 128, one row of 64 heads: 27 us for
// 84 MB (75.5 of keys, the sums in and out), 3.1 TB/s.
template <int D>
struct WeightsGeo {
  static constexpr int kWarps = D == 256 ? 8 : 16;
  static constexpr int kStages = 3;
  static constexpr int kKeyBytes = 36 * D;   // key half of a page
  static constexpr int kRingBytes = kStages * kKeyBytes;
  static constexpr int kPreOff = kWarps * kRingBytes;
  static constexpr int kBarOff = kPreOff + (kMaxBatch + 2) * 4;
  static constexpr int kBytes = kBarOff + kWarps * kStages * 8;
  static_assert(kBytes <= 232448, "dynamic shared memory");
};

template <int D>
__global__ void __launch_bounds__(WeightsGeo<D>::kWarps * 32, 1) weights_kernel(const __grid_constant__ AttnParams p) {
  using G = WeightsGeo<D>;
  constexpr int W = G::kWarps, S = G::kStages, ROWS = 1 << 20;   // an item: all rows of a sequence and head
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre = reinterpret_cast<int*>(smem + G::kPreOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = p.c.batch;
  uint8_t* ring = smem + warp * G::kRingBytes;
  const uint32_t ring_s = smem_u32(ring), bar0 = smem_u32(smem + G::kBarOff) + warp * S * 8;
  if (lane < S) mbar_init(bar0 + 8 * lane, 1);
  fence_mbar_init();
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  bool bad = false;
  for (int b = threadIdx.x; b < batch; b += W * 32) {
    pre[b + 1] = counted((long long)p.c.heads * span_of(p, b, bad).pages);
  }
  __syncthreads();
  if (warp == 0) running_sum(pre, batch, lane, bad, *p.refused != 0);
  __syncthreads();
  const long long T = pre[batch], all = (long long)gridDim.x * W, me = (long long)blockIdx.x * W + warp;
  const int u0 = (int)(T * me / all), u1 = (int)(T * (me + 1) / all);
  bool ok = true;
  if (u0 < u1) {
    Cursor c;
    seek<ROWS>(p, pre, u0, c, bad);
    PageFeed<D, ROWS> feed(c);
    int issued = u0;
    auto issue = [&](int k) {
      const uint8_t* src = feed.next(p, pre, lane, bad);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar0 + 8 * k, G::kKeyBytes);
        bulk_load(ring_s + k * G::kKeyBytes, src, G::kKeyBytes, bar0 + 8 * k);
      }
      ++issued;
    };
    for (int k = 0; k < S && issued < u1; ++k) issue(k);
    QueryTile<D> q;
    float norm[2];
    auto load_rows = [&](int r0) {
      load_queries<D>(p, c.s, c.head, r0, lane, q);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = r0 + 2 * (lane & 3) + k, i = p.by_group(row);
        norm[k] = -INFINITY;   // no weight from rows that are not there or see nothing
        if (i < c.s.n) {
          const float x = p.lse[(size_t)(c.s.first + i) * p.q_heads + c.head * p.group + row - i * p.group] * -kLog2e;
          if (x != INFINITY) norm[k] = x;
        }
      }
    };
    const bool single = p.max_q * p.group <= 8;   // one row tile: loaded once per item
    if (single) load_rows(0);
    int stage = 0;
    uint32_t parity = 0;
    for (int u = u0; u < u1; ++u) {
      const int base = c.page * kPage, past = c.s.past;
      // lane 4r's slots, read ahead
      float* out = p.weights + ((size_t)c.b * p.c.heads + c.head) * p.weights_cols + base + tile_perm(lane >> 2);
      float sum[4][2];
      const bool owner = (lane & 3) == 0;
#pragma unroll
      for (int x = 0; x < 8; ++x)
        sum[x >> 1][x & 1] = owner && base + tile_perm(lane >> 2) + 8 * x < c.s.len ? out[8 * x] : 0.0f;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar0 + 8 * stage, parity));
      if (!ok) break;
      // rows that see the page: causal rows from the page's first slot on, and
      // with a window up to the last that still reaches it
      const int i0 = p.causal ? max(0, base - past) : 0;
      const int i1 = p.window > 0 ? min(c.s.n, base + kPage - 1 + p.window - past) : c.s.n;
      for (int r0 = i0 * p.group / 8 * 8; r0 < i1 * p.group; r0 += 8) {
        if (!single) load_rows(r0);
        const bool whole = __all_sync(0xffffffffu, base >= max(q.lo[0], q.lo[1]) && base + kPage <= min(q.hi[0], q.hi[1]));
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          float x[1][4];
          scores_16<D, 1>(ring + stage * G::kKeyBytes, mt, lane, &q, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int slot = base + 16 * mt + tile_perm(lane >> 2) + 8 * (e >> 1);
            const float w = exp2_approx(fmaf(x[0][e], q.factor[e & 1], norm[e & 1]));
            sum[mt][e >> 1] += whole || (slot >= q.lo[e & 1] && slot < q.hi[e & 1]) ? w : 0.0f;
          }
        }
      }
      __syncwarp();
      if (issued < u1) issue(stage);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        float y = sum[x >> 1][x & 1];
        y += __shfl_xor_sync(0xffffffffu, y, 1);
        y += __shfl_xor_sync(0xffffffffu, y, 2);
        if (owner && base + tile_perm(lane >> 2) + 8 * x < c.s.len) out[8 * x] = y;
      }
      if (++stage == S) {
        stage = 0;
        parity ^= 1;
      }
      if (u + 1 == u1) break;
      if (++c.page == c.s.page0 + c.s.pages) {
        next_item<ROWS>(p, pre, c, bad);
        if (single) load_rows(0);
      }
    }
    if (!ok && lane == 0) {   // gave up: nothing may land after the CTA is gone
      atomicOr(p.error, 1u);
      for (int k = 0; k < S; ++k) mbar_wait(bar0 + 8 * k, k < stage ? parity ^ 1 : parity);
    }
  }
  if (bad) atomicOr(p.error, kErrIndex);
}

}  // namespace kv4
}  // namespace busfill
