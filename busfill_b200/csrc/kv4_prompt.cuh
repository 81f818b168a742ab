// Attention over the 4-bit cache for many query rows per sequence and head
// (prompts), on tcgen05.
//
// The same sums as kv4_attn.cuh, in the regime that the tensor pipe bounds:
// 4 R L D flops for R query rows and L tokens against one pass of 9/8 L D bytes.
// A work item is 128 or 256 query rows (rows of one key/value head: tokens x
// heads of the group) against the tokens that they see, in tiles of kTile
// tokens:
//   S_i = Q_i K^T    (SS: both operands in shared memory, 128-byte swizzle)
//   P_i = exp2(S_i f - m)   in registers, one row per thread; fp16 into TMEM
//                    over S_i's columns
//   O_i += P_i V     (TS: P from TMEM; V as it lies in the cache, token by
//                    token, is the MN-major operand)
// The two row tiles i = 0, 1 take turns: while one's S is in the softmax
// threads, the tensor pipe works on the other. Codes are dequantized once per
// tile and CTA into a ring of fp16 operands, exactly ((c - 8) d has at most 11
// significant bits). Exponentials are taken against a reference 2^kRaise below
// a maximum of earlier scores; O is rescaled only when a score lies more than
// kOver (in log2) above the reference. P is rounded to fp16 once (the tensor
// core's operand); with the reference where it is, relatively for weights down
// to 2^-22 of the largest (with the reference at the maximum: to 2^-14, and
// what lay 2^-20 below a sink without a value was off by 1 to 9 %).
//
// Warps: 0 copies raw pages into a ring (bulk copies); 1 issues the MMAs and
// owns TMEM; 2 hands out the work; 4-7 and 8-11 softmax of row tile 0 and 1,
// thread = row; 12-15 dequantize. Registers move from the other warps to the
// softmax (64 and 192 of 128 at launch).
//
// Work split: the list of all items is cut into ranges of equal cost, one per
// CTA of a persistent grid, so ragged and causal shapes balance by themselves;
// an item costs its tiles and kItemCost more, and a range ends at an item's
// edge where that is near. An item that is cut leaves fp32 partial sums in the
// workspace, which the CTA that finishes last joins in the order of the ranges
// (repeatable). Warp 2 walks the list and hands out what comes next as
// descriptors in shared memory: the index arithmetic stays off the other warps.
//
// Measured, 64 query heads over 8 of 128: one prompt of 8000 tokens 1020 us
// (1030 TFLOP/s) after a pause, 1140 us sustained at the power cap; 3 of 1000
// 104 us. A pair
// of tiles takes 4500 cycles where its MMAs take 2080: the chain of score,
// softmax and P V that the two row tiles take turns in bounds it, not the
// exponentials (without a quarter of them 5 % less). An item's start and end
// (queries, first scores, epilogue) take some 8 us.
//
// Every wait is bounded (ptx.cuh: kWaitTimeoutNs).
#pragma once

#include "kv4_attn.cuh"

namespace busfill {
namespace kv4 {

// D[tmem] (+)= A[smem] B[smem]^T, kind::f16
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major, 128-byte swizzle: rows of 64 MN values (128 B) per K index, 8-row
// atoms of 1024 B along K (stride byte offset), blocks of 64 MN values
// `block_bytes` apart (leading byte offset).
__device__ __forceinline__ uint64_t make_sdesc_mn_sw128(uint32_t saddr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(block_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t kIdescBMnMajor = 1u << 16;

// 32 consecutive fp32 columns of this warp's lanes
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// Eight query elements (16-bit pairs in v) as fp16 operands: bf16 is brought to
// a row maximum in [2^9, 2^10) by a power of two (the row is on LANES
// neighbouring lanes), so that fp16 holds what bf16 held; fac takes its
// inverse. sign is the scale's.
template <int LANES>
__device__ __forceinline__ void normalize_query8(uint4& v, int bf16, float sign, float& fac) {
  if (bf16) {
    auto pair = [](uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); };
    auto bits = [](__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); };
    __nv_bfloat162 top = __hmax2(__hmax2(__habs2(pair(v.x)), __habs2(pair(v.y))),
                                 __hmax2(__habs2(pair(v.z)), __habs2(pair(v.w))));
#pragma unroll
    for (int y = 1; y < LANES; y <<= 1) top = __hmax2(top, pair(__shfl_xor_sync(0xffffffffu, bits(top), y)));
    const unsigned e = __bfloat16_as_ushort(__hmax(top.x, top.y)) >> 7;   // biased exponent; 255: not finite
    const int ex = e == 0 || e == 255 ? 0 : max(-126, min(126, 136 - (int)e));
    const __nv_bfloat162 up = __bfloat162bfloat162(
        __ushort_as_bfloat16((unsigned short)((127 + ex) << 7 | (sign < 0.0f ? 0x8000 : 0))));
    fac = fmaxf(fac * __uint_as_float((unsigned)(127 - ex) << 23), 1e-37f);   // not 0: -inf * fac stays -inf
    auto half = [&](uint32_t u) {
      const uint32_t x = bits(__hmul2(pair(u), up));   // exact
      return h2_as_u32(__floats2half2_rn(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)));
    };
    v = make_uint4(half(v.x), half(v.y), half(v.z), half(v.w));
  } else if (sign < 0.0f) {
    v.x ^= 0x80008000u, v.y ^= 0x80008000u, v.z ^= 0x80008000u, v.w ^= 0x80008000u;
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

namespace prompt {

constexpr int kThreads = 512;
constexpr int kSoftmaxWarp0 = 4, kDequantWarp0 = 12;
constexpr float kOver = 15.0f;   // how far, in log2, a score may lie above the row's reference (p < 2^15 in fp16)
// How far, in log2, below the maximum found the reference is set. What is left to
// kOver is how far a row may grow unfollowed (prompt of 8000 tokens: 15, 8 and 7
// left 1160 us, 4 left 1320, as some row of a warp's 32 outgrows it too often).
constexpr float kRaise = 8.0f;

template <int D>
struct Geo {
  using F = Fmt<D>;
  static constexpr int kTile = D == 256 ? 64 : 128;        // tokens of a tile
  static constexpr int kRowTiles = D == 256 ? 1 : 2;       // row tiles of 128 rows
  static constexpr int kRows = 128 * kRowTiles;
  static constexpr int kChunks = D / 64;                   // 128-byte column chunks
  static constexpr int kTilePages = kTile / kPage;
  static constexpr int kHalfPage = 36 * D;                 // keys (or values) of a page, scales behind
  static constexpr int kRawBytes = kTilePages * kHalfPage;
  static constexpr int kSlots = 4;                         // dequantized half tiles
  static constexpr int kRawStages = D == 64 ? 6 : 3;
  static constexpr int kSlotBytes = kTile * D * 2;
  static constexpr int kQTileBytes = 128 * D * 2;
  // shared memory
  static constexpr int kSlotOff = 0;
  static constexpr int kQOff = kSlotOff + kSlots * kSlotBytes;
  static constexpr int kRawOff = kQOff + kRowTiles * kQTileBytes;
  static constexpr int kFacOff = kRawOff + kRawStages * kRawBytes;      // factor of every row
  static constexpr int kBarOff = kFacOff + kRows * 4;
  static constexpr int kDescs = 4;                         // descriptors in flight
  static constexpr int bRawFull = 0, bRawEmpty = bRawFull + kRawStages, bKvFull = bRawEmpty + kRawStages,
                       bKvEmpty = bKvFull + kSlots, bS = bKvEmpty + kSlots, bP = bS + 2, bO = bP + 4, bQ = bO + 4,
                       bDescFull = bQ + 2, bDescEmpty = bDescFull + kDescs, bParts = bDescEmpty + kDescs,
                       bLast = bParts + 1, bFinal = bLast + 1, kBars = bFinal + 1;
  static constexpr int kMiscOff = kBarOff + kBars * 8;
  static constexpr int kDescOff = (kMiscOff + 16 + 15) / 16 * 16;
  static constexpr int kPreOff = kDescOff + kDescs * 64;   // cost before each sequence
  static constexpr int kBytes = kPreOff + (kMaxBatch + 1) * 4;
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kAlloc <= 232448, "dynamic shared memory");
  // TMEM columns
  static constexpr int kS = 0, kO = kRowTiles * kTile;
  static_assert(kO + kRowTiles * D <= 512, "TMEM");
  // a partial result: O [D][rows], m [rows], l [rows]
  static constexpr int kPartFloats = kRows * (D + 2);
};

// An item: group t of kRows rows of (sequence, head); tiles [tile0, tile0 + tiles).
struct Item {
  int b, head, t;
  int groups;          // of the sequence
  int tile0, tiles;
  Span s;
};
// What a CTA does of an item.
struct Work {
  int b, head, first, n;         // first row and rows of the sequence
  int len, row0, tile0, tiles;   // tiles 0: the end
  int page0, past;               // of the sequence's Span
  int kind, c_first, c_last, row_tiles;
};
enum { kWhole = 0, kTail = 1, kHead = 2 };   // kTail: began in an earlier CTA; kHead: goes on in the next
static_assert(sizeof(Work) <= 64, "descriptor slots");
// Tiles that the start and the end of an item are worth (queries, epilogue,
// refilling the pipeline).
constexpr int kItemCost = 2;
// A range is worth at least kMinCost tiles, and its end moves to an item's edge
// where that is at most kSnap tiles away: a cut costs some 12 us (write, fence,
// counter, join). Us with kSnap 0 (queries 2 us slower) / 3 / 4 / 8: 8 x 512
// rows on 512 tokens 52 / 29 / 28 / 29, 64 rows on 4096 tokens 39 / 39 / 41 /
// 47, 8 x 64 rows on 4096 tokens 58 / 57 / 59 / 66. With kMinCost 1 / 4 / 6, 64 rows on 4096 tokens:
// 51 / 39 / 52.
constexpr int kMinCost = 4;
constexpr int kSnap = 3;
static_assert(kSnap >= kItemCost, "a cut leaves tiles on both sides");
// how far behind its start an item of cost c is not cut
__device__ __forceinline__ int near_start(int c) { return min(kSnap, c / 2); }

template <int D>
__device__ __forceinline__ int groups_of(const AttnParams& p, const Span& s) {
  return s.len > 0 ? (s.n * p.group + Geo<D>::kRows - 1) / Geo<D>::kRows : 0;
}
// the tiles that some row of group t sees (one, all masked, if they see nothing)
template <int D>
__device__ __forceinline__ int tiles_of(const AttnParams& p, const Span& s, int t, int& tile0) {
  constexpr int R = Geo<D>::kRows, K = Geo<D>::kTile;
  const int i0 = p.by_group(t * R), i1 = min(s.n - 1, p.by_group(t * R + R - 1));
  int lo, hi, x;
  sees(p, s, i0, lo, x);
  sees(p, s, i1, x, hi);
  tile0 = min(lo, s.len - 1) / K;
  return max(1, (hi + K - 1) / K - tile0);
}

}  // namespace prompt

template <int D>
__global__ void __launch_bounds__(prompt::kThreads, 1) prompt_kernel(const __grid_constant__ AttnParams p) {
  using namespace prompt;
  using G = prompt::Geo<D>;
  using F = Fmt<D>;
  constexpr int K = G::kTile, RT = G::kRowTiles, NB = F::kBlocks;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  const uint32_t sbase = smem_u32(smem);
  auto BAR = [&](int i) { return sbase + G::kBarOff + 8u * (uint32_t)i; };
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + G::kMiscOff);   // [0] TMEM base, [1] "last" flag
  int* pre = reinterpret_cast<int*>(smem + G::kPreOff);
  float* factors = reinterpret_cast<float*>(smem + G::kFacOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = p.c.batch;

  if (warp == 0) {
    for (int i = lane; i < G::kBars; i += 32) {
      int n = 1;
      if ((i >= G::bRawEmpty && i < G::bKvEmpty) || (i >= G::bP && i < G::bP + 4) || (i >= G::bQ && i < G::bQ + 2))
        n = 4;
      if (i >= G::bDescEmpty && i < G::bDescEmpty + G::kDescs) n = 14;   // all warps but 2 and 3
      if (i == G::bParts) n = 8;
      mbar_init(BAR(i), n);
    }
    fence_mbar_init();
  } else if (warp == 1) {
    tmem_alloc(sbase + G::kMiscOff, 512);
    tmem_relinquish();
  }
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  // cost of every sequence (a warp each), then the running sum
  bool bad = false;
  for (int b = warp; b < batch; b += kThreads / 32) {
    const Span s = span_of(p, b, bad);
    const int groups = groups_of<D>(p, s);
    long long n = 0;
    int x;
    for (int t = lane; t < groups; t += 32) n += tiles_of<D>(p, s, t, x) + kItemCost;
    const long long cost = warp_total(n) * p.c.heads;
    if (lane == 0) pre[b + 1] = counted(cost);
    if (s.len == 0) store_empty_rows<D>(p, s.first, s.n, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) running_sum_first(p, pre, lane, bad);
  __syncthreads();
  const uint32_t tmem = misc[0];

  bool ok = true;
  auto wait = [&](int bar, uint32_t phase) -> bool {   // the warp waits for completion number `phase` of the barrier
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(BAR(bar), phase & 1));
    return ok;
  };
  auto failed = [&](unsigned bit) {
    if (lane == 0) atomicOr(p.error, bit);
  };
  uint32_t taken = 0;   // descriptors this warp has seen
  auto next_piece = [&]() -> Work {
    Work x;
    const int st = taken % G::kDescs;
    if (!wait(G::bDescFull + st, taken / G::kDescs)) {
      x.tiles = 0;
      return x;
    }
    x = *reinterpret_cast<const Work*>(smem + G::kDescOff + 64 * st);
    __syncwarp();
    if (lane == 0) mbar_arrive(BAR(G::bDescEmpty + st));
    ++taken;
    return x;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 2) {
      // ---------------- work list ----------------
      const int T = pre[batch];
      const long long ctas = max(1, min((int)gridDim.x, T / kMinCost));
      const bool idle = (int)blockIdx.x >= ctas;
      const int u0 = idle ? 0 : (int)((long long)T * blockIdx.x / ctas);
      const int u1 = idle ? 0 : (int)((long long)T * (blockIdx.x + 1) / ctas);
      uint32_t n = 0;
      auto push = [&](const Work& x) -> bool {
        const int st = n % G::kDescs;
        if (!wait(G::bDescEmpty + st, n / G::kDescs + 1)) return false;
        if (lane == 0) {
          *reinterpret_cast<Work*>(smem + G::kDescOff + 64 * st) = x;
          mbar_arrive(BAR(G::bDescFull + st));
        }
        __syncwarp();
        ++n;
        return true;
      };
      if (u0 < u1) {
        // the item at cost u0
        Item it;
        int lo = 0, hi = batch;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          (pre[mid] <= u0 ? lo : hi) = mid;
        }
        it.b = lo;
        it.s = span_of(p, lo, bad);
        it.groups = groups_of<D>(p, it.s);
        const int per_head = (pre[lo + 1] - pre[lo]) / p.c.heads;
        int r = u0 - pre[lo];
        it.head = r / per_head;
        r -= it.head * per_head;
        for (int t0 = 0;; t0 += 32) {
          int x0;
          const int c = t0 + lane < it.groups ? tiles_of<D>(p, it.s, t0 + lane, x0) + kItemCost : 0;
          int x = c;
#pragma unroll
          for (int m = 1; m < 32; m <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, m);
            if (lane >= m) x += y;
          }
          const unsigned over = __ballot_sync(0xffffffffu, x > r);
          if (over) {
            const int k = __ffs(over) - 1;
            it.t = t0 + k;
            r -= __shfl_sync(0xffffffffu, x - c, k);
            break;
          }
          r -= __shfl_sync(0xffffffffu, x, 31);
        }
        // A range ends at cost u: between tiles of the item that begins at x and
        // costs c, unless that is near an edge of the item.
        auto cut = [&](int u, int x, int c) {
          const int o = u - x;
          return o <= near_start(c) ? 0 : o + kSnap >= c ? c - kItemCost : o - kItemCost;
        };
        // the CTA whose range holds cost y
        auto cta_of = [&](int y) { return (int)((((long long)y + 1) * ctas - 1) / T); };
        for (int x = u0 - r;;) {
          it.tiles = tiles_of<D>(p, it.s, it.t, it.tile0);
          const int c = it.tiles + kItemCost, from = cut(u0, x, c), to = cut(u1, x, c);
          if (to > from) {
            Work y;
            y.b = it.b, y.head = it.head, y.first = it.s.first, y.n = it.s.n, y.len = it.s.len;
            y.page0 = it.s.page0, y.past = it.s.past;
            y.row0 = it.t * G::kRows, y.tile0 = it.tile0 + from, y.tiles = to - from;
            y.kind = from > 0 ? kTail : to < it.tiles ? kHead : kWhole;
            y.c_first = cta_of(x + near_start(c)), y.c_last = cta_of(x + c - kSnap - 1);
            y.row_tiles = RT == 2 && it.s.n * p.group - y.row0 > 128 ? 2 : 1;
            if (!push(y)) break;
            // its queries on their way to L2
            for (int k = lane; k < G::kRows; k += 32) {
              const int row = y.row0 + k, tok = p.by_group(row);
              if (tok < y.n) {
                const uint16_t* q = static_cast<const uint16_t*>(p.q) + (size_t)(y.first + tok) * p.q_token +
                                    (size_t)(y.head * p.group + row - tok * p.group) * p.q_head;
#pragma unroll
                for (int c = 0; c < D; c += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + c));
              }
            }
          }
          x += c;
          if (x >= u1) break;
          if (++it.t == it.groups) {
            it.t = 0;
            if (++it.head == p.c.heads) {
              it.head = 0;
              do ++it.b;
              while (it.b < batch && pre[it.b + 1] == pre[it.b]);
              if (it.b >= batch) break;
              it.s = span_of(p, it.b, bad);
              it.groups = groups_of<D>(p, it.s);
            }
          }
        }
      }
      Work end{};
      push(end);
      if (!ok) failed(1u);
    } else if (warp == 0) {
      // ---------------- raw pages ----------------
      uint32_t n = 0;
      for (Work x = next_piece(); ok && x.tiles > 0; x = next_piece()) {
        const int pages = (x.len + kPage - 1) / kPage;
        for (int j = 0; ok && j < x.tiles; ++j) {
          const int page0 = (x.tile0 + j) * G::kTilePages;
          // pages [skip, have) of the tile: the ones before every row's window
          // may have been given back, and are not looked up
          const int skip = max(0, x.page0 - page0), have = min(G::kTilePages, pages - page0);
          auto there = [&](int k) { return k >= skip && k < have; };
          const uint8_t* src[G::kTilePages];
#pragma unroll
          for (int k = 0; k < G::kTilePages; ++k)
            src[k] = p.c.pages +
                     ((size_t)(there(k) ? page_of(p.c, p.c.table, p.c.table_cols, x.b, page0 + k, bad) : 0) * p.c.heads +
                      x.head) * F::kPageBytes;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int st = n % G::kRawStages;
            if (!wait(G::bRawEmpty + st, n / G::kRawStages + 1)) break;
            if (elect_one()) {
              mbar_arrive_expect_tx(BAR(G::bRawFull + st), (have - skip) * G::kHalfPage);
#pragma unroll
              for (int k = 0; k < G::kTilePages; ++k)
                if (there(k))
                  bulk_load(sbase + G::kRawOff + st * G::kRawBytes + k * G::kHalfPage, src[k] + half * G::kHalfPage,
                            G::kHalfPage, BAR(G::bRawFull + st));
            }
            __syncwarp();
            ++n;
          }
        }
      }
      if (!ok) failed(1u);
      // nothing may land after the CTA is gone
      ok = true;
      for (uint32_t k = n > G::kRawStages ? n - G::kRawStages : 0; k < n; ++k)
        if (!wait(G::bRawFull + k % G::kRawStages, k / G::kRawStages)) break;
    } else if (warp == 1) {
      // ---------------- MMA ----------------
      constexpr uint32_t kIdescS = make_idesc_f16_f32(128, K), kIdescO = make_idesc_f16_f32(128, D) | kIdescBMnMajor;
      uint32_t half = 0;             // half tiles consumed
      uint32_t done[2] = {0, 0};     // tiles of row tile i whose P was waited for
      uint32_t items[2] = {0, 0};
      // descriptors are made once and stepped by their address field (16-byte
      // units): built anew for every MMA, their arithmetic kept the issuing
      // thread at 115 cycles an MMA of 65
      const uint64_t q_desc = make_sdesc_sw128(sbase + G::kQOff), k_desc = make_sdesc_sw128(sbase + G::kSlotOff),
                     v_desc = make_sdesc_mn_sw128(sbase + G::kSlotOff, K * 128);
      auto issue_s = [&](int i, uint32_t slot) {
        const uint64_t a = q_desc + (uint32_t)(i * G::kQTileBytes / 16), b = k_desc + slot * (G::kSlotBytes / 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_f16_ss(tmem + G::kS + i * K, a + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16,
                     b + ((k / 4) * K * 128 + (k % 4) * 32) / 16, kIdescS, k > 0);
        tc_commit(BAR(G::bS + i));
      };
      auto one_piece = [&](int nr, int tiles) -> bool {
        for (int i = 0; i < nr; ++i)
          if (!wait(G::bQ + i, items[i]++)) return false;
        if (!wait(G::bKvFull + half % G::kSlots, half / G::kSlots)) return false;
        tc_fence_after();
        if (elect_one()) {
          for (int i = 0; i < nr; ++i) issue_s(i, half % G::kSlots);
          tc_commit(BAR(G::bKvEmpty + half % G::kSlots));
        }
        __syncwarp();
        ++half;
        for (int j = 0; j < tiles; ++j) {
          const uint32_t vs = half % G::kSlots, ks = (half + 1) % G::kSlots;
          const bool more = j + 1 < tiles;
          if (!wait(G::bKvFull + vs, half / G::kSlots)) return false;
          if (more && !wait(G::bKvFull + ks, (half + 1) / G::kSlots)) return false;
          for (int i = 0; i < nr; ++i) {
            auto issue_o = [&](int part) {
              const uint64_t b = v_desc + vs * (G::kSlotBytes / 16);
#pragma unroll
              for (int x = 0; x < K / 32; ++x) {
                const int k = part * (K / 32) + x;
                mma_f16_ts(tmem + G::kO + i * D, tmem + G::kS + i * K + 8 * k,
                           b + k * 16 * 128 / 16, kIdescO, j > 0 || k > 0);
              }
            };
            if (!wait(G::bP + i, done[i])) return false;
            tc_fence_after();
            if (elect_one()) {
              issue_o(0);
              tc_commit(BAR(G::bO + i));
            }
            __syncwarp();
            if (!wait(G::bP + 2 + i, done[i]++)) return false;
            tc_fence_after();
            if (elect_one()) {
              issue_o(1);
              tc_commit(BAR(G::bO + 2 + i));
              if (more) issue_s(i, ks);
              if (i + 1 == nr) {
                tc_commit(BAR(G::bKvEmpty + vs));
                if (more) tc_commit(BAR(G::bKvEmpty + ks));
              }
            }
            __syncwarp();
          }
          half += more ? 2 : 1;
        }
        return true;
      };
      for (Work x = next_piece(); ok && x.tiles > 0; x = next_piece())
        if (!one_piece(x.row_tiles, x.tiles)) break;
      if (!ok) failed(4u);
      // every MMA has completed before TMEM is freed
      ok = true;
      tc_fence_after();
      if (elect_one()) tc_commit(BAR(G::bFinal));
      __syncwarp();
      if (!wait(G::bFinal, 0)) failed(32u);
    }
  } else if (warp >= kDequantWarp0) {
    // ---------------- dequantize ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int w = warp - kDequantWarp0, j = lane & 3;
    uint32_t n = 0;
    for (Work x0 = next_piece(); ok && x0.tiles > 0; x0 = next_piece()) {
      const int len = x0.len, low = x0.page0 * kPage;
      int base = x0.tile0 * K;
#pragma unroll 1
      for (int left = 2 * x0.tiles; left > 0; --left, ++n) {
        const int half = left & 1;   // keys, then values
        const int st = n % G::kRawStages, slot = n % G::kSlots;
        if (!wait(G::bRawFull + st, n / G::kRawStages)) break;
        if (!wait(G::bKvEmpty + slot, n / G::kSlots + 1)) break;
        const uint8_t* raw = smem + G::kRawOff + st * G::kRawBytes;
        uint8_t* dst = smem + G::kSlotOff + slot * G::kSlotBytes;
#pragma unroll
        for (int pass = 0; pass < K / 32; ++pass) {
          // lane j of a token's four: words j of all its blocks
          const int tok = w * (K / 4) + pass * 8 + (lane >> 2);
          const uint8_t* pg = raw + (tok / kPage) * G::kHalfPage;
          const int t = tok & (kPage - 1);
          uint32_t x[NB];
          __half2 d[NB];
          if (half == 0) {
            uint32_t sc[NB / 2];
            load_words<NB>(pg + t * F::kRow + j * 4 * NB, x);
            load_words<NB / 2>(pg + F::kKeyScale + t * 2 * NB, sc);
#pragma unroll
            for (int b = 0; b < NB; ++b)
              d[b] = b & 1 ? __high2half2(u32_as_h2(sc[b / 2])) : __low2half2(u32_as_h2(sc[b / 2]));
          } else {
            uint32_t y[NB];   // value words 2j and 2j + 1 of all blocks
            load_words<NB>(pg + t * F::kRow + ((2 * j) ^ value_swizzle<D>(t)) * 2 * NB, y);
            // slots behind the sequence and of pages that were not brought hold anything
            const bool live = base + tok < len && base + tok >= low;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              x[b] = prmt(y[b / 2], y[NB / 2 + b / 2], b & 1 ? 0x7632u : 0x5410u);
              const __half s = *reinterpret_cast<const __half*>(pg + 32 * D + (b * kPage + tile_perm(t)) * 2);
              d[b] = __half2half2(live ? s : __ushort_as_half(0));
            }
          }
          // odd tokens write their blocks in swapped pairs, so that the 8
          // lanes of a store phase cover all banks
          if (t & 1) {
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
              const uint32_t tx = x[b];
              x[b] = x[b + 1], x[b + 1] = tx;
              const __half2 td = d[b];
              d[b] = d[b + 1], d[b + 1] = td;
            }
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const int blk = b ^ (t & 1);
            const int piece = 4 * (blk & 1) + j;   // 16-byte piece of the 128-byte row
            *reinterpret_cast<uint4*>(dst + (b >> 1) * K * 128 + tok * 128 + ((piece ^ (tok & 7)) << 4)) =
                dequant_key8(x[b], d[b], minus_72(d[b]));
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(BAR(G::bRawEmpty + st));
          mbar_arrive(BAR(G::bKvFull + slot));
        }
        base += half * K;
      }
    }
    if (!ok) failed(8u);
  } else {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int i = (warp - kSoftmaxWarp0) / 4, q = warp & 3;   // row tile, lane quarter
    const int my_row = 32 * q + lane;
    const uint32_t tm = tmem + ((uint32_t)(32 * q) << 16);
    const uint32_t ts = tm + G::kS + i * K, to = tm + G::kO + i * D;
    uint32_t done = 0, joins = 0;
    const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
    // Queries of a piece's row tile to shared memory, lanes together on a row,
    // 16 bytes each: copied asynchronously, then brought to fp16's range where
    // they lie. Short loops: 16 rows' loads and normalizations unrolled were
    // fetched from beyond the instruction cache for every item (7 us).
    constexpr int LPR = D / 8, RPI = 32 / LPR, NQ = 32 / RPI;
    auto load_q = [&](const Work& x) {
      const int c = lane % LPR, r0 = 32 * q + lane / LPR;
      const uint32_t q_tile = (uint32_t)(G::kQOff + i * G::kQTileBytes + (c / 8) * 128 * 128);
      auto at = [&](int r) { return q_tile + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + (size_t)x.first * p.q_token +
                            (size_t)(x.head * p.group) * p.q_head + 8 * c;
#pragma unroll 2
      for (int k = 0; k < NQ; ++k) {
        const int r = r0 + k * RPI, row = x.row0 + i * 128 + r, tok = p.by_group(row);
        const bool have = tok < x.n;
        cp_async16(sbase + at(r), have ? src + (size_t)tok * p.q_token + (size_t)(row - tok * p.group) * p.q_head : src,
                   have);
      }
      cp_async_wait_all();
      const float fac0 = fmaxf(fabsf(p.scale_log2), 1e-30f);   // -inf * fac stays -inf
      auto in_place = [&](auto bf16) {
        constexpr int BATCH = 4;
#pragma unroll 1
        for (int k0 = 0; k0 < NQ; k0 += BATCH) {
          uint4 v[BATCH];
          float fac[BATCH];
#pragma unroll
          for (int k = 0; k < BATCH; ++k) v[k] = *reinterpret_cast<const uint4*>(smem + at(r0 + (k0 + k) * RPI));
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            fac[k] = fac0;
            normalize_query8<LPR>(v[k], bf16(), sign, fac[k]);
          }
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            *reinterpret_cast<uint4*>(smem + at(r0 + (k0 + k) * RPI)) = v[k];
            if (c == 0) factors[i * 128 + r0 + (k0 + k) * RPI] = fac[k];
          }
        }
      };
      if (p.bf16)
        in_place(std::true_type());
      else if (sign < 0.0f)
        in_place(std::false_type());
      else
        factors[i * 128 + my_row] = fac0;
      fence_proxy_async_shared();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(G::bQ + i));
    };
    // 32 columns of an output row
    auto put32 = [&](size_t at, const float* x, float scale) {
      uint32_t e[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const float a = x[2 * y] * scale, b = x[2 * y + 1] * scale;
        if (p.bf16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
          e[y] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          e[y] = h2_as_u32(__floats2half2_rn(a, b));
        }
      }
      uint16_t* to_row = static_cast<uint16_t*>(p.out) + at;
      if (p.wide_out) {   // whole 32-byte sectors
#pragma unroll
        for (int y = 0; y < 16; y += 8)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to_row + 2 * y), "r"(e[y]),
                       "r"(e[y + 1]), "r"(e[y + 2]), "r"(e[y + 3]), "r"(e[y + 4]), "r"(e[y + 5]), "r"(e[y + 6]),
                       "r"(e[y + 7])
                       : "memory");
      } else {
#pragma unroll
        for (int y = 0; y < 16; y += 4)
          *reinterpret_cast<uint4*>(to_row + 2 * y) = make_uint4(e[y], e[y + 1], e[y + 2], e[y + 3]);
      }
    };

    Work x = next_piece();
    if (ok && x.tiles > 0 && i < x.row_tiles) load_q(x);
    while (ok && x.tiles > 0) {
      const bool active = i < x.row_tiles;
      const int row = x.row0 + i * 128 + my_row, tok = p.by_group(row);
      const bool live = active && tok < x.n;
      float m = -INFINITY, l = 0.0f;
      Work nx;
      if (active) {
        const float f = factors[i * 128 + my_row];
        // slots seen, from the piece's first token on
        int lo = 0, hi = 0x7fffffff;
        if (live) {
          hi = (p.causal ? min(x.len, x.past + tok + 1) : x.len) - x.tile0 * K;
          lo = (p.window > 0 ? max(0, x.past + tok + 1 - p.window) : 0) - x.tile0 * K;
        }
        for (int j = 0; j < x.tiles; ++j, ++done, lo -= K, hi -= K) {
          if (!wait(G::bS + i, done)) break;
          tc_fence_after();
          const bool edge = __any_sync(0xffffffffu, hi < K || lo > 0);
          // Half a row at a time: P goes out in two halves, so that the first
          // one's MMAs run while the second one's exponentials are taken. The
          // exponentials are taken against the maximum known so far, while
          // the half's own is found beside them: only where that is more than
          // 2^kOver above the reference (at the start, and then rarely) are
          // they taken again. Short loops stay in the instruction cache.
#pragma unroll 1
          for (int h = 0; ok && h < 2; ++h) {
            constexpr int H = K / 2;
            uint32_t pk[H / 2];
            float sum[4];
#pragma unroll 1
            for (bool again = false;; again = true) {
              float x[H];
#pragma unroll
              for (int c2 = 0; c2 < H; c2 += 32)
                tmem_ld_x32(ts + h * H + c2, reinterpret_cast<uint32_t*>(x) + c2);
              tc_wait_ld();
              if (edge) {
                const int first = lo - h * H, last = hi - h * H;
#pragma unroll
                for (int k = 0; k < H; ++k) x[k] = k < last && k >= first ? x[k] : -INFINITY;
              }
              const float off = m == -INFINITY ? 0.0f : -m;
              float top[4] = {x[0], x[1], x[2], x[3]};
              sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
#pragma unroll
              for (int k = 0; k < H; k += 2) {
                float a = x[k], b = x[k + 1];
                if (k >= 4) top[k / 2 & 3] = max3(top[k / 2 & 3], a, b);
                fma_f32x2(a, b, f, off);
                a = exp2_approx(a);
                b = exp2_approx(b);
                add_f32x2(sum[k & 2], sum[(k & 2) + 1], a, b);
                pk[k / 2] = h2_as_u32(__floats2half2_rn(a, b));
              }
              const float mt = fmaxf(max3(top[0], top[1], top[2]), top[3]) * f;
              if (again || !__any_sync(0xffffffffu, mt > m + kOver || (m == -INFINITY && mt > m))) break;
              const float m2 = fmaxf(m, mt - kRaise);
              const float a = m == m2 ? 1.0f : exp2_approx(m - m2);
              m = m2;
              l *= a;
              if (j == 0 && h == 0) continue;
              // O so far: the MMAs of the half before this one. (Barriers per
              // half: the one before that is done, and its completion is not
              // mistaken for this one's.)
              if (!wait(G::bO + 2 * (h ^ 1) + i, h ? done : done - 1)) break;
              tc_fence_after();
#pragma unroll 1
              for (int c2 = 0; c2 < D; c2 += 32) {
                uint32_t o[32];
                tmem_ld_x32(to + c2, o);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
                tmem_st_x32(to + c2, o);
              }
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (H == 64)
              tmem_st_x32(ts + h * H / 2, pk);
            else
              tmem_st_x16(ts + h * H / 2, pk);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            // a barrier per half: warps run apart
            if (lane == 0) mbar_arrive(BAR(G::bP + 2 * h + i));
          }
        }
      }
      // the next piece's queries go to shared memory now that this one's last
      // scores are there, so that its first MMAs run during the epilogue
      nx = next_piece();
      if (ok && nx.tiles > 0 && i < nx.row_tiles) load_q(nx);
      if (active) {
        if (ok) wait(G::bO + 2 + i, done - 1);
        tc_fence_after();
      }
      if (!ok) break;
      const size_t out_at = live ? (size_t)(x.first + tok) * p.o_token +
                                       (size_t)(x.head * p.group + row - tok * p.group) * p.o_head
                                 : 0;
      auto put_lse = [&](float mm, float ll) {
        if (p.lse)
          p.lse[(size_t)(x.first + tok) * p.q_heads + x.head * p.group + row - tok * p.group] =
              ll > 0.0f ? (mm + log2f(ll)) * kLn2 : ll == 0.0f ? -INFINITY : ll;
      };
      if (x.kind == kWhole) {
        if (active) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
          for (int c2 = 0; c2 < D; c2 += 32) {   // TMEM loads take the whole warp
            float o[32];
            tmem_ld_x32(to + c2, reinterpret_cast<uint32_t*>(o));
            tc_wait_ld();
            if (live) put32(out_at + c2, o, inv);
          }
          if (live) put_lse(m, l);
        }
      } else {
        // a cut item: this CTA's part to its slot of the workspace
        const int r = i * 128 + my_row;
        if (active) {
          float* to_part = p.part + ((size_t)blockIdx.x * 2 + (x.kind == kTail ? 0 : 1)) * G::kPartFloats;
#pragma unroll 1
          for (int c2 = 0; c2 < D; c2 += 32) {
            uint32_t o[32];
            tmem_ld_x32(to + c2, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) to_part[(c2 + k) * G::kRows + r] = __uint_as_float(o[k]);
          }
          to_part[D * G::kRows + r] = m;
          to_part[(D + 1) * G::kRows + r] = l;
        }
        __threadfence();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(G::bParts));
        if (warp == kSoftmaxWarp0) {
          if (!wait(G::bParts, joins)) break;
          if (lane == 0) {
            __threadfence();
            const bool last = atom_add_acq_rel_gpu(p.counters + x.c_first, 1u) == (unsigned)(x.c_last - x.c_first);
            if (last) p.counters[x.c_first] = 0;
            misc[1] = last;
            mbar_arrive(BAR(G::bLast));
          }
          __syncwarp();
        }
        if (!wait(G::bLast, joins++)) break;
        if (misc[1] && live) {
          __threadfence();
          const int n = x.c_last - x.c_first + 1;
          auto theirs = [&](int k) {
            return p.part + ((size_t)(x.c_first + k) * 2 + (k == 0 ? 1 : 0)) * G::kPartFloats;
          };
          float mm = -INFINITY, ll = 0.0f;
          for (int k = 0; k < n; ++k) mm = fmaxf(mm, __ldcg(theirs(k) + D * G::kRows + r));
          // a piece that saw nothing has m = -inf, l = 0 and o = 0
          auto share = [&](int k) {
            const float mk = __ldcg(theirs(k) + D * G::kRows + r);
            return mk == -INFINITY ? 1.0f : exp2_approx(mk - mm);
          };
          for (int k = 0; k < n; ++k) ll = fmaf(__ldcg(theirs(k) + (D + 1) * G::kRows + r), share(k), ll);
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll 1
          for (int c2 = 0; c2 < D; c2 += 32) {
            float o[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            int y = 0;
#pragma unroll 1
            for (; y + 1 < n; y += 2) {   // two parts' loads in flight
              const float a = share(y), b = share(y + 1);
              float u[32], v[32];
#pragma unroll
              for (int k = 0; k < 32; ++k) u[k] = __ldcg(theirs(y) + (c2 + k) * G::kRows + r);
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = __ldcg(theirs(y + 1) + (c2 + k) * G::kRows + r);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = fmaf(v[k], b, fmaf(u[k], a, o[k]));
            }
            if (y < n) {
              const float a = share(y);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = fmaf(__ldcg(theirs(y) + (c2 + k) * G::kRows + r), a, o[k]);
            }
            put32(out_at + c2, o, inv);
          }
          put_lse(mm, ll);
        }
      }
      x = nx;
    }
    if (!ok) failed(16u);
  }
  if (bad) atomicOr(p.error, kErrIndex);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv4
}  // namespace busfill
