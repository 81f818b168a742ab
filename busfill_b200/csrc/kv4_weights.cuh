// The attention weight that many query rows give every cached token, on
// tcgen05 (few rows: weights_kernel in kv4_attn.cuh):
//   weights[s] += sum over rows r of exp2(score[r,s] f[r] - lse2[r])
//
// The scores are computed transposed, S^T = K Q^T: tokens are the MMA's M rows,
// so a TMEM lane, and with it a thread, owns a token and adds up its row of
// S^T in registers; no reduction crosses threads. Half the MMAs of the
// attention itself (2 R L D flops) and one exp2 per score (16 a clock and SM).
// Measured, 3 prompts of 1000 tokens, 64 heads over 8 of 128: 82 us, where the
// exponentials alone are 27; the rest is the first keys and queries of a range
// (5 us) and the loaders, which 16 warps keep just ahead of the sums (8 warps,
// with the masks read from shared memory: 10 us more).
//
// An item is 128 TT tokens of one (sequence, head); its keys are dequantized
// once and stay while blocks of 128 query rows pass by. The blocks of all
// items are cut into equal ranges, one per CTA; a cut item's partial sums go
// through the workspace and the CTA that comes last adds them in the order of
// the ranges.
//
// Warps: 0 issues the MMAs and owns TMEM; 4-7 and 8-11 add up, thread = token;
// 12-27 bring keys and queries as fp16 operands.
#pragma once

#include "kv4_prompt.cuh"

namespace busfill {
namespace kv4 {
namespace wsum {

constexpr int kThreads = 896;
constexpr int kLoadWarps = 16, kLoadWarp0 = 12;

template <int D>
struct Geo {
  static constexpr int kTiles = D == 256 ? 1 : 2;          // 128-token tiles of an item
  static constexpr int kTokens = 128 * kTiles;
  static constexpr int kKeyBufs = D == 256 ? 1 : 2;
  static constexpr int kKeyTile = 128 * D * 2;
  static constexpr int kKeyBytes = kTiles * kKeyTile;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kStages = 2;                        // query blocks, each with its S^T in TMEM
  static constexpr int kKeyOff = 0, kQOff = kKeyBufs * kKeyBytes;
  static constexpr int kConstOff = kQOff + kStages * kQBytes;   // [factor, -lse2][row]
  static constexpr int kBarOff = kConstOff + kStages * 128 * 8;
  static constexpr int bKFull = 0, bKEmpty = bKFull + kKeyBufs, bQFull = bKEmpty + kKeyBufs,
                       bQEmpty = bQFull + kStages, bS = bQEmpty + kStages, bFinal = bS + kStages, kBars = bFinal + 1;
  static constexpr int kMiscOff = kBarOff + kBars * 8;
  static constexpr int kPreOff = (kMiscOff + 8 + 15) / 16 * 16;
  static constexpr int kAlloc = kPreOff + (kMaxBatch + 1) * 4 + 1024;
  static_assert(kAlloc <= 232448, "dynamic shared memory");
};

struct Item {
  int b, head, t, tiles;    // tile t of the sequence's [tile0, tile0 + tiles)
  int tile0;
  int block0, blocks;       // query blocks that see it
  Span s;
};

template <int D>
__device__ __forceinline__ int tiles_of(const Span& s, int& tile0) {
  constexpr int T = Geo<D>::kTokens;
  tile0 = s.page0 * kPage / T;
  return s.pages > 0 ? (s.len + T - 1) / T - tile0 : 0;
}
template <int D>
__device__ __forceinline__ int blocks_of(const AttnParams& p, const Span& s, int t, int& block0) {
  constexpr int T = Geo<D>::kTokens;
  const int base = t * T, past = s.past;
  const int i0 = p.causal ? max(0, base - past) : 0;
  const int i1 = p.window > 0 ? min(s.n, base + T - 1 + p.window - past) : s.n;
  block0 = i0 * p.group / 128;
  return i1 > i0 ? (i1 * p.group + 127) / 128 - block0 : 0;
}

}  // namespace wsum

template <int D>
__global__ void __launch_bounds__(wsum::kThreads, 1) weights_prompt_kernel(const __grid_constant__ AttnParams p) {
  using G = wsum::Geo<D>;
  using F = Fmt<D>;
  using wsum::Item;
  constexpr int NB = F::kBlocks, TT = G::kTiles;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  const uint32_t sbase = smem_u32(smem);
  auto BAR = [&](int i) { return sbase + G::kBarOff + 8u * (uint32_t)i; };
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + G::kMiscOff);
  int* pre = reinterpret_cast<int*>(smem + G::kPreOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = p.c.batch;

  if (warp == 0) {
    tmem_alloc(sbase + G::kMiscOff, 512);
    tmem_relinquish();
  } else if (warp == 1) {
    for (int i = lane; i < G::kBars; i += 32) {
      const bool load = i < G::bKEmpty || (i >= G::bQFull && i < G::bQEmpty);
      // a query stage is free when its MMAs are done and every adding warp has read S^T
      mbar_init(BAR(i), load ? wsum::kLoadWarps : i >= G::bQEmpty && i < G::bS ? 1 + 4 * TT : 1);
    }
    fence_mbar_init();
  }
  pdl_wait_prerequisites();
  pdl_launch_dependents();
  bool bad = false;
  for (int b = warp; b < batch; b += wsum::kThreads / 32) {
    const Span s = span_of(p, b, bad);
    int t0, x;
    const int tiles = wsum::tiles_of<D>(s, t0);
    long long n = 0;
    for (int t = lane; t < tiles; t += 32) n += wsum::blocks_of<D>(p, s, t0 + t, x);
    const long long cost = warp_total(n) * p.c.heads;
    if (lane == 0) pre[b + 1] = counted(cost);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) running_sum(pre, batch, lane, bad, *p.refused != 0);
  __syncthreads();
  const uint32_t tmem = misc[0];
  const int T = pre[batch];
  const long long ctas = min((int)gridDim.x, T);
  const bool idle = (int)blockIdx.x >= ctas;
  const int u0 = idle ? 0 : (int)((long long)T * blockIdx.x / ctas);
  const int u1 = idle ? 0 : (int)((long long)T * (blockIdx.x + 1) / ctas);

  Item first{};
  int skip = 0;
  auto open = [&](Item& it, int b) {
    it.b = b;
    it.s = span_of(p, b, bad);
    it.tiles = wsum::tiles_of<D>(it.s, it.tile0);
  };
  if (u0 < u1) {
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (pre[mid] <= u0 ? lo : hi) = mid;
    }
    open(first, lo);
    const int per_head = (pre[lo + 1] - pre[lo]) / p.c.heads;
    int r = u0 - pre[lo];
    first.head = r / per_head;
    r -= first.head * per_head;
    for (int t0 = 0;; t0 += 32) {
      int x0;
      const int n = t0 + lane < first.tiles ? wsum::blocks_of<D>(p, first.s, first.tile0 + t0 + lane, x0) : 0;
      int x = n;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, m);
        if (lane >= m) x += y;
      }
      const unsigned over = __ballot_sync(0xffffffffu, x > r);
      if (over) {
        const int k = __ffs(over) - 1;
        first.t = t0 + k;
        skip = r - __shfl_sync(0xffffffffu, x - n, k);
        break;
      }
      r -= __shfl_sync(0xffffffffu, x, 31);
    }
    first.blocks = wsum::blocks_of<D>(p, first.s, first.tile0 + first.t, first.block0);
  }
  auto for_pieces = [&](auto f) {
    Item it = first;
    int from = skip;
    for (int u = u0; u < u1;) {
      const int n = min(it.blocks - from, u1 - u);
      if (!f(it, from, n, u)) return;
      u += n;
      from = 0;
      if (u >= u1) return;
      do {   // the next tile that some row sees
        if (++it.t == it.tiles) {
          it.t = 0;
          if (++it.head == p.c.heads) {
            it.head = 0;
            int b = it.b;
            do ++b;
            while (b < batch && pre[b + 1] == pre[b]);
            if (b >= batch) return;
            open(it, b);
          }
        }
        it.blocks = wsum::blocks_of<D>(p, it.s, it.tile0 + it.t, it.block0);
      } while (it.blocks == 0);
    }
  };
  bool ok = true;
  auto wait = [&](int bar, uint32_t phase) -> bool {
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(BAR(bar), phase & 1));
    return ok;
  };

  if (warp == 0) {
    // ---------------- MMA ----------------
    constexpr uint32_t kIdesc = make_idesc_f16_f32(128, 128);
    // descriptors are made once and stepped by their address field
    const uint64_t k_desc = make_sdesc_sw128(sbase + G::kKeyOff), q_desc = make_sdesc_sw128(sbase + G::kQOff);
    uint32_t item = 0, n = 0;
    for_pieces([&](const Item&, int, int blocks, int) {
      const int kb = item % G::kKeyBufs;
      if (!wait(G::bKFull + kb, item / G::kKeyBufs)) return false;
      for (int j = 0; j < blocks; ++j, ++n) {
        const int st = n % G::kStages;
        // the loaders refill a stage only after its S^T has been read
        if (!wait(G::bQFull + st, n / G::kStages)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b = q_desc + (uint32_t)(st * G::kQBytes / 16);
#pragma unroll
          for (int i = 0; i < TT; ++i) {
            const uint64_t a = k_desc + (uint32_t)((kb * G::kKeyBytes + i * G::kKeyTile) / 16);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_f16_ss(tmem + (st * TT + i) * 128, a + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16,
                         b + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16, kIdesc, k > 0);
          }
          tc_commit(BAR(G::bS + st));
          tc_commit(BAR(G::bQEmpty + st));
          if (j + 1 == blocks) tc_commit(BAR(G::bKEmpty + kb));
        }
        __syncwarp();
      }
      ++item;
      return true;
    });
    if (!ok && lane == 0) atomicOr(p.error, 4u);
    ok = true;
    tc_fence_after();
    if (elect_one()) tc_commit(BAR(G::bFinal));
    __syncwarp();
    if (!wait(G::bFinal, 0) && lane == 0) atomicOr(p.error, 32u);
  } else if (warp >= wsum::kLoadWarp0) {
    // ---------------- keys and queries ----------------
    const int w = warp - wsum::kLoadWarp0, j = lane & 3;
    const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
    uint32_t item = 0, n = 0;
    for_pieces([&](const Item& it, int from, int blocks, int) {
      const int kb = item % G::kKeyBufs;
      if (!wait(G::bKEmpty + kb, item / G::kKeyBufs + 1)) return false;
      uint8_t* dst = smem + G::kKeyOff + kb * G::kKeyBytes;
      const int base = (it.tile0 + it.t) * G::kTokens;
#pragma unroll
      for (int pass = 0; pass < G::kTokens / (8 * wsum::kLoadWarps); ++pass) {
        const int tok = (pass * wsum::kLoadWarps + w) * 8 + (lane >> 2);
        uint32_t x[NB], sc[NB / 2];
#pragma unroll
        for (int b = 0; b < NB; ++b) x[b] = 0;
#pragma unroll
        for (int b = 0; b < NB / 2; ++b) sc[b] = 0;
        const int t = tok & (kPage - 1);
        if (base + tok < it.s.len && base + tok >= it.s.page0 * kPage) {   // not before every row's window
          const int pg = page_of(p.c, p.c.table, p.c.table_cols, it.b, (base + tok) / kPage, bad);
          const uint8_t* src = p.c.pages + ((size_t)pg * p.c.heads + it.head) * F::kPageBytes;
          load_words<NB>(src + t * F::kRow + j * 4 * NB, x);
          load_words<NB / 2>(src + F::kKeyScale + t * 2 * NB, sc);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const __half2 d = b & 1 ? __high2half2(u32_as_h2(sc[b / 2])) : __low2half2(u32_as_h2(sc[b / 2]));
          const int piece = 4 * (b & 1) + j, r = tok & 127;
          *reinterpret_cast<uint4*>(dst + (tok >> 7) * G::kKeyTile + (b >> 1) * 128 * 128 + r * 128 +
                                    ((piece ^ (r & 7)) << 4)) = dequant_key8(x[b], d, minus_72(d));
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(G::bKFull + kb));
      ++item;
      // A block's rows are on their way while its stage is still in use; lane r
      // holds the constants of the warp's row r.
      constexpr int LPR = D / 8, RPI = 32 / LPR, NR = 128 / wsum::kLoadWarps, NI = NR / RPI;
      const int c = lane % LPR;
      uint4 v[NI];
      float lse;
      auto fetch = [&](int blk) {
        const int row0 = (it.block0 + from + blk) * 128 + w * NR;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const int row = row0 + k * RPI + lane / LPR, tok = p.by_group(row);
          v[k] = make_uint4(0, 0, 0, 0);
          if (tok < it.s.n)
            v[k] = __ldg(reinterpret_cast<const uint4*>(
                static_cast<const uint16_t*>(p.q) + (size_t)(it.s.first + tok) * p.q_token +
                (size_t)(it.head * p.group + row - tok * p.group) * p.q_head + 8 * c));
        }
        const int row = row0 + lane % NR, tok = p.by_group(row);
        lse = -INFINITY;   // rows that are not there or see nothing give no weight
        if (tok < it.s.n)
          lse = p.lse[(size_t)(it.s.first + tok) * p.q_heads + it.head * p.group + row - tok * p.group];
      };
      fetch(0);
      for (int blk = 0; blk < blocks; ++blk, ++n) {
        const int st = n % G::kStages;
        if (!wait(G::bQEmpty + st, n / G::kStages + 1)) return false;
        float* consts = reinterpret_cast<float*>(smem + G::kConstOff) + st * 256 + w * NR;
        uint8_t* q_block = smem + G::kQOff + st * G::kQBytes + (c / 8) * 128 * 128;
        const float fac0 = fmaxf(fabsf(p.scale_log2), 1e-30f);   // -inf * fac stays -inf
        auto store = [&](auto bf16) {
          float fac[NI];
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            fac[k] = fac0;
            normalize_query8<LPR>(v[k], bf16(), sign, fac[k]);
          }
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            const int r = k * RPI + lane / LPR, rr = w * NR + r;
            *reinterpret_cast<uint4*>(q_block + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[k];
            if (c == 0) consts[r] = fac[k];
          }
        };
        if (p.bf16)
          store(std::true_type());
        else
          store(std::false_type());
        if (lane < NR) consts[128 + lane] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(G::bQFull + st));
        if (blk + 1 < blocks) fetch(blk + 1);
      }
      return true;
    });
    if (!ok && lane == 0) atomicOr(p.error, 8u);
  } else if (warp >= 4 && warp < 4 + 4 * TT) {
    // ---------------- add up ----------------
    // A warp whose wait ran out goes on through its pieces without waiting, so
    // that the named barriers (no timeout) always fill.
    const int i = (warp - 4) / 4, q = warp & 3;
    const int mine = i * 128 + 32 * q + lane;   // token of the item
    const uint32_t tm = tmem + ((uint32_t)(32 * q) << 16);
    float* my_part = p.part + (size_t)blockIdx.x * 2 * G::kTokens;
    uint32_t n = 0;
    for_pieces([&](const Item& it, int from, int blocks, int u) {
      const int slot = (it.tile0 + it.t) * G::kTokens + mine;
      // the rows that see the thread's token: [row_a, row_z)
      const long long at = slot - it.s.past;   // the row that stands at it
      const int row_a = p.causal ? (int)max(0ll, min(at, (long long)it.s.n)) * p.group : 0;
      const int row_z = slot >= it.s.len ? 0
                        : p.window > 0   ? (int)max(0ll, min(at + p.window, (long long)it.s.n)) * p.group
                                         : it.s.n * p.group;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int blk = 0; blk < blocks && ok; ++blk, ++n) {
        const int st = n % G::kStages;
        if (!wait(G::bS + st, n / G::kStages)) break;
        tc_fence_after();
        const float* consts = reinterpret_cast<const float*>(smem + G::kConstOff) + st * 256;
        const int row0 = (it.block0 + from + blk) * 128, a = row_a - row0, z = row_z - row0;
        const bool whole = __all_sync(0xffffffffu, a <= 0 && z >= min(128, it.s.n * p.group - row0));
        const bool none = __all_sync(0xffffffffu, z <= 0 || a >= 128);
#pragma unroll 1
        for (int c = none ? 128 : 0; c < 128; c += 32) {
          float s[32];
          tmem_ld_x32(tm + (st * TT + i) * 128 + c, reinterpret_cast<uint32_t*>(s));
          tc_wait_ld();
          if (!whole) {
#pragma unroll
            for (int k = 0; k < 32; ++k) s[k] = c + k >= a && c + k < z ? s[k] : -INFINITY;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 f = *reinterpret_cast<const float4*>(consts + c + k),
                         t = *reinterpret_cast<const float4*>(consts + 128 + c + k);
            fma_f32x2(s[k], s[k + 1], f.x, f.y, t.x, t.y);
            fma_f32x2(s[k + 2], s[k + 3], f.z, f.w, t.z, t.w);
            add_f32x2(sum[0], sum[1], exp2_approx(s[k]), exp2_approx(s[k + 1]));
            add_f32x2(sum[2], sum[3], exp2_approx(s[k + 2]), exp2_approx(s[k + 3]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(G::bQEmpty + st));
      }
      float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
      const bool live = ok && slot < it.s.len;
      float* to = p.weights + ((size_t)it.b * p.c.heads + it.head) * p.weights_cols + slot;
      if (from == 0 && blocks == it.blocks) {
        if (live) *to += total;
        return true;
      }
      my_part[(size_t)(from > 0 ? 0 : 1) * G::kTokens + mine] = total;
      __threadfence();
      named_bar_sync(1, 128 * TT);
      const int item0 = u - from, end = item0 + it.blocks;
      const int c_first = (int)((((long long)item0 + 1) * ctas - 1) / T), c_last = (int)(((long long)end * ctas - 1) / T);
      if (threadIdx.x == 128)
        misc[1] = atom_add_acq_rel_gpu(p.counters + c_first, 1u) == (unsigned)(c_last - c_first) ? 1u : 0u;
      named_bar_sync(1, 128 * TT);
      if (misc[1]) {
        __threadfence();
        total = 0.0f;
        for (int k = c_first; k <= c_last; ++k)
          total += __ldcg(p.part + ((size_t)k * 2 + (k == c_first ? 1 : 0)) * G::kTokens + mine);
        if (live) *to += total;
        if (threadIdx.x == 128) p.counters[c_first] = 0;
      }
      named_bar_sync(1, 128 * TT);
      return true;
    });
    if (!ok && lane == 0) atomicOr(p.error, 16u);
  }
  if (bad) atomicOr(p.error, kErrIndex);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv4
}  // namespace busfill
