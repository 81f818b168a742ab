// The 4-bit K/V cache on the device: where a page keeps its codes and scales
// (include/busfill.h gives the format), and how a kernel finds the page of a
// slot and the sequence of a row without following an index out of range.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "host.h"
#include "ptx.cuh"

namespace busfill {
namespace kv4 {

constexpr int kPage = 64;            // tokens of one head in a page
constexpr float kMaxScale = 896.0f;  // largest |d|: 72 d stays below 65504

template <int D>
struct Fmt {
  static_assert(D == 64 || D == 128 || D == 256, "head dimension");
  static constexpr int kBlocks = D / 32;     // blocks (scales) of a token
  static constexpr int kRow = D / 2;         // bytes of a token's codes
  static constexpr int kKeyScale = 32 * D;   // offsets in a page
  static constexpr int kValue = 36 * D;
  static constexpr int kValueScale = 68 * D;
  static constexpr int kPageBytes = 72 * D;
};

// The 16-bit value words of a token are exchanged by this XOR on their group
// index c (a group: kBlocks words), so that the tokens 0,3,4,7 (and 1,2,5,6)
// that the lanes of one load read lie on different shared-memory banks.
template <int D>
__host__ __device__ __forceinline__ int value_swizzle(int t) {
  return D == 128 ? 4 * ((t >> 2) & 1) : D == 256 ? 2 * ((t >> 1) & 3) : 0;
}
// Matrix row r of an 8-token tile holds this token (its own inverse), and a
// token's value scale sits in this column: 0,1,3,2,4,5,7,6.
__host__ __device__ __forceinline__ int tile_perm(int t) { return t ^ ((t >> 1) & 1); }

// n / d for 0 <= n < 2^31 by a multiplication (set up on the host by divide_by)
struct Divisor {
  unsigned mul, shift;
  __device__ __forceinline__ int operator()(int n) const {
    return (int)((__umulhi((unsigned)n, mul) + (unsigned)n) >> shift);
  }
};
inline Divisor divide_by(unsigned d) {
  unsigned shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {(unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}

struct View {
  uint8_t* pages;
  const int* table;
  const int* kv_len;
  int num_pages, table_cols, batch, heads;
};

// Cached tokens of sequence b, cut to what its table row can hold.
__device__ __forceinline__ int cached(const View& c, int b, bool& bad) {
  const int n = c.kv_len[b];
  if (n < 0) {
    bad = true;
    return 0;
  }
  if (n > c.table_cols * kPage) {
    bad = true;
    return c.table_cols * kPage;
  }
  return n;
}

// Page `i` of sequence b (page 0 where the table's entry is out of range).
__device__ __forceinline__ int page_of(const View& c, const int* table, int cols, int b, int i, bool& bad) {
  const int pg = table[(size_t)b * cols + i];
  if ((unsigned)pg >= (unsigned)c.num_pages) {
    bad = true;
    return 0;
  }
  return pg;
}

// Rows of sequence b in the step's tensors: [first, first + n), inside [0, tokens].
__device__ __forceinline__ void rows_of(const int* q_start, int b, int tokens, int& first, int& n, bool& bad) {
  if (!q_start) {
    first = b;
    n = 1;
    return;
  }
  first = q_start[b];
  const int end = q_start[b + 1];
  if (first < 0 || end < first || end > tokens) {
    bad = true;
    first = 0;
    n = 0;
    return;
  }
  n = end - first;
}

// The sequence whose rows may include `row`: the last one that starts at or
// before it (-1: none). The warp's 32 lanes search together, 32 starts a load.
__device__ __forceinline__ int sequence_of(const int* q_start, int batch, int row, int lane) {
  if (!q_start) return row < batch ? row : -1;
  int base = 0;
  if (batch > 32) {
    const int i = 32 * lane;
    const int c = __popc(__ballot_sync(0xffffffffu, i < batch && q_start[i < batch ? i : 0] <= row));
    if (c == 0) return -1;
    base = 32 * (c - 1);
  }
  const int i = base + lane;
  const int c = __popc(__ballot_sync(0xffffffffu, i < batch && q_start[i < batch ? i : 0] <= row));
  return base + c - 1;
}

// fp32 of a 16-bit element of either type, and back (one rounding)
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(__half& y, float x) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_float(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }

// The eight 16-bit elements of a 16-byte piece.
template <typename T>
__device__ __forceinline__ void to_floats(const uint4& v, float* x) {
  alignas(16) T e[8];
  *reinterpret_cast<uint4*>(e) = v;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float(e[i]);
}

// 16 bytes to shared memory; zeros unless `have`
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// (a, b) = (a, b) * s + t, (a, b) * s and (a, b) += t as packed fp32 pairs (sm_100)
__device__ __forceinline__ void fma_f32x2(float& a, float& b, float s, float t) {
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %2};\n\t"
      "mov.b64 z, {%3, %3};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(s), "f"(t));
}
__device__ __forceinline__ void mul_f32x2(float& a, float& b, float s) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %2};\n\t"
      "mul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(s));
}
__device__ __forceinline__ void add_f32x2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}

__device__ __forceinline__ void fma_f32x2(float& a, float& b, float s0, float s1, float t0, float t1) {   // pairwise
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "mov.b64 z, {%4, %5};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(s0), "f"(s1), "f"(t0), "f"(t1));
}

// N consecutive 32-bit words, aligned to their size (16 bytes at most), by the widest loads.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

// Two fp16 values (c - 8) d of the codes that `bits` holds at bits 4-7 of its
// halves: 0x5400 | code << 4 is the fp16 number 64 + c, and with 72 d exact
// (d has 7 significant bits) one fused multiply-add gives the exact product.
__device__ __forceinline__ uint32_t dequant2(uint32_t bits, __half2 d, __half2 minus72d) {
  return h2_as_u32(__hfma2(u32_as_h2(lop3_and_or(bits, 0x00f000f0u, 0x54005400u)), d, minus72d));
}
__device__ __forceinline__ __half2 minus_72(__half2 d) { return __hmul2(d, __float2half2_rn(-72.0f)); }

// The eight fp16 values of a key word (nibble i of the low half: channel 2i,
// of the high half: 2i + 1), in channel order.
__device__ __forceinline__ uint4 dequant_key8(uint32_t w, __half2 d, __half2 m) {
  return make_uint4(dequant2(w << 4, d, m), dequant2(w, d, m), dequant2(w >> 4, d, m), dequant2(w >> 8, d, m));
}

}  // namespace kv4
}  // namespace busfill
