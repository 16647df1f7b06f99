// seq_pages.cuh -- how the kernels that read pages by TMA (K7, K8) bring a tile
// of keys into shared memory, and what they (and K5) do with codes and masked values.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "seq.cuh"

namespace attnb {

// The page numbers of a sequence, 32 at a time in the lanes of one warp: a tile
// then costs no read of the table that anything waits for.
struct PageWindow {
  int b = -1, first = 0;  // window of sequence b (selected blocks: of list b) from this slot on
  int page;               // this lane's slot
  // Number of the page at `slot` (the same for the whole warp; all lanes
  // call), num_pages, which lies outside the pool and reads as zeros, for slots
  // past `used` and for bad numbers.
  template <bool SEL>
  __device__ __forceinline__ int get(const SeqAttnArgs& a, const SeqPiece& w, int slot, int used) {
    const int of = SEL && a.sel_blocks ? w.v : w.b;
    if (of != b || slot < first || slot >= first + 32) {
      b = of;
      first = slot;
      const int mine = slot + (int)(threadIdx.x & 31);
      page = a.pages.num_pages;
      if (mine < used) {
        const int at = SEL ? piece_slot(a, w, mine) : mine;
        const int p = __ldg(a.seqs.table + w.b * a.seqs.table_stride + at);
        if (p >= 0 && p < a.pages.num_pages) page = p;
        else raise_index(a.index_status);
      }
    }
    const int p = __shfl_sync(0xffffffffu, page, slot - first);
    return slot < used ? p : a.pages.num_pages;
  }
  // The same of slots `slot` to `slot` + count - 1 (count <= 8) at once: lane i has that of
  // slot + (i & 7).
  template <bool SEL>
  __device__ __forceinline__ int get_eight(const SeqAttnArgs& a, const SeqPiece& w, int slot,
                                           int count, int used) {
    const int of = SEL && a.sel_blocks ? w.v : w.b;
    if (of != b || slot < first || slot + count > first + 32) b = -1;  // all of them in one window
    get<SEL>(a, w, slot, used);
    const int mine = slot + (int)(threadIdx.x & 7);
    const int p = __shfl_sync(0xffffffffu, page, mine - first);
    return mine < used ? p : a.pages.num_pages;
  }
};

// 128-byte rows with the TMA's 128-byte swizzle: byte offset of 16-byte unit u
// of row r (tile base 1024-byte aligned).
__device__ __forceinline__ uint32_t sw128(int r, int u) {
  return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4));
}

// 4-bit codes lie as they do in a page, vector after vector (Dh / 32 units of 16 bytes each), in
// such rows: byte offset of unit i.  Rows of their own for the vectors, of 64 bytes, are copied
// 4 us of 88 more slowly.  (Eight vectors' units are in different banks for Dh 64 and 128.)
__device__ __forceinline__ uint32_t i4_unit(int i) { return sw128(i >> 3, i & 7); }

// a * b + c of two pairs of f16.
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// 4-bit codes in f16.  Two codes masked out of a word are the subnormals
// code * 2^-24 (mask 000f000f) or 16 code * 2^-24 (00f000f0); with their factors r,
//     (code * 2^-24) * (r * 2^5) - r * 2^-16 = r * (code - 8) * 2^-19,
// exact: a multiple of 2^-19 below 2^-8, in one FMA of two.
constexpr uint32_t kI4Low = 0x000f000fu, kI4High = 0x00f000f0u;
constexpr float kI4Unit = 0x1p19f;  // what such values are to be multiplied by
// Against such small values queries are brought up to 2^14 (2^15 next to overflow): room
// below for sixteenths of them, and little left of the unit for the factors of scores, which
// stay finite for queries and keys up to 2^124.
constexpr float kI4Rows = 0x1p13f;  // (i4_row_scale has the exponent too)
struct I4Factors {
  uint32_t low, high, add;  // pairs of f16: r 2^5, r 2^1, -r 2^-16
};
// From two factors in bits 0-7 and 16-23.
__device__ __forceinline__ I4Factors i4_factors(uint32_t r) {
  const uint32_t x = (r & 0x00ff00ffu) | 0x64006400u;  // 1024 + r
  return {fma_f16x2(x, 0x50005000u, 0xf800f800u),       // 2^5, -2^15
          fma_f16x2(x, 0x40004000u, 0xe800e800u),       // 2^1, -2^11
          fma_f16x2(x, 0x81008100u, 0x24002400u)};      // -2^-16, 2^-6
}

// Four codes to two pairs of f16, exactly.
template <int T>
__device__ __forceinline__ void codes_to_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
  if constexpr (T == kE4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
  } else {
    // 1024 + (code + 128) has the shifted code as its last mantissa bits.
    const uint32_t x = four ^ 0x80808080u;
    const __half2 base = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&a), base);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&b), base);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    hi = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The power of two that brings a row whose largest magnitude is `top` to
// [1, 2), so that its values fit f16 with an error of at most 2^-25 of the
// largest; 1 for rows of zeros and rows that are not finite.
__device__ __forceinline__ float row_scale(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);  // top >= 0
  if (e == 0 || e == 255) return 1.f;
  return __uint_as_float((uint32_t)max(254 - e, 1) << 23);  // [2, 4) next to overflow
}

// kI4Rows times that, for queries over 4-bit codes.  At most 2^127, so that it stays finite: rows that are
// smaller than 2^-114 come out below 2^13, and as exactly, since bf16's values are multiples of
// 2^-133.
__device__ __forceinline__ float i4_row_scale(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);
  if (top == 0.f || e == 255) return kI4Rows;
  return __uint_as_float((uint32_t)min(max(254 - e, 1) + 13, 254) << 23);
}

// The larger one, or NaN where one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Values in masked places.  A product P . V with P = 0 for a masked key still
// takes an infinity or a NaN of V into the sum.  In the tiles that need a mask
// such values are therefore zeroed in shared memory and noted as the first key
// that holds one, by dimension and kind; the rows that do see that key get the
// value back at the end.  Kinds: 0 NaN, 1 +inf, 2 -inf.

// What row values become: `seen` keys are visible to the row.
__device__ __forceinline__ float poisoned(float x, const int* nan, const int* pos, const int* neg,
                                          int d, int seen) {
  const bool p = pos[d] < seen, n = neg[d] < seen;
  if (nan[d] < seen || (p && n)) return __int_as_float(0x7fffffff);
  if (p) return x + INFINITY;
  if (n) return x - INFINITY;
  return x;
}

}  // namespace attnb
