// kv_pages.cu -- K5: writing packed tokens into the pages of a KV cache, as they
// are or as 8-bit codes, and reading them back.
//
// A vector x of Dh values (one token, one KV head) is stored in e4m3 or int8 as
//     a = max |x|,   code = round(x * C / a),   scale = a / C    (C = 448 or 127)
// with ties to even, so the largest value is the largest code and the value
// read back is code * scale.  x * C / a is decided exactly: for 16-bit x the
// product has at most 20 bits and the fp32 quotient cannot land on a tie that
// the exact one is not on (the two differ by 2^-18 of it at least, half a unit
// in the last place of fp32 is 2^-24); for fp32 x the quotient is taken in 64
// bits, by the same argument (product 33 bits, distance 2^-42).  A vector
// of zeros has scale 0; one with an Inf or NaN has scale NaN and codes 0, so
// that it cannot be read back as something finite.
//
// Bound by memory: a token is read once and its codes written once.  A CTA takes
// some tokens that follow one another, all heads of K and V.  Where a token
// lives takes a search and three dependent reads, as long as hundreds of
// streamed bytes, so one thread per token finds the places of all of them first.
// Then a group of 8 to 32 lanes takes one vector, 8 elements a lane (one 16-byte
// read of a 16-bit row), so that the maximum is a few shuffles and no vector is
// read twice; rows that are not aligned for that are read element by element.
#include <algorithm>
#include <cmath>

#include "seq.cuh"
#include "seq_elem.cuh"
#include "runtime.h"

namespace attnb {
namespace {

constexpr int kThreads = 256;

// The sequence that packed token t belongs to: the last b with cu[b] <= t
// (clamped as in seq_rows), or -1 when its range does not hold t.
__device__ __forceinline__ int seq_of(const SeqTable& sq, int t, int& first, int& count) {
  int lo = 0, hi = sq.batch;  // cu[lo] <= t is kept true for lo > 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(sq.cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  seq_rows(sq.cu, lo, sq.total, first, count);
  return t >= first && t < first + count ? lo : -1;
}

// Place of packed token t in a [.., H, page, ..] pool for head 0, or -1.
__device__ __forceinline__ int64_t place_of(const SeqTable& sq, const KvPages& pg, int t,
                                            int* index_status) {
  int first, count;
  const int b = seq_of(sq, t, first, count);
  if (b < 0) return -1;
  const int64_t pos = (int64_t)__ldg(sq.lens + b) - count + (t - first);
  if (pos < 0 || pos >= ((int64_t)sq.max_pages << pg.page_shift)) {
    raise_index(index_status);
    return -1;
  }
  const int page = seq_page(sq, pg, b, (int)pos, index_status);
  if (page < 0) return -1;
  return (((int64_t)page * pg.H) << pg.page_shift) + (pos & ((1 << pg.page_shift) - 1));
}

template <int TX>
__device__ __forceinline__ float quotient(float x, float a, float top) {
  if constexpr (TX == kF32) {
    // Rounded to odd, so that the rounding to a code that follows sees on which
    // side of a tie the 64-bit quotient lies.
    const double q = (double)x * (double)top / (double)a;
    float f = (float)q;
    if ((double)f != q && (__float_as_uint(f) & 1u) == 0u) {
      const bool away = fabs((double)f) > fabs(q);
      f = __uint_as_float(__float_as_uint(f) + (away ? -1 : 1));
    }
    return f;
  }
  if (TX == kBF16 && a > 0x1p100f) {  // x * top stays finite
    x *= 0x1p-64f;
    a *= 0x1p-64f;
  }
  return x * top / a;
}

__device__ __forceinline__ uint32_t pack_codes(const float (&q)[4], elem_t<kE4M3>*) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint32_t pack_codes(const float (&q)[4], elem_t<kI8>*) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= ((uint32_t)__float2int_rn(q[i]) & 0xFFu) << (8 * i);
  return r;
}

constexpr int kMaxTokens = 32;  // per CTA

// Where the CTA's tokens [t0, t0 + n) live: the place of head 0, -1 for a place
// out of range and -2 for a row of no sequence.
__device__ __forceinline__ void find_places(const SeqTable& sq, const KvPages& pg, int t0, int n,
                                            int64_t* at, int* index_status) {
  if ((int)threadIdx.x < n) {
    int first, count;
    const int t = t0 + threadIdx.x;
    at[threadIdx.x] = seq_of(sq, t, first, count) < 0 ? -2 : place_of(sq, pg, t, index_status);
  }
  __syncthreads();
}

// 8 elements from d on, those past Dh as zeros.
template <class E>
__device__ __forceinline__ void load8(const E* p, int d, int Dh, bool vec, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (vec) {  // Dh is a multiple of 8
    if (d >= Dh) return;
    struct alignas(sizeof(E) * 8 >= 16 ? 16 : 8) Eight {
      E e[8];
    };
    const Eight f = *reinterpret_cast<const Eight*>(p + d);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(f.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < Dh) x[i] = to_float(p[d + i]);
  }
}
template <class E>
__device__ __forceinline__ void store8(E* p, int d, int Dh, bool vec, const float (&x)[8]) {
  if (vec) {
    if (d >= Dh) return;
    struct alignas(sizeof(E) * 8 >= 16 ? 16 : 8) Eight {
      E e[8];
    };
    Eight f;
#pragma unroll
    for (int i = 0; i < 8; ++i) from_float(x[i], f.e[i]);
    *reinterpret_cast<Eight*>(p + d) = f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < Dh) from_float(x[i], p[d + i]);
  }
}

// One vector per group of LANES lanes.
template <int TX, int TC, int LANES>
__global__ void __launch_bounds__(kThreads)
    append_kernel(const RowsView K, const RowsView V, const KvPages pg, const SeqTable sq,
                  const int tokens, const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = TC == kE4M3 || TC == kI8;
  __shared__ int64_t places[kMaxTokens];
  const int e = threadIdx.x % LANES, d = e * 8;
  const int Dh = pg.Dh, H2 = 2 * pg.H;
  grid_dep_wait();
  const int t0 = blockIdx.x * tokens, n = min(tokens, sq.total - t0);
  find_places(sq, pg, t0, n, places, index_status);
  // A group's lanes share their vector; the other groups of the warp may have left.
  const unsigned mask =
      LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
#pragma unroll 2
  for (int i = threadIdx.x / LANES; i < n * H2; i += kThreads / LANES) {
    const int tl = i / H2, kvh = i - tl * H2;
    const bool is_v = kvh >= pg.H;
    const int h = is_v ? kvh - pg.H : kvh;
    const RowsView& src = is_v ? V : K;
    const EX* p = static_cast<const EX*>(src.data) + (int64_t)(t0 + tl) * src.sT + (int64_t)h * src.sH;
    float x[8];
    load8(p, d, Dh, vec, x);
    const int64_t at0 = places[tl];
    if (at0 < 0) continue;
    const int64_t at = at0 + ((int64_t)h << pg.page_shift);
    EC* out = static_cast<EC*>(is_v ? pg.v : pg.k) + at * Dh;
    if constexpr (CODED) {
      constexpr float C = TC == kE4M3 ? 448.f : 127.f;
      float top = 0.f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(x[j]));
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
      bad = (__ballot_sync(mask, bad) & mask) != 0;
      if (e == 0)
        (is_v ? pg.v_scale : pg.k_scale)[at] = bad ? __int_as_float(0x7fffffff) : top / C;
      if (bad) top = 0.f;
      // x * (C / a) is off by less than 2^-22 of it: where 2^-22 up and down give
      // the same codes, those are the ones; else (next to a tie) the quotient
      // decides.  C / a overflows for tiny a, and is not used for large ones.
      const float inv = top > 0x1p-100f && top < 0x1p100f ? C / top : 0.f;
      uint32_t r2[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float up[4], down[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = x[4 * k + j] * inv;
          up[j] = q * (1.f + 0x1p-22f);
          down[j] = q * (1.f - 0x1p-22f);
        }
        r2[k] = pack_codes(up, out);
        if (r2[k] != pack_codes(down, out) || inv == 0.f) {
          float q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            q[j] = top > 0.f ? quotient<TX>(x[4 * k + j], top, C) : 0.f;
          r2[k] = pack_codes(q, out);
        }
      }
      const uint2 r = make_uint2(r2[0], r2[1]);
      if (vec) {
        if (d < Dh) *reinterpret_cast<uint2*>(out + d) = r;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d + j < Dh)
            reinterpret_cast<uint8_t*>(out)[d + j] = (uint8_t)((j < 4 ? r.x : r.y) >> (8 * (j & 3)));
      }
    } else {
      store8(out, d, Dh, vec, x);
    }
  }
}

template <int TX, int TC, int LANES>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const KvPages pg, const RowsView K, const RowsView V, const SeqTable sq,
                const int tokens, const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = TC == kE4M3 || TC == kI8;
  __shared__ int64_t places[kMaxTokens];
  const int d = threadIdx.x % LANES * 8;
  const int Dh = pg.Dh, H2 = 2 * pg.H;
  grid_dep_wait();
  const int t0 = blockIdx.x * tokens, n = min(tokens, sq.total - t0);
  find_places(sq, pg, t0, n, places, index_status);
#pragma unroll 2
  for (int i = threadIdx.x / LANES; i < n * H2; i += kThreads / LANES) {
    const int tl = i / H2, kvh = i - tl * H2;
    const bool is_v = kvh >= pg.H;
    const int h = is_v ? kvh - pg.H : kvh;
    const int64_t at0 = places[tl];
    if (at0 == -2) continue;  // a row of no sequence stays as it is
    const int64_t at = at0 + ((int64_t)h << pg.page_shift);
    float x[8];
    if (at0 >= 0) {
      load8(static_cast<const EC*>(is_v ? pg.v : pg.k) + at * Dh, d, Dh, vec, x);
      if constexpr (CODED) {
        const float scale = (is_v ? pg.v_scale : pg.k_scale)[at];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= scale;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    const RowsView& dst = is_v ? V : K;
    store8(static_cast<EX*>(dst.data) + (int64_t)(t0 + tl) * dst.sT + (int64_t)h * dst.sH, d, Dh,
           vec, x);
  }
}

bool vec_rows(const RowsView& r) {
  // 8 elements are read as 16 bytes (32-bit ones as two times 16).
  const int unit = 16 / elem_bytes(r.type);
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.sT % unit == 0 && r.sH % unit == 0 &&
         r.Dh % 8 == 0;
}
bool vec_pages(const KvPages& p) {
  const int b = std::min(16, 8 * elem_bytes(p.type));
  return reinterpret_cast<uintptr_t>(p.k) % b == 0 && reinterpret_cast<uintptr_t>(p.v) % b == 0 &&
         p.Dh % 8 == 0;
}

// f(type of the rows, type of the pages, lanes per vector).
template <class F>
void dispatch(const RowsView& K, const KvPages& pg, F&& f) {
  auto sizes = [&](auto tx, auto tc) {
    using std::integral_constant;
    if (pg.Dh <= 64) f(tx, tc, integral_constant<int, 8>{});
    else if (pg.Dh <= 128) f(tx, tc, integral_constant<int, 16>{});
    else f(tx, tc, integral_constant<int, 32>{});
  };
  with_value_type(K.type, [&](auto tx) {
    if (pg.type == kE4M3) sizes(tx, std::integral_constant<int, kE4M3>{});
    else if (pg.type == kI8) sizes(tx, std::integral_constant<int, kI8>{});
    else sizes(tx, tx);
  });
}

// Tokens per CTA: as many as leave six CTAs to an SM, so that few tokens spread
// over the machine and many share the search.
int tokens_per_cta(const SeqTable& sq, int num_sms) {
  return std::max(1, std::min(kMaxTokens, sq.total / (6 * num_sms)));
}

}  // namespace

void kv_pages_append_launch(const RowsView& K, const RowsView& V, const KvPages& pg,
                            const SeqTable& sq, int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg);
  const int tokens = tokens_per_cta(sq, num_sms);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value, LN = decltype(lanes)::value;
    ATTNB_CUDA(launch_pdl(append_kernel<TX, TC, LN>, dim3((sq.total + tokens - 1) / tokens),
                          dim3(kThreads), 0, s, K, V, pg, sq, tokens, vec, index_status));
  });
}

void kv_pages_read_launch(const KvPages& pg, const RowsView& K, const RowsView& V,
                          const SeqTable& sq, int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg);
  const int tokens = tokens_per_cta(sq, num_sms);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value, LN = decltype(lanes)::value;
    ATTNB_CUDA(launch_pdl(read_kernel<TX, TC, LN>, dim3((sq.total + tokens - 1) / tokens),
                          dim3(kThreads), 0, s, pg, K, V, sq, tokens, vec, index_status));
  });
}

}  // namespace attnb
