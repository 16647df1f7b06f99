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
// Bound by memory: a token is read once and its codes written once.  A group of
// 8 to 32 lanes takes one vector of K or V with 4 elements a lane and step, so
// that the maximum is a few shuffles and no vector is read twice; rows that are
// not aligned for that are read element by element.
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

// One vector per group of LANES lanes; NC groups of 4 elements per lane.
template <int TX, int TC, int LANES, int NC>
__global__ void __launch_bounds__(kThreads)
    append_kernel(const RowsView K, const RowsView V, const KvPages pg, const SeqTable sq,
                  const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = TC == kE4M3 || TC == kI8;
  const int per_block = kThreads / LANES;
  const int e = threadIdx.x % LANES;
  const int Dh = pg.Dh;
  const int64_t vectors = (int64_t)sq.total * 2 * pg.H;
  grid_dep_wait();
  for (int64_t i = (int64_t)blockIdx.x * per_block + threadIdx.x / LANES; i < vectors;
       i += (int64_t)gridDim.x * per_block) {
    // A group's lanes share i; the other groups of the warp may have left.
    const unsigned mask =
        LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
    const int h = (int)(i % pg.H);
    const int64_t tv = i / pg.H;
    const bool is_v = tv >= sq.total;
    const int t = (int)(is_v ? tv - sq.total : tv);
    const RowsView& src = is_v ? V : K;
    const EX* p = static_cast<const EX*>(src.data) + (int64_t)t * src.sT + (int64_t)h * src.sH;
    float x[NC][4];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (c * LANES + e) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][j] = 0.f;
      if (vec) {
        if (d < Dh) load4(p + d, x[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < Dh) x[c][j] = to_float(p[d + j]);
      }
    }
    const int64_t at0 = place_of(sq, pg, t, index_status);
    if (at0 < 0) continue;
    const int64_t at = at0 + ((int64_t)h << pg.page_shift);
    float top = 0.f;
    if constexpr (CODED) {
      constexpr float C = TC == kE4M3 ? 448.f : 127.f;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top = fmaxf(top, fabsf(x[c][j]));
          bad |= !(fabsf(x[c][j]) <= 3.402823466e38f);
        }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(mask, top, o));
        bad |= __shfl_xor_sync(mask, (int)bad, o) != 0;
      }
      if (e == 0)
        (is_v ? pg.v_scale : pg.k_scale)[at] = bad ? __int_as_float(0x7fffffff) : top / C;
      if (bad) top = 0.f;
      EC* out = static_cast<EC*>(is_v ? pg.v : pg.k) + at * Dh;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (c * LANES + e) * 4;
        if (d >= Dh) continue;
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = top > 0.f ? quotient<TX>(x[c][j], top, C) : 0.f;
        const uint32_t r = pack_codes(q, out);
        if (vec) {
          *reinterpret_cast<uint32_t*>(out + d) = r;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d + j < Dh) reinterpret_cast<uint8_t*>(out)[d + j] = (uint8_t)(r >> (8 * j));
        }
      }
    } else {
      EC* out = static_cast<EC*>(is_v ? pg.v : pg.k) + at * Dh;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (c * LANES + e) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < Dh) from_float(x[c][j], out[d + j]);
      }
    }
  }
}

template <int TX, int TC, int LANES, int NC>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const KvPages pg, const RowsView K, const RowsView V, const SeqTable sq,
                const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = TC == kE4M3 || TC == kI8;
  const int per_block = kThreads / LANES;
  const int e = threadIdx.x % LANES;
  const int Dh = pg.Dh;
  const int64_t vectors = (int64_t)sq.total * 2 * pg.H;
  grid_dep_wait();
  for (int64_t i = (int64_t)blockIdx.x * per_block + threadIdx.x / LANES; i < vectors;
       i += (int64_t)gridDim.x * per_block) {
    const int h = (int)(i % pg.H);
    const int64_t tv = i / pg.H;
    const bool is_v = tv >= sq.total;
    const int t = (int)(is_v ? tv - sq.total : tv);
    int first, count;
    if (seq_of(sq, t, first, count) < 0) continue;  // a row of no sequence stays as it is
    const int64_t at0 = place_of(sq, pg, t, index_status);
    const int64_t at = at0 + ((int64_t)h << pg.page_shift);
    const float scale = CODED && at0 >= 0 ? __ldg((is_v ? pg.v_scale : pg.k_scale) + at) : 1.f;
    const EC* p = static_cast<const EC*>(is_v ? pg.v : pg.k) + at * Dh;
    const RowsView& dst = is_v ? V : K;
    EX* out = static_cast<EX*>(dst.data) + (int64_t)t * dst.sT + (int64_t)h * dst.sH;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (c * LANES + e) * 4;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (at0 >= 0) {
        if (vec) {
          if (d < Dh) load4(p + d, x);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d + j < Dh) x[j] = to_float(p[d + j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < Dh) from_float(CODED ? x[j] * scale : x[j], out[d + j]);
    }
  }
}

bool vec_rows(const RowsView& r) {
  const int b = 4 * elem_bytes(r.type);
  return reinterpret_cast<uintptr_t>(r.data) % b == 0 && r.sT % 4 == 0 && r.sH % 4 == 0 &&
         r.Dh % 4 == 0;
}
bool vec_pages(const KvPages& p) {
  const int b = 4 * elem_bytes(p.type);
  return reinterpret_cast<uintptr_t>(p.k) % b == 0 && reinterpret_cast<uintptr_t>(p.v) % b == 0 &&
         p.Dh % 4 == 0;
}

// f(type of the rows, type of the pages, lanes per vector, 4-element groups per lane).
template <class F>
void dispatch(const RowsView& K, const KvPages& pg, F&& f) {
  auto sizes = [&](auto tx, auto tc) {
    using std::integral_constant;
    if (pg.Dh <= 64) f(tx, tc, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (pg.Dh <= 128) f(tx, tc, integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else f(tx, tc, integral_constant<int, 32>{}, integral_constant<int, 2>{});
  };
  with_value_type(K.type, [&](auto tx) {
    if (pg.type == kE4M3) sizes(tx, std::integral_constant<int, kE4M3>{});
    else if (pg.type == kI8) sizes(tx, std::integral_constant<int, kI8>{});
    else sizes(tx, tx);
  });
}

int grid_of(const SeqTable& sq, const KvPages& pg, int lanes, int num_sms) {
  const int64_t vectors = (int64_t)sq.total * 2 * pg.H;
  const int per_block = kThreads / lanes;
  return (int)std::min<int64_t>((vectors + per_block - 1) / per_block, (int64_t)num_sms * 8);
}

}  // namespace

void kv_pages_append_launch(const RowsView& K, const RowsView& V, const KvPages& pg,
                            const SeqTable& sq, int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes, auto nc) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value;
    constexpr int LN = decltype(lanes)::value, NC = decltype(nc)::value;
    ATTNB_CUDA(launch_pdl(append_kernel<TX, TC, LN, NC>, dim3(grid_of(sq, pg, LN, num_sms)),
                          dim3(kThreads), 0, s, K, V, pg, sq, vec, index_status));
  });
}

void kv_pages_read_launch(const KvPages& pg, const RowsView& K, const RowsView& V,
                          const SeqTable& sq, int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes, auto nc) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value;
    constexpr int LN = decltype(lanes)::value, NC = decltype(nc)::value;
    ATTNB_CUDA(launch_pdl(read_kernel<TX, TC, LN, NC>, dim3(grid_of(sq, pg, LN, num_sms)),
                          dim3(kThreads), 0, s, pg, K, V, sq, vec, index_status));
  });
}

}  // namespace attnb
