// kv_pages.cu -- K5: writing packed tokens into the pages of a KV cache, as they
// are or as 8-bit codes, and reading them back.
//
// A vector x of Dh values (one token, one KV head) is stored in e4m3 or int8 as
//     a = max |x|,   code = round(x * C / a),   scale = a / C    (C = 448 or 127)
// with ties to even, so the largest value is the largest code and the value
// read back is code * scale.  The code is that of the exact x * C / a, found
// without a division: for 16-bit x from x * (C / a), which is off by 2^-23 at
// most, rounded to 21 bits: x * C has at most 18 bits and a tie times a at most 19, so
// a quotient that is not on a tie is 2^-19 away from it and stays on its side, and
// one on a tie is put back on it.  For fp32 x the product's bounds up and down
// decide where they agree, elsewhere the quotient in 64 bits (product 33 bits,
// distance 2^-42).  Where C / a leaves fp32's range all take the quotient.  A vector
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
// Measured: 11.7k bf16 tokens of 8 heads x 128 written as e4m3 in 31 us and read
// back in 28 us (72 MB each); issue of instructions and latency, not HBM.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "seq_pages.cuh"
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

// 8 elements of a row as they lie in memory.
template <class E>
struct alignas(sizeof(E) * 8 >= 16 ? 16 : 8) Eight {
  E e[8];
};

// Elements from d on, those past Dh as zero bits.
template <class E>
__device__ __forceinline__ Eight<E> load8(const E* p, int d, int Dh, bool vec) {
  Eight<E> f;
  memset(&f, 0, sizeof(f));
  if (vec) {  // Dh is a multiple of 8
    if (d < Dh) f = *reinterpret_cast<const Eight<E>*>(p + d);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < Dh) f.e[i] = p[d + i];
  }
  return f;
}
template <class E>
__device__ __forceinline__ void store8(E* p, int d, int Dh, bool vec, const Eight<E>& f) {
  if (vec) {
    if (d < Dh) *reinterpret_cast<Eight<E>*>(p + d) = f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < Dh) p[d + i] = f.e[i];
  }
}

// Steps through the CTA's vectors, a group's share of them: token by token, all
// heads of K, then of V.  No division but at the start.
struct Walk {
  int tl, kvh, dt, dr, H2;
  __device__ __forceinline__ Walk(int first, int step, int heads2) : H2(heads2) {
    tl = first / H2;
    kvh = first - tl * H2;
    dt = step / H2;
    dr = step - dt * H2;
  }
  __device__ __forceinline__ void next() {
    tl += dt;
    kvh += dr;
    if (kvh >= H2) {
      kvh -= H2;
      ++tl;
    }
  }
};

// One vector per group of LANES lanes at a time: the CTAs of an SM keep enough
// reads going, and more registers would cost some of those (prompts of 11.7k tokens
// to e4m3 and back: 61 us; 79 with two vectors in flight, 80 with four).
template <int TX, int TC, int LANES>
__global__ void __launch_bounds__(kThreads)
    append_kernel(const RowsView K, const RowsView V, const KvPages pg, const SeqTable sq,
                  const int tokens, const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = TC == kE4M3 || TC == kI8;
  __shared__ int64_t places[kMaxTokens];
  const int e = threadIdx.x % LANES, d = e * 8;
  const int Dh = pg.Dh;
  grid_dep_wait();
  const int t0 = blockIdx.x * tokens, n = min(tokens, sq.total - t0);
  find_places(sq, pg, t0, n, places, index_status);
  // A group's lanes share their vector; the other groups of the warp may have left.
  const unsigned mask =
      LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
  for (Walk at(threadIdx.x / LANES, kThreads / LANES, 2 * pg.H); at.tl < n; at.next()) {
    const bool is_v = at.kvh >= pg.H;
    const int h = is_v ? at.kvh - pg.H : at.kvh;
    const int64_t first = places[at.tl];
    if (first < 0) continue;
    const int64_t place = first + ((int64_t)h << pg.page_shift);
    const RowsView& src = is_v ? V : K;
    const Eight<EX> raw = load8(static_cast<const EX*>(src.data) + (int64_t)(t0 + at.tl) * src.sT +
                                    (int64_t)h * src.sH,
                                d, Dh, vec);
    EC* out = static_cast<EC*>(is_v ? pg.v : pg.k) + place * Dh;
    if constexpr (CODED) {
      constexpr float C = TC == kE4M3 ? 448.f : 127.f;
      float x[8], top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = to_float(raw.e[j]);
        top = max_nan(top, fabsf(x[j]));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(mask, top, o));
      const bool bad = !(top <= 3.402823466e38f);  // a NaN stays one through the maximum
      if (e == 0)
        (is_v ? pg.v_scale : pg.k_scale)[place] = bad ? __int_as_float(0x7fffffff) : top / C;
      if (bad) top = 0.f;
      // C / a overflows for tiny a, and is not used for large ones.
      const float inv = top > 0x1p-100f && top < 0x1p100f ? C / top : 0.f;
      uint32_t r[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float q[4];
        bool exact = inv == 0.f;
        if constexpr (TX == kF32) {
          // x * (C / a) is off by less than 2^-22 of it: where 2^-22 up and down
          // give the same codes, those are the ones; else the quotient decides.
          float down[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x0 = x[4 * k + j] * inv;
            q[j] = x0 * (1.f + 0x1p-22f);
            down[j] = x0 * (1.f - 0x1p-22f);
          }
          r[k] = pack_codes(q, out);
          exact = exact || r[k] != pack_codes(down, out);
        } else {
          // Off by 2^-23 at most.  To 21 bits, what should be a tie is one again,
          // and what should not stays on its side (it is 2^-19 away).
#pragma unroll
          for (int j = 0; j < 4; ++j)
            q[j] = __uint_as_float((__float_as_uint(x[4 * k + j] * inv) + 4u) & ~7u);
          r[k] = pack_codes(q, out);
        }
        if (exact) {
#pragma unroll
          for (int j = 0; j < 4; ++j) q[j] = top > 0.f ? quotient<TX>(x[4 * k + j], top, C) : 0.f;
          r[k] = pack_codes(q, out);
        }
      }
      Eight<EC> codes;
      memcpy(&codes, r, 8);
      store8(out, d, Dh, vec, codes);
    } else {
      store8(out, d, Dh, vec, raw);
    }
  }
}

// Codes times scale, two at a time.
template <int TX, int TC>
__device__ __forceinline__ Eight<elem_t<TX>> decode8(const Eight<elem_t<TC>>& codes, float scale) {
  uint32_t c[2];
  memcpy(c, &codes, 8);
  float x[8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t h[2];
    codes_to_f16<TC>(c[k], h[0], h[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      x[4 * k + 2 * j] = f.x * scale;
      x[4 * k + 2 * j + 1] = f.y * scale;
    }
  }
  Eight<elem_t<TX>> out;
  if constexpr (TX == kF32) {
    memcpy(&out, x, 32);
  } else {
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      y[j] = TX == kBF16 ? pack_bf16(x[2 * j], x[2 * j + 1]) : pack_f16(x[2 * j], x[2 * j + 1]);
    memcpy(&out, y, 16);
  }
  return out;
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
  const int Dh = pg.Dh;
  grid_dep_wait();
  const int t0 = blockIdx.x * tokens, n = min(tokens, sq.total - t0);
  find_places(sq, pg, t0, n, places, index_status);
  for (Walk at(threadIdx.x / LANES, kThreads / LANES, 2 * pg.H); at.tl < n; at.next()) {
    const bool is_v = at.kvh >= pg.H;
    const int h = is_v ? at.kvh - pg.H : at.kvh;
    const int64_t first = places[at.tl];
    if (first == -2) continue;  // a row of no sequence stays as it is
    const RowsView& dst = is_v ? V : K;
    EX* out = static_cast<EX*>(dst.data) + (int64_t)(t0 + at.tl) * dst.sT + (int64_t)h * dst.sH;
    Eight<EC> raw;
    memset(&raw, 0, sizeof(raw));
    float scale = 1.f;
    if (first >= 0) {  // a bad place reads as zeros
      const int64_t place = first + ((int64_t)h << pg.page_shift);
      raw = load8(static_cast<const EC*>(is_v ? pg.v : pg.k) + place * Dh, d, Dh, vec);
      if constexpr (CODED) scale = (is_v ? pg.v_scale : pg.k_scale)[place];
    }
    if constexpr (CODED) store8(out, d, Dh, vec, decode8<TX, TC>(raw, scale));
    else store8(out, d, Dh, vec, raw);
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

// Tokens per CTA: as many as leave four CTAs to an SM (all of them fit at once),
// so that few tokens spread over the machine and many share the search.
int tokens_per_cta(const SeqTable& sq, int num_sms) {
  return std::max(1, std::min(kMaxTokens, (sq.total + 4 * num_sms - 1) / (4 * num_sms)));
}

}  // namespace

void kv_pages_append_launch(const RowsView& K, const RowsView& V, const KvPages& pg,
                            const SeqTable& sq, int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg);
  const int tokens = tokens_per_cta(sq, num_sms);
  ProfScope prof("kv_pages", s);
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
  ProfScope prof("kv_pages", s);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value, LN = decltype(lanes)::value;
    ATTNB_CUDA(launch_pdl(read_kernel<TX, TC, LN>, dim3((sq.total + tokens - 1) / tokens),
                          dim3(kThreads), 0, s, pg, K, V, sq, tokens, vec, index_status));
  });
}

}  // namespace attnb
