// kv_pages.cu -- K5: writing packed tokens into the pages of a KV cache, as they
// are or as codes of 8 or 4 bits, rotated by their positions on the way where asked,
// and reading them back.
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
// In 4 bits a vector is stored as
//     a = max |x|,   a_g = max |x| over 32 dimensions,   r_g = ceil(255 a_g / a),
//     code = round(x * 1785 / (a r_g)),   scale = a / 1785
// (1785 = 7 * 255), codes from -7 to 7 held as 1 to 15: a strong channel costs the other
// groups nothing, code * r_g stays below 2048, so that it is a whole number which f16 holds
// exactly, and one scale per vector is left for the attention to apply.  Factors and
// codes are those of the exact quotients: a candidate from the fp32 quotient is
// settled by comparing products, 255 a_g with r a, and 3570 |x| with (2m + 1) a r.
// For 16-bit x these have at most 23 bits and are exact in fp32, once tiny and huge vectors are
// brought near 1; for fp32 x they are taken in 64 bits.
//
// Rotation: x' = x cos t -+ y sin t with y the other one of the pair and t = position *
// inv_freq.  The angle is reduced to a fraction of a turn in 64 bits (at
// position 100000 an fp32 product is off by 0.004), once per token and
// pair of a CTA for all heads.  Sine and cosine are those of the fraction in fp32, turned by
// what its rounding left over (up to 9.4e-8, as much as their own last place); then everything is
// fp32.  The result is rounded to the rows'
// type once and stored as that: the same numbers as rotating first and
// appending then.
//
// Bound by memory: a token is read once and its codes written once.  A CTA takes
// some tokens that follow one another, all heads of K and V.  Where a token
// lives takes a search and three dependent reads, as long as hundreds of
// streamed bytes, so one thread per token finds the places of all of them first.
// Then a group of 8 to 32 lanes takes one vector, 8 elements a lane (one 16-byte
// read of a 16-bit row), so that the maximum is a few shuffles and no vector is
// read twice; rows that are not aligned for that are read element by element.
// Rotating appends take Q's rows in CTAs of their own.  A lane has four whole pairs (elements i and
// i + pairs, or eight in a row), so that nothing is read twice, and goes on through the heads of a
// token with the same sines and cosines, four rows in flight: 12k tokens of 32 query and 8 KV
// heads of 128, bf16 (300 MB) 55 us, 5.4 TB/s; with pairs that lie in two lanes and a
// read of both halves 176 us.  Into 4 bits: 4.8k tokens of 16/4 heads 23 us, by instructions.
//
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

// Place of position `pos` of sequence b in a [.., H, page, ..] pool for head 0, or -1.
__device__ __forceinline__ int64_t place_of(const SeqTable& sq, const KvPages& pg, int b,
                                            int64_t pos, int* index_status) {
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
// out of range and -2 for a row of no sequence.  Their positions go to `position`
// where that is given.
__device__ __forceinline__ void find_places(const SeqTable& sq, const KvPages& pg, int t0, int n,
                                            int64_t* at, int* index_status,
                                            int64_t* position = nullptr) {
  if ((int)threadIdx.x < n) {
    int first, count;
    const int t = t0 + threadIdx.x, b = seq_of(sq, t, first, count);
    const int64_t pos = b < 0 ? 0 : (int64_t)__ldg(sq.lens + b) - count + (t - first);
    at[threadIdx.x] = b < 0 ? -2 : place_of(sq, pg, b, pos, index_status);
    if (position) position[threadIdx.x] = pos;
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
// heads of K, then of V (and of Q).  No division but at the start.
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

// The share of one lane (dimensions d to d + 7) in 4 bits: its eight codes and its
// group's factor.  own, top: the largest magnitudes of the group and of the vector,
// finite.
template <int TX>
__device__ __forceinline__ uint32_t i4_codes(const float (&x)[8], float own, float top, int& factor) {
  // 16-bit values: products exact in fp32, once the vector is brought near 1.
  using Wide = std::conditional_t<TX == kF32, double, float>;
  float near = 1.f;
  if (TX != kF16) near = top > 0x1p60f ? 0x1p-64f : top < 0x1p-60f ? 0x1p64f : 1.f;
  factor = 0;
  if (!(own > 0.f)) return 0x88888888u;
  const float a = top * near;
  own *= near;
  factor = 1;
  if (own == 0.f) return 0x88888888u;  // brought below fp32's least: under 2^-146 of the largest
  int r = min(max((int)ceilf(__fdividef(own, a) * 255.f), 1), 255);
  const Wide want = (Wide)own * (Wide)255;
  if ((Wide)(r - 1) * (Wide)a >= want) --r;
  if ((Wide)r * (Wide)a < want) ++r;
  factor = r;
  const Wide ar = (Wide)a * (Wide)r;
  const float inv = __fdividef(1785.f, (float)ar);
  // Candidates by an addition that leaves code + 8 in the last bits; each is right unless
  // its remainder is half a step or more.
  constexpr float kMagic = 12582912.f + 8.f;
  constexpr uint32_t kMagicBits = 0x4b400000u;  // of 12582912
  uint32_t bits[8];
  bool off = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = x[j] * near, f = fmaf(y, inv, kMagic);
    bits[j] = __float_as_uint(f);
    const Wide rest = (Wide)y * (Wide)1785 - (Wide)(f - kMagic) * ar;
    off |= (Wide)2 * (rest < (Wide)0 ? -rest : rest) >= ar;
  }
  if (off) {  // a tie, or next to one
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (int)(bits[j] - kMagicBits) - 8;
      const Wide rest = (Wide)(x[j] * near) * (Wide)1785 - (Wide)c * ar;
      const Wide two = (Wide)2 * (rest < (Wide)0 ? -rest : rest);
      if (two > ar || (two == ar && (c & 1))) bits[j] += rest < (Wide)0 ? ~0u : 1u;
    }
  }
  uint32_t codes = 0;
#pragma unroll
  for (int j = 7; j >= 0; --j) codes = codes * 16u + bits[j];
  return codes - kMagicBits * 0x11111111u;
}

// cos and sin of every token and pair of the CTA, [n][pairs].
__device__ __forceinline__ void turn_angles(const Rope& rope, const int64_t* position, int n,
                                            float2* turns) {
  for (int i = threadIdx.x; i < n * rope.pairs; i += kThreads) {
    const int t = i / rope.pairs, p = i - t * rope.pairs;
    const double turn = (double)position[t] * (double)__ldg(rope.inv_freq + p) * 0.15915494309189535;
    const double rest = turn - rint(turn);  // of a turn, at most a half
    const float part = (float)rest;
    float s, c;
    sincospif(2.f * part, &s, &c);
    // What part is off by, up to 2^-26 of a turn, turns the two by a small angle.
    const float small = (float)(rest - (double)part) * 6.28318531f;
    turns[i] = make_float2(fmaf(-s, small, c), fmaf(c, small, s));
  }
}

// The lane's eight elements of the row at p, turned; turns: its token's.
template <class E>
__device__ __forceinline__ Eight<E> turned8(const E* p, const Eight<E>& raw, const Rope& rope, int d,
                                            int Dh, bool vec, const float2* turns) {
  Eight<E> other = raw;
  const int half = rope.pairs;
  if (!rope.interleaved && d < 2 * half) {
    if (vec && half % 8 == 0) {
      other = load8(p, d < half ? d + half : d - half, Dh, true);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int x = d + j;
        if (x < 2 * half) other.e[j] = p[x < half ? x + half : x - half];
      }
    }
  }
  Eight<E> out = raw;
  if (half % 8 == 0 && d < 2 * half) {  // all eight turn, and their angles lie together
    const bool second = !rope.interleaved && d >= half;
    float2 cs[8];
    const float4* four = reinterpret_cast<const float4*>(
        turns + (rope.interleaved ? d / 2 : second ? d - half : d));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!rope.interleaved || j < 2) {
        const float4 c = four[j];
        cs[2 * j] = make_float2(c.x, c.y);
        cs[2 * j + 1] = make_float2(c.z, c.w);
      }
    }
    if (rope.interleaved) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = to_float(raw.e[2 * j]), b = to_float(raw.e[2 * j + 1]);
        from_float(fmaf(a, cs[j].x, -(b * cs[j].y)), out.e[2 * j]);
        from_float(fmaf(b, cs[j].x, a * cs[j].y), out.e[2 * j + 1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = to_float(other.e[j]) * cs[j].y;
        from_float(fmaf(to_float(raw.e[j]), cs[j].x, second ? y : -y), out.e[j]);
      }
    }
    return out;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int x = d + j;
    if (x >= 2 * half) continue;
    const bool second = rope.interleaved ? (j & 1) : x >= half;
    const float2 cs = turns[rope.interleaved ? x >> 1 : second ? x - half : x];
    const float near = to_float(raw.e[j ^ 1]), far = to_float(other.e[j]);
    const float y = rope.interleaved ? near : far;
    from_float(fmaf(to_float(raw.e[j]), cs.x, second ? y * cs.y : -(y * cs.y)), out.e[j]);
  }
  return out;
}

// Four elements as they lie in memory, and as floats; rounded once on the way back.
template <int T>
struct Four {
  using Raw = std::conditional_t<T == kF32, float4, uint2>;
  Raw raw;
  __device__ __forceinline__ void load(const elem_t<T>* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(elem_t<T>* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void get(float (&x)[4]) const {
    if constexpr (T == kF32) {
      x[0] = raw.x, x[1] = raw.y, x[2] = raw.z, x[3] = raw.w;
    } else if constexpr (T == kBF16) {
      x[0] = __uint_as_float(raw.x << 16), x[1] = __uint_as_float(raw.x & 0xffff0000u);
      x[2] = __uint_as_float(raw.y << 16), x[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
      x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
  }
  __device__ __forceinline__ void set(float a, float b, float c, float d) {
    if constexpr (T == kF32) raw = make_float4(a, b, c, d);
    else if constexpr (T == kBF16) raw = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
    else raw = make_uint2(pack_f16(a, b), pack_f16(c, d));
  }
};

// Vectors of the CTA's n tokens, `heads` each, from src to dst as they are, or turned (pairs > 0).
// to(tl) is where token tl's first vector goes, null for one that is left out.  The layout has
// to allow reads of four elements (vec) and pairs that are a multiple of four: a lane takes four
// whole pairs, or eight dimensions that stay, and so reads nothing twice.  A group of lanes
// takes several heads of one token in turn, four of them in flight.
template <int TX, int LANES, class To>
__device__ __forceinline__ void move_rows(const elem_t<TX>* src, int64_t src_t, int64_t src_h, To to,
                                          int64_t dst_h, int heads, int Dh, int pairs,
                                          bool interleaved, const float2* turns, int turns_t,
                                          int n) {
  using E = elem_t<TX>;
  constexpr int U = 4, GROUPS = kThreads / LANES;
  const int e = threadIdx.x % LANES;
  const bool turned = e < pairs / 4;
  const int d = turned && !interleaved ? 4 * e : 8 * e;
  const int d2 = turned && !interleaved ? pairs + 4 * e : d + 4;
  if (d2 >= Dh) return;
  // Few tokens: several groups share one.
  const int slices = min(heads, max(1, GROUPS / n)), per = (heads + slices - 1) / slices;
  for (int item = threadIdx.x / LANES; item < n * slices; item += GROUPS) {
    const int tl = item / slices, h0 = (item - tl * slices) * per, h1 = min(heads, h0 + per);
    E* o = to(tl);
    if (!o) continue;
    o += h0 * dst_h;
    const E* p = src + tl * src_t + h0 * src_h;
    float4 c0 = {}, c1 = {};
    if (turned) {
      const float4* cs = reinterpret_cast<const float4*>(turns + tl * turns_t) + 2 * e;
      c0 = cs[0];
      c1 = cs[1];
    }
    for (int h = h0; h < h1; h += U) {
      Four<TX> x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u < h1) {
          x[u].load(p + d);
          y[u].load(p + d2);
        }
        p += src_h;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u < h1) {
          if (turned) {
            float a[4], b[4];
            x[u].get(a);
            y[u].get(b);
            if (interleaved) {
              x[u].set(fmaf(a[0], c0.x, -(a[1] * c0.y)), fmaf(a[1], c0.x, a[0] * c0.y),
                       fmaf(a[2], c0.z, -(a[3] * c0.w)), fmaf(a[3], c0.z, a[2] * c0.w));
              y[u].set(fmaf(b[0], c1.x, -(b[1] * c1.y)), fmaf(b[1], c1.x, b[0] * c1.y),
                       fmaf(b[2], c1.z, -(b[3] * c1.w)), fmaf(b[3], c1.z, b[2] * c1.w));
            } else {
              x[u].set(fmaf(a[0], c0.x, -(b[0] * c0.y)), fmaf(a[1], c0.z, -(b[1] * c0.w)),
                       fmaf(a[2], c1.x, -(b[2] * c1.y)), fmaf(a[3], c1.z, -(b[3] * c1.w)));
              y[u].set(fmaf(b[0], c0.x, a[0] * c0.y), fmaf(b[1], c0.z, a[1] * c0.w),
                       fmaf(b[2], c1.x, a[2] * c1.y), fmaf(b[3], c1.z, a[3] * c1.w));
            }
          }
          x[u].store(o + d);
          y[u].store(o + d2);
        }
        o += dst_h;
      }
    }
  }
}

// The rows Q of the CTA's tokens, turned into QO.
template <int TX, int LANES>
__device__ __forceinline__ void turn_rows(const RowsView& Q, const RowsView& QO, const Rope& rope,
                                          const int64_t* places, const float2* turns, int t0,
                                          int n, bool vec) {
  using E = elem_t<TX>;
  const E* const from = static_cast<const E*>(Q.data) + (int64_t)t0 * Q.sT;
  E* const to = static_cast<E*>(QO.data) + (int64_t)t0 * QO.sT;
  const int e = threadIdx.x % LANES, Dh = Q.Dh;
  if (vec && rope.pairs % 4 == 0) {
    move_rows<TX, LANES>(
        from, Q.sT, Q.sH, [&](int tl) { return places[tl] == -2 ? nullptr : to + tl * QO.sT; },
        QO.sH, Q.heads, Dh, rope.pairs, rope.interleaved, turns, rope.pairs, n);
    return;
  }
  const unsigned mask =
      LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
  for (Walk at(threadIdx.x / LANES, kThreads / LANES, Q.heads); at.tl < n; at.next()) {
    if (places[at.tl] == -2) continue;
    const E* p = from + at.tl * Q.sT + at.kvh * Q.sH;
    const Eight<E> raw = load8(p, 8 * e, Dh, vec);
    const Eight<E> out = turned8(p, raw, rope, 8 * e, Dh, vec, turns + at.tl * rope.pairs);
    __syncwarp(mask);  // a row may be turned in place: all have read
    store8(to + at.tl * QO.sT + at.kvh * QO.sH, 8 * e, Dh, vec, out);
  }
}

// One vector per group of LANES lanes at a time: the CTAs of an SM keep enough
// reads going, and more registers would cost some of those (prompts of 11.7k tokens
// to e4m3 and back: 61 us; 79 with two vectors in flight, 80 with four).
// With ROPE the first q_ctas CTAs take Q's rows, the others K and V.
template <int TX, int TC, int LANES, bool ROPE>
__global__ void __launch_bounds__(kThreads, ROPE ? 4 : 1)
    append_kernel(const RowsView K, const RowsView V, const RowsView Q, const RowsView QO,
                  const KvPages pg, const SeqTable sq, const Rope rope, const int q_ctas,
                  const int tokens, const bool vec, int* index_status) {
  using EX = elem_t<TX>;
  using EC = elem_t<TC>;
  constexpr bool CODED = elem_coded(TC);
  __shared__ int64_t places[kMaxTokens], position[ROPE ? kMaxTokens : 1];
  extern __shared__ __align__(16) float2 turns[];
  const int e = threadIdx.x % LANES, d = e * 8;
  const int Dh = pg.Dh;
  grid_dep_wait();
  const bool is_q = ROPE && (int)blockIdx.x < q_ctas;
  const int t0 = (blockIdx.x - (is_q ? 0 : q_ctas)) * tokens, n = min(tokens, sq.total - t0);
  find_places(sq, pg, t0, n, places, index_status, ROPE ? position : nullptr);
  if constexpr (ROPE) {
    turn_angles(rope, position, n, turns);
    __syncthreads();
    if (is_q) {
      turn_rows<TX, LANES>(Q, QO, rope, places, turns, t0, n, vec);
      return;
    }
    if constexpr (TC == TX) {
      if (vec && rope.pairs % 4 == 0) {
        const int64_t head = (int64_t)Dh << pg.page_shift;
        auto move = [&](const RowsView& src, void* pages, int pairs) {
          move_rows<TX, LANES>(
              static_cast<const EX*>(src.data) + (int64_t)t0 * src.sT, src.sT, src.sH,
              [&](int tl) {
                return places[tl] < 0 ? nullptr : static_cast<EX*>(pages) + places[tl] * Dh;
              },
              head, pg.H, Dh, pairs, rope.interleaved, turns, rope.pairs, n);
        };
        move(K, pg.k, rope.pairs);
        move(V, pg.v, 0);
        return;
      }
    }
  }
  // A group's lanes share their vector; the other groups of the warp may have left.
  const unsigned mask =
      LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
  for (Walk at(threadIdx.x / LANES, kThreads / LANES, 2 * pg.H); at.tl < n; at.next()) {
    const bool is_v = at.kvh >= pg.H;
    const int h = is_v ? at.kvh - pg.H : at.kvh;
    const int64_t first = places[at.tl];
    if (first < 0) continue;
    const EX* row = static_cast<const EX*>(is_v ? V.data : K.data) +
                    (int64_t)(t0 + at.tl) * (is_v ? V.sT : K.sT) +
                    (int64_t)h * (is_v ? V.sH : K.sH);
    Eight<EX> raw = load8(row, d, Dh, vec);
    if (ROPE && !is_v) raw = turned8(row, raw, rope, d, Dh, vec, turns + at.tl * rope.pairs);
    const int64_t place = first + ((int64_t)h << pg.page_shift);
    if constexpr (TC == kI4) {
      float x[8], own = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = to_float(raw.e[j]);
        own = max_nan(own, fabsf(x[j]));
      }
      own = max_nan(own, __shfl_xor_sync(mask, own, 1));  // 32 dimensions are four lanes
      own = max_nan(own, __shfl_xor_sync(mask, own, 2));
      float top = own;
#pragma unroll
      for (int o = LANES / 2; o > 2; o >>= 1) top = max_nan(top, __shfl_xor_sync(mask, top, o));
      const bool bad = !(top <= 3.402823466e38f);
      if (e == 0)
        (is_v ? pg.v_scale : pg.k_scale)[place] = bad ? __int_as_float(0x7fffffff) : top / 1785.f;
      int factor;
      const uint32_t codes = i4_codes<TX>(x, bad ? 0.f : own, top, factor);
      if (d < Dh)
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(is_v ? pg.v : pg.k) +
                                     place * (Dh / 2) + d / 2) = codes;
      const int bytes = i4_group_bytes(Dh);
      if (e % 4 == 0)  // a lane of the group writes its factor, and zeros behind the last group
        for (int g = e / 4; g < bytes; g += LANES / 4)
          (is_v ? pg.v_group : pg.k_group)[place * bytes + g] = g == e / 4 ? (uint8_t)factor : 0;
    } else if constexpr (CODED) {
      EC* out = static_cast<EC*>(is_v ? pg.v : pg.k) + place * Dh;
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
      store8(static_cast<EC*>(is_v ? pg.v : pg.k) + place * Dh, d, Dh, vec, raw);
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
  constexpr bool CODED = elem_coded(TC);
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
    if constexpr (TC == kI4) {
      Eight<EX> back;
      memset(&back, 0, sizeof(back));
      if (first >= 0 && d < Dh) {
        const int64_t place = first + ((int64_t)h << pg.page_shift);
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(
            static_cast<const uint8_t*>(is_v ? pg.v : pg.k) + place * (Dh / 2) + d / 2);
        const float scale = (is_v ? pg.v_scale : pg.k_scale)[place];
        float x[8];
        i4_values(codes, (is_v ? pg.v_group : pg.k_group)[place * i4_group_bytes(Dh) + d / kI4Group],
                  x);
#pragma unroll
        for (int j = 0; j < 8; ++j) from_float(x[j] * scale, back.e[j]);
      }
      store8(out, d, Dh, vec, back);
    } else {
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
}

bool vec_rows(const RowsView& r) {
  // 8 elements are read as 16 bytes (32-bit ones as two times 16).
  const int unit = 16 / elem_bytes(r.type);
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.sT % unit == 0 && r.sH % unit == 0 &&
         r.Dh % 8 == 0;
}
bool vec_pages(const KvPages& p) {
  if (p.type == kI4) return true;  // their own reads and writes, of 4 bytes
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
    else if (pg.type == kI4) sizes(tx, std::integral_constant<int, kI4>{});
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
    ATTNB_CUDA(launch_pdl(append_kernel<TX, TC, LN, false>,
                          dim3((sq.total + tokens - 1) / tokens), dim3(kThreads), 0, s, K, V,
                          RowsView{}, RowsView{}, pg, sq, Rope{}, 0, tokens, vec, index_status));
  });
}

void kv_pages_append_rope_launch(const RowsView& Q, const RowsView& QO, const RowsView& K,
                                 const RowsView& V, const KvPages& pg, const SeqTable& sq,
                                 const Rope& rope, int* index_status, int num_sms,
                                 cudaStream_t s) {
  const bool vec = vec_rows(K) && vec_rows(V) && vec_pages(pg) &&
                   (Q.heads == 0 || (vec_rows(Q) && vec_rows(QO)));
  const int tokens = tokens_per_cta(sq, Q.heads ? num_sms / 2 : num_sms);
  ProfScope prof("kv_pages", s);
  dispatch(K, pg, [&](auto tx, auto tc, auto lanes) {
    constexpr int TX = decltype(tx)::value, TC = decltype(tc)::value, LN = decltype(lanes)::value;
    const int ctas = (sq.total + tokens - 1) / tokens, q_ctas = Q.heads ? ctas : 0;
    ATTNB_CUDA(launch_pdl(append_kernel<TX, TC, LN, true>, dim3(ctas + q_ctas), dim3(kThreads),
                          tokens * rope.pairs * sizeof(float2), s, K, V, Q, QO, pg, sq, rope,
                          q_ctas, tokens, vec, index_status));
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
