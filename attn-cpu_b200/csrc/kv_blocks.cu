// kv_blocks.cu -- K10: choosing the blocks of a long context that a token attends to.
//
// A block is one page of a sequence.  Its bounds are the least and the greatest
// value of its keys in each dimension, so that for a query q
//     q . k <= sum_d max(q_d least_d, q_d greatest_d)     for every key k of the block
// (the bounds of coded pages are rounded to nearest, and the sum may be below by as much).
// The score of a block for a token and a KV head is that bound summed over the query
// heads that read the KV head.  It is linear in the positive and the negative part of
// the queries: with q- = sum over heads of min(q, 0) and q+ = sum of max(q, 0),
//     score = q- . least + q+ . greatest,
// one product of 2 Dh numbers for all heads.  (That holds for finite numbers; where the result is not
// finite the score is made anew by its definition.)  Sums are in 64 bits: products of 16-bit or
// fp32 values and their sum are then off by 2^-53 or so, and which of two blocks is
// better does not hang on the order of a sum.
//
// Bounds are made of the blocks that new tokens complete.  Scores become 64-bit keys that sort as
// they do, and the greatest are chosen from those, in the same kernel where a row is short (keys
// in shared memory), else in a second one.  Equal scores: the lower block.  A NaN counts as
// greatest.
//
// Bound by latency: what a row waits for is offsets and lengths, then the table, then the
// bounds, a microsecond each from HBM, and after that the conversions to 64 bits, 16 a
// cycle and SM.  Measured, in graphs: 32 steps over 8000-32768 keys, 8 KV heads of 128 (90000
// blocks of 512 bytes) 22 us, one of 131071 keys in blocks of 32 16 us; bounds of a step 6 us.
#include <algorithm>
#include <cmath>
#include <climits>

#include "runtime.h"
#include "seq_elem.cuh"
#include "seq_pages.cuh"

namespace attnb {
namespace {

constexpr int kBoundsThreads = 256;
constexpr int kScoreThreads = 256;
constexpr int kScoreRound = kScoreThreads / 8 * 2;  // blocks of one round of a CTA of the score kernel
constexpr int kScoreMost = 8 * kScoreRound;         // blocks of one CTA
constexpr int kPickThreads = 512;
constexpr int kPickKeys = 4096;   // of a row, held in shared memory
constexpr int kPickParts = 2048;  // of the scores' range
constexpr size_t kScoreBytes = 64u << 20;  // workspace for scores, at most (or one token's)

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Tokens that a sequence of length `len` holds, as far as its table goes.
__device__ __forceinline__ int held(int len, const SeqTable& sq, int page_shift,
                                    int* index_status) {
  const long long room = (long long)sq.max_pages << page_shift;
  if (len < 0 || len > room) raise_index(index_status);
  return (int)min((long long)max(len, 0), room);
}

// ------------------------------------------------------------------ bounds
// Value d of the key at `place`.
template <int TC>
__device__ __forceinline__ float key_value(const KvPages& pg, int64_t place, int d) {
  if constexpr (TC == kI4) {
    const uint8_t* row = static_cast<const uint8_t*>(pg.k) + place * (pg.Dh / 2);
    const int code = (row[d >> 1] >> (4 * (d & 1))) & 15;
    const int factor = pg.k_group[place * i4_group_bytes(pg.Dh) + d / kI4Group];
    return (float)((code - 8) * factor) * pg.k_scale[place];
  } else {
    const float x = to_float(static_cast<const elem_t<TC>*>(pg.k)[place * pg.Dh + d]);
    return elem_coded(TC) ? x * pg.k_scale[place] : x;
  }
}

// Dimensions d to d + 7 of the key at `place`; codes without their scale.
template <int TC>
__device__ __forceinline__ void key_eight(const KvPages& pg, int64_t place, int d, float (&x)[8]) {
  if constexpr (TC == kI4) {
    const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>(
        static_cast<const uint8_t*>(pg.k) + place * (pg.Dh / 2) + d / 2));
    i4_values(codes, __ldg(pg.k_group + place * i4_group_bytes(pg.Dh) + d / kI4Group), x);
  } else {
    const elem_t<TC>* p = static_cast<const elem_t<TC>*>(pg.k) + place * pg.Dh + d;
    load4(p, *reinterpret_cast<float(*)[4]>(x));
    load4(p + 4, *reinterpret_cast<float(*)[4]>(x + 4));
  }
}

// A CTA takes every gridDim.x-th of the pairs (completed block, head).  vec: groups of 8 to
// 32 lanes take a key, 8 dimensions a lane, so that the keys of a page are read in a few
// rounds; else a thread takes a dimension.
template <int TC, int TB>
__global__ void __launch_bounds__(kBoundsThreads)
    bounds_kernel(const KvPages pg, void* bounds, const SeqTable sq, const bool vec,
                  int* index_status) {
  using EB = elem_t<TB>;
  __shared__ long long warps[32];
  __shared__ int before[kBoundsThreads], block0[kBoundsThreads];
  __shared__ float2 part[kBoundsThreads / 32][256];
  const int tid = threadIdx.x, page = 1 << pg.page_shift;
  grid_dep_wait();
  for (int b0 = 0; b0 < sq.batch; b0 += kBoundsThreads) {
    int j0 = 0, count = 0;
    if (b0 + tid < sq.batch) {
      const int b = b0 + tid, len = held(__ldg(sq.lens + b), sq, pg.page_shift, index_status);
      int first, n;
      seq_rows(sq.cu, b, INT_MAX, first, n);
      j0 = (len - min(n, len)) >> pg.page_shift;
      count = (len >> pg.page_shift) - j0;
    }
    long long excl;
    const long long total = block_scan(count, excl, warps);  // at most batch * max_pages
    before[tid] = (int)excl;
    block0[tid] = j0;
    __syncthreads();
    for (long long i = blockIdx.x; i < total * pg.H; i += gridDim.x) {
      const int at = (int)(i / pg.H), h = (int)(i - (long long)at * pg.H);
      int lo = 0, hi = kBoundsThreads;  // the last sequence with before <= at
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= at) lo = mid;
        else hi = mid;
      }
      const int number = seq_page(sq, pg, b0 + lo, (block0[lo] + at - before[lo]) << pg.page_shift,
                                  index_status);
      if (number < 0) continue;  // the same for the whole block
      const int64_t place = ((int64_t)number * pg.H + h) << pg.page_shift;
      EB* out = static_cast<EB*>(bounds) + ((int64_t)number * pg.H + h) * 2 * pg.Dh;
      if (vec) {
        const int lanes = pg.Dh <= 64 ? 8 : pg.Dh <= 128 ? 16 : 32, d = tid % lanes * 8;
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo[e] = INFINITY;
          hi[e] = -INFINITY;
        }
        if (d < pg.Dh) {
#pragma unroll 4
          for (int key = tid / lanes; key < page; key += kBoundsThreads / lanes) {
            float x[8];
            key_eight<TC>(pg, place + key, d, x);
            const float scale = elem_coded(TC) ? __ldg(pg.k_scale + place + key) : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = elem_coded(TC) ? x[e] * scale : x[e];
              lo[e] = min_nan(lo[e], v);
              hi[e] = max_nan(hi[e], v);
            }
          }
        }
        // The groups of a warp meet by shuffles, the warps in shared memory.
        for (int o = 16; o >= lanes; o >>= 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            lo[e] = min_nan(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
            hi[e] = max_nan(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
          }
        }
        __syncthreads();  // the block before has been read
        if ((tid & 31) < lanes) {
#pragma unroll
          for (int e = 0; e < 8; ++e) part[tid >> 5][d + e] = make_float2(lo[e], hi[e]);
        }
        __syncthreads();
        for (int i = tid; i < pg.Dh; i += kBoundsThreads) {
          float2 x = part[0][i];
          for (int w = 1; w < kBoundsThreads / 32; ++w)
            x = make_float2(min_nan(x.x, part[w][i].x), max_nan(x.y, part[w][i].y));
          from_float(x.x, out[i]);
          from_float(x.y, out[pg.Dh + i]);
        }
      } else {
        for (int d = tid; d < pg.Dh; d += kBoundsThreads) {
          float2 x = make_float2(INFINITY, -INFINITY);
#pragma unroll 8
          for (int key = 0; key < page; ++key) {
            const float v = key_value<TC>(pg, place + key, d);
            x = make_float2(min_nan(x.x, v), max_nan(x.y, v));
          }
          from_float(x.x, out[d]);
          from_float(x.y, out[pg.Dh + d]);
        }
      }
    }
    __syncthreads();  // before and block0 have been read
  }
}

// ------------------------------------------------------------------ scores
struct BlockArgs {
  RowsView q;
  const void* bounds;
  SeqTable seqs;
  int num_pages, H, G, page_shift;
  int keep_first, keep_last, take;
  int token0, tokens;     // the part of the rows that this launch takes
  int chunk;              // blocks of one CTA of the score kernel
  uint64_t* keys;         // [tokens][H][max_pages]
  int32_t* blocks;        // [all tokens][H][take]
  int* index_status;
};

// The place of packed token t.  `threads` threads find it side by side: each tries every so many
// of the sequences, offsets and lengths read at once, where a search would wait for one read
// after the other.
struct TokenPlace {
  int b;    // its sequence, -1: none
  int pos;  // its position, negative where its sequence holds less than it brings
};
// This thread's finding, as a number of which the greatest counts; 0: none.
__device__ __forceinline__ unsigned long long find_token(const SeqTable& sq, int page_shift, int t,
                                                         int tid, int threads, int* index_status) {
  unsigned long long found = 0;
  for (int b = tid; b < sq.batch; b += threads) {
    const int len = __ldg(sq.lens + b);
    int first, count;
    seq_rows(sq.cu, b, sq.total, first, count);
    if (t >= first && t < first + count) {
      const int pos = held(len, sq, page_shift, index_status) - count + (t - first);
      found = (unsigned long long)(b + 1) << 32 | (unsigned)pos;
    }
  }
  return found;
}
__device__ __forceinline__ TokenPlace token_place(unsigned long long found) {
  return {(int)(found >> 32) - 1, (int)(unsigned)found};
}
// For all threads of a block.
__device__ __forceinline__ TokenPlace block_token(const SeqTable& sq, int page_shift, int t,
                                                  unsigned long long* sh, int* index_status) {
  if (threadIdx.x == 0) *sh = 0;
  __syncthreads();
  const unsigned long long found =
      find_token(sq, page_shift, t, threadIdx.x, blockDim.x, index_status);
  if (found) atomicMax(sh, found);
  __syncthreads();
  return token_place(*sh);
}

// Unsigned numbers that sort as the scores do.
__device__ __forceinline__ uint64_t sort_key(double x) {
  if (x != x) return ~0ull;
  if (x == 0.0) x = 0.0;  // -0 is 0
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (1ull << 63);
}

__device__ __forceinline__ double key_score(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ (1ull << 63) : ~k));
}

// Sums of the queries' negative and positive parts over the query heads of a KV head: q-, q+, zeros.
// The eight lanes that read at once find their pairs side by side.
template <int TB, int NU>
__device__ __forceinline__ void query_parts(const BlockArgs& a, int t, int h, double* parts) {
  using EB = elem_t<TB>;
  constexpr int PER = 16 / sizeof(EB);
  const int Dh = a.q.Dh;
  for (int d = threadIdx.x; d < NU * 8 * PER; d += kScoreThreads) {
    const bool high = d >= Dh;
    double sum = 0.0;
    if (d < 2 * Dh) {
      const EB* q = static_cast<const EB*>(a.q.data) + (int64_t)(a.token0 + t) * a.q.sT +
                    (int64_t)h * a.G * a.q.sH + (high ? d - Dh : d);
#pragma unroll 4
      for (int g = 0; g < a.G; ++g) {
        const float x = to_float(q[g * a.q.sH]);  // (a NaN goes to both)
        sum += (double)(high ? (x < 0.f ? 0.f : x) : (x > 0.f ? 0.f : x));
      }
    }
    parts[((d / (8 * PER) * (PER / 2) + d % PER / 2) * 8 + d / PER % 8) * 2 + d % 2] = sum;
  }
}

// The score of a block as it is defined, from its bounds (null: zeros) and the G queries from q on.  The
// eight lanes of a block call, and all have it.
template <class EB>
__device__ __noinline__ double defined_score(const EB* q, int64_t stride, int G, int Dh,
                                             const EB* bounds) {
  double sum = 0.0;
  for (int d = threadIdx.x & 7; d < Dh; d += 8) {
    const double least = bounds ? (double)to_float(bounds[d]) : 0.0;
    const double greatest = bounds ? (double)to_float(bounds[Dh + d]) : 0.0;
    for (int g = 0; g < G; ++g) {
      const double x = (double)to_float(q[g * stride + d]), lo = x * least, hi = x * greatest;
      sum += lo != lo || lo > hi ? lo : hi;  // a NaN of either one
    }
  }
  const unsigned mask = 0xffu << (threadIdx.x & 24);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
  return sum;
}

// Scores of blocks [from, to) of sequence b, at most kScoreMost, to keys: eight lanes a
// block, each with every eighth unit of 16 bytes of its bounds, two blocks in flight.  The
// queries' sums are read from shared memory: in registers they would leave too few CTAs an SM
// for the latency of the reads that come before the bounds (32 us for 32 sequences of
// 8000-32768 keys).  NU: units a lane.  All threads call.
template <int TB, int NU>
__device__ __forceinline__ void score_blocks(const BlockArgs& a, int b, int t, int h, int from,
                                             int to, bool vec, const double* parts, int* pages,
                                             uint64_t* keys) {
  using EB = elem_t<TB>;
  constexpr int PER = 16 / sizeof(EB);
  const int tid = threadIdx.x, e = tid & 7, Dh = a.q.Dh;
  for (int j = from + tid; j < to; j += kScoreThreads) {
    int page = __ldg(a.seqs.table + b * a.seqs.table_stride + j);
    if (page < 0 || page >= a.num_pages) {
      raise_index(a.index_status);  // bounds of zeros
      page = -1;
    }
    pages[j - from] = page;
  }
  __syncthreads();
  bool odd = false;
  for (int j0 = from; j0 < to; j0 += kScoreRound) {
    uint4 y[2][NU];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = j0 + k * (kScoreRound / 2) + (tid >> 3);
      const int page = j < to ? pages[j - from] : -1;
      const EB* p = static_cast<const EB*>(a.bounds) + ((int64_t)page * a.H + h) * 2 * Dh;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int d = (u * 8 + e) * PER;
        y[k][u] = make_uint4(0, 0, 0, 0);
        if (page >= 0 && d < 2 * Dh) {
          if (vec) {  // 2 Dh is a multiple of PER
            y[k][u] = *reinterpret_cast<const uint4*>(p + d);
          } else {
            EB* v = reinterpret_cast<EB*>(&y[k][u]);
#pragma unroll
            for (int i = 0; i < PER; ++i)
              if (d + i < 2 * Dh) v[i] = p[d + i];
          }
        }
      }
    }
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int i = 0; i < PER / 2; ++i) {
        const double2 two = reinterpret_cast<const double2*>(parts)[(u * (PER / 2) + i) * 8 + e];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const EB* v = reinterpret_cast<const EB*>(&y[k][u]);
          s[k] = fma(two.x, (double)to_float(v[2 * i]), s[k]);
          s[k] = fma(two.y, (double)to_float(v[2 * i + 1]), s[k]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
      const int j = j0 + k * (kScoreRound / 2) + (tid >> 3);
      odd |= !(fabs(s[k]) < INFINITY) && j < to;
      if (e == 0 && j < to) keys[j - from] = sort_key(s[k]);
    }
  }
  // Where bounds or queries are infinite the products above may have had an infinity and the zero of
  // the other sign's part: what is not finite is made anew.  (Within the loop this would cost it
  // registers.)
  if (!__any_sync(0xffffffffu, odd)) return;
  __syncwarp();  // keys that a group's first lane wrote are read by all of it
  const EB* q = static_cast<const EB*>(a.q.data) + (int64_t)(a.token0 + t) * a.q.sT +
                (int64_t)h * a.G * a.q.sH;
  for (int j = from + (tid >> 3); j < to; j += kScoreThreads / 8) {
    if (fabs(key_score(keys[j - from])) < INFINITY) continue;  // the same for all eight lanes
    const int page = pages[j - from];
    const double score = defined_score(
        q, a.q.sH, a.G, Dh,
        page < 0 ? nullptr
                 : static_cast<const EB*>(a.bounds) + ((int64_t)page * a.H + h) * 2 * Dh);
    if (e == 0) keys[j - from] = sort_key(score);
  }
}

// A CTA takes a.chunk blocks of a token and KV head.
template <int TB, int NU>
__global__ void __launch_bounds__(kScoreThreads, NU <= 4 ? 4 : NU <= 8 ? 2 : 1)
    score_kernel(const BlockArgs a, const bool vec) {
  __shared__ __align__(16) double parts[NU * 8 * 16 / sizeof(elem_t<TB>)];
  __shared__ int pages[kScoreMost];
  __shared__ unsigned long long found;
  const int row = blockIdx.y, t = row / a.H, h = row - t * a.H;
  grid_dep_wait();
  query_parts<TB, NU>(a, t, h, parts);
  const TokenPlace at = block_token(a.seqs, a.page_shift, a.token0 + t, &found, a.index_status);
  if (at.b < 0 || at.pos < 0) return;
  const int own = at.pos >> a.page_shift;
  if (own + 1 <= a.take) return;  // all of them
  const int from = a.keep_first + blockIdx.x * a.chunk;
  const int to = min(own + 1 - a.keep_last, from + a.chunk);
  if (from >= to) return;
  score_blocks<TB, NU>(a, at.b, t, h, from, to, vec, parts, pages,
                       a.keys + (int64_t)row * a.seqs.max_pages + from);
}

// ------------------------------------------------------------------ choice
// The parts of a list that need no score; how many of the n others are wanted, 0 if the list is
// complete.  `who` of `all` threads call.
__device__ __forceinline__ int plain_part(const BlockArgs& a, const TokenPlace& at, int row,
                                          int32_t*& out, int& n, int who, int all) {
  if (at.b < 0) return 0;  // rows of no sequence stay
  const int t = row / a.H, h = row - t * a.H;
  const int own = at.pos < 0 ? -1 : at.pos >> a.page_shift;
  out = a.blocks + ((int64_t)(a.token0 + t) * a.H + h) * a.take;
  if (own + 1 <= a.take) {
    for (int i = who; i < a.take; i += all) out[i] = i <= own ? i : -1;
    return 0;
  }
  for (int i = who; i < a.keep_first; i += all) out[i] = i;
  for (int i = who; i < a.keep_last; i += all)
    out[a.take - a.keep_last + i] = own + 1 - a.keep_last + i;
  out += a.keep_first;
  n = own + 1 - a.keep_first - a.keep_last;
  return a.take - a.keep_first - a.keep_last;  // < n
}

// The `want` greatest of up to kWarpKeys keys, by one warp with the keys in registers.  The key that
// is taken last is built from its first bit that not all keys share, each bit set if enough
// keys are still at or above; it ends where as many are as are wanted.  (1064 rows of 80-310
// keys: 23 us with a CTA each.)
constexpr int kWarpKeys = 512;
__device__ __forceinline__ void pick_warp(const uint64_t* keys, int n, int want, int keep_first,
                                          int32_t* out) {
  constexpr int EACH = kWarpKeys / 32;
  const int lane = threadIdx.x & 31;
  uint64_t k[EACH], lo = ~0ull, hi = 0;  // no key is 0
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    k[i] = i * 32 + lane < n ? keys[i * 32 + lane] : 0;
    if (k[i]) lo = min(lo, k[i]);
    hi = max(hi, k[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, (uint64_t)__shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, (uint64_t)__shfl_xor_sync(0xffffffffu, hi, o));
  }
  uint64_t last = hi;
  int rest = want;  // of the keys equal to it
  if (lo != hi) {
    int bit = 63 - __clzll((long long)(lo ^ hi)), count = 0;
    last = bit == 63 ? 0 : hi >> (bit + 1) << (bit + 1);
    for (; bit >= 0; --bit) {
      const uint64_t next = last | 1ull << bit;
      unsigned c = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) c += k[i] >= next;
      count = (int)__reduce_add_sync(0xffffffffu, c);
      if (count >= want) last = next;
      if (count == want) break;
    }
    if (bit < 0) {
      unsigned c = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) c += k[i] > last;
      rest -= (int)__reduce_add_sync(0xffffffffu, c);
    } else {
      --last;  // all above it, and none of its equals
      rest = 0;
    }
  }
  const unsigned before = (1u << lane) - 1;
  int at = 0, same = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (i * 32 >= n) break;
    const bool equal = k[i] == last;
    const unsigned eq = __ballot_sync(0xffffffffu, equal);
    const bool taken = k[i] > last || (equal && same + __popc(eq & before) < rest);
    const unsigned tk = __ballot_sync(0xffffffffu, taken);
    if (taken) out[at + __popc(tk & before)] = keep_first + i * 32 + lane;
    at += __popc(tk);
    same += __popc(eq);
  }
}

// The `want` greatest of n keys, by a block; up to `hold` keys from global memory are put in `mine`
// (null: they are read from where they are).  The key that is taken last is found by a
// histogram over equal parts of the scores' range and the ranks of the few in its part; where that
// part is full (many equal scores, or scores far off the others) or the range is not
// finite, by digits of 8 bits from the first bit in which keys differ.
template <int kPickThreads>
struct PickShared {
  static constexpr int W = kPickThreads / 32;
  int hist[kPickParts];
  int warp_sum[W], warp_eq[W];
  uint64_t warp_lo[W], warp_hi[W];
  uint64_t few_key[kPickThreads], last_key;
  int few_at[kPickThreads];
  int digit, left, few;
};
template <int kPickThreads>
__device__ __forceinline__ void pick_block(const uint64_t* keys, uint64_t* mine, int hold, int n,
                                           int want, int keep_first, int32_t* out,
                                           PickShared<kPickThreads>& sh) {
  constexpr int W = kPickThreads / 32;
  int(&hist)[kPickParts] = sh.hist;
  int(&warp_sum)[W] = sh.warp_sum;
  int(&warp_eq)[W] = sh.warp_eq;
  uint64_t(&warp_lo)[W] = sh.warp_lo;
  uint64_t(&warp_hi)[W] = sh.warp_hi;
  uint64_t(&few_key)[kPickThreads] = sh.few_key;
  int(&few_at)[kPickThreads] = sh.few_at;
  int &digit = sh.digit, &left = sh.left, &few = sh.few;
  uint64_t& last_key = sh.last_key;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t lo = ~0ull, hi = 0;
#pragma unroll 4
  for (int i = tid; i < n; i += kPickThreads) {
    const uint64_t k = keys[i];
    if (mine && n <= hold) mine[i] = k;
    lo = min(lo, k);
    hi = max(hi, k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, (uint64_t)__shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, (uint64_t)__shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lane == 0) {
    warp_lo[warp] = lo;
    warp_hi[warp] = hi;
  }
  if (tid == 0) few = 0;
  for (int i = tid; i < kPickParts; i += kPickThreads) hist[i] = 0;
  __syncthreads();
  for (int w = 0; w < W; ++w) {
    lo = min(lo, warp_lo[w]);
    hi = max(hi, warp_hi[w]);
  }
  if (mine && n <= hold) keys = mine;
  // Sum over the threads up to this one.
  auto scan = [&](int sum) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    for (int i = 0; i < warp; ++i) sum += warp_sum[i];
    return sum;
  };
  // Taken are the keys with (key >> shift) > top and, of those equal to it, the first `rest`.
  int shift = 0, rest = want;
  uint64_t top = hi;
  const double low = key_score(lo), range = key_score(hi) - low;
  bool done = lo == hi;
  if (!done && range < INFINITY && range > 0.0) {  // (false for NaN)
    const double per = (kPickParts - 0.5) / range;
    // Not falling in the key, whatever is rounded.
    auto part = [&](uint64_t k) {
      return min((int)((key_score(k) - low) * per), kPickParts - 1);
    };
    if (per < INFINITY) {
      for (int i = tid; i < n; i += kPickThreads) atomicAdd(&hist[part(keys[i])], 1);
      __syncthreads();
      // From the greatest part down: thread i has a run of parts that ends at the i-th from above.
      constexpr int RUN = kPickParts / kPickThreads;
      int count = 0;
#pragma unroll
      for (int k = 0; k < RUN; ++k) count += hist[kPickParts - 1 - tid * RUN - k];
      int sum = scan(count);
      if (sum >= want && sum - count < want) {
        sum -= count;
        for (int k = 0; k < RUN; ++k) {
          const int p = kPickParts - 1 - tid * RUN - k, c = hist[p];
          if (sum + c >= want) {
            digit = p;
            left = want - sum;
            break;
          }
          sum += c;
        }
      }
      __syncthreads();
      const int p = digit, c = hist[p];
      if (c <= kPickThreads) {
        for (int i = tid; i < n; i += kPickThreads) {
          const uint64_t k = keys[i];
          if (part(k) == p) {
            const int slot = atomicAdd(&few, 1);
            few_key[slot] = k;
            few_at[slot] = i;
          }
        }
        __syncthreads();
        if (tid < c) {
          const uint64_t k = few_key[tid];
          const int i = few_at[tid];
          int above = 0, same = 0;  // before it
          for (int f = 0; f < c; ++f) {
            above += few_key[f] > k;
            same += few_key[f] == k && few_at[f] < i;
          }
          if (above + same == left - 1) {
            last_key = k;
            warp_eq[0] = same + 1;
          }
        }
        __syncthreads();
        top = last_key;
        rest = warp_eq[0];
        done = true;
        __syncthreads();
      } else {
        __syncthreads();  // all have read hist[p], which the digits start by clearing
      }
    }
  }
  if (!done) {
    // All keys agree above bit `shift`.
    shift = 64 - __clzll((long long)(lo ^ hi));
    top = shift == 64 ? 0 : hi >> shift;
    while (shift > 0) {
      const int wide = min(8, shift), above = shift;
      shift -= wide;
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kPickThreads) {
        const uint64_t k = keys[i];
        if (above == 64 || k >> above == top)
          atomicAdd(&hist[(int)(k >> shift) & ((1 << wide) - 1)], 1);
      }
      __syncthreads();
      // From the greatest digit down: thread i has digit 255 - i.
      const int count = tid < 256 ? hist[255 - tid] : 0, sum = scan(count);
      if (sum >= rest && sum - count < rest) {
        digit = 255 - tid;
        left = rest - (sum - count);
      }
      __syncthreads();
      const bool all = hist[digit] == left;
      top = (above == 64 ? 0 : top << wide) | (uint64_t)digit;
      rest = left;
      __syncthreads();
      if (all) break;
    }
  }
  // In their order, a warp a run of them: first how many there are, then their places.
  const int run = ((n + W - 1) / W + 31) & ~31, first = warp * run, end = min(n, first + run);
  int above = 0, same = 0;
  for (int i0 = first; i0 < end; i0 += 32) {
    const uint64_t k = i0 + lane < end ? keys[i0 + lane] >> shift : 0;
    above += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k > top));
    same += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k == top));
  }
  if (lane == 0) {
    warp_sum[warp] = above;
    warp_eq[warp] = same;
  }
  __syncthreads();
  above = same = 0;
  for (int w = 0; w < warp; ++w) {
    above += warp_sum[w];
    same += warp_eq[w];
  }
  for (int i0 = first; i0 < end; i0 += 32) {
    const uint64_t k = i0 + lane < end ? keys[i0 + lane] >> shift : 0;
    const bool over = i0 + lane < end && k > top, equal = i0 + lane < end && k == top;
    const unsigned ab = __ballot_sync(0xffffffffu, over), eq = __ballot_sync(0xffffffffu, equal);
    const int ab_before = above + __popc(ab & ((1u << lane) - 1));
    const int eq_before = same + __popc(eq & ((1u << lane) - 1));
    if (over || (equal && eq_before < rest))
      out[ab_before + min(eq_before, rest)] = keep_first + i0 + lane;
    above += __popc(ab);
    same += __popc(eq);
  }
}

// A CTA for a token and a KV head whose scores are there.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const BlockArgs a, const int hold) {
  __shared__ PickShared<kPickThreads> sh;
  __shared__ unsigned long long found;
  extern __shared__ uint64_t mine[];
  const int row = blockIdx.x;
  grid_dep_wait();
  const TokenPlace at =
      block_token(a.seqs, a.page_shift, a.token0 + row / a.H, &found, a.index_status);
  int32_t* out = nullptr;
  int n = 0;
  const int want = plain_part(a, at, row, out, n, threadIdx.x, kPickThreads);
  if (want == 0) return;
  pick_block<kPickThreads>(a.keys + (int64_t)row * a.seqs.max_pages + a.keep_first, mine, hold, n,
                           want, a.keep_first, out, sh);
}

// Scores and choice in one: a CTA for a token and a KV head, keys in shared memory.
template <int TB, int NU>
__global__ void __launch_bounds__(kScoreThreads, NU <= 4 ? 4 : NU <= 8 ? 2 : 1)
    select_kernel(const BlockArgs a, const bool vec) {
  __shared__ __align__(16) double parts[NU * 8 * 16 / sizeof(elem_t<TB>)];
  __shared__ union {
    int pages[kScoreMost];
    PickShared<kScoreThreads> pick;
  } sh;
  __shared__ unsigned long long found;
  extern __shared__ uint64_t mine[];
  const int row = blockIdx.x, t = row / a.H, h = row - t * a.H;
  grid_dep_wait();
  query_parts<TB, NU>(a, t, h, parts);
  const TokenPlace at = block_token(a.seqs, a.page_shift, a.token0 + t, &found, a.index_status);
  int32_t* out = nullptr;
  int n = 0;
  const int want = plain_part(a, at, row, out, n, threadIdx.x, kScoreThreads);
  if (want == 0) return;
  for (int from = 0; from < n; from += kScoreMost) {
    if (from > 0) __syncthreads();  // the pages before have been read
    score_blocks<TB, NU>(a, at.b, t, h, a.keep_first + from, a.keep_first + min(n, from + kScoreMost),
                         vec, parts, sh.pages, mine + from);
  }
  __syncthreads();
  if (n > kWarpKeys)
    pick_block<kScoreThreads>(mine, nullptr, 0, n, want, a.keep_first, out, sh.pick);
  else if (threadIdx.x < 32)
    pick_warp(mine, n, want, a.keep_first, out);
}

size_t keys_per_token(int H, int max_pages) { return (size_t)H * std::max(max_pages, 1) * 8; }

}  // namespace

void kv_blocks_bounds_launch(const KvPages& pg, void* bounds, int bounds_type, const SeqTable& sq,
                             int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = pg.Dh % 8 == 0 && reinterpret_cast<uintptr_t>(pg.k) % (4 * elem_bytes(pg.type)) == 0;
  ProfScope prof("kv_blocks", s);
  auto go = [&](auto tc, auto tb) {
    ATTNB_CUDA(launch_pdl(bounds_kernel<decltype(tc)::value, decltype(tb)::value>,
                          dim3(2 * num_sms), dim3(kBoundsThreads), 0, s, pg, bounds, sq, vec,
                          index_status));
  };
  with_value_type(bounds_type, [&](auto tb) {
    if (pg.type == kE4M3) go(std::integral_constant<int, kE4M3>{}, tb);
    else if (pg.type == kI8) go(std::integral_constant<int, kI8>{}, tb);
    else if (pg.type == kI4) go(std::integral_constant<int, kI4>{}, tb);
    else go(tb, tb);
  });
}

size_t kv_blocks_workspace_bytes(int tokens, int H, int max_pages) {
  if (max_pages <= kWarpKeys) return 256;  // keys in shared memory, however many rows there are
  const size_t each = keys_per_token(H, max_pages);
  return std::min<size_t>(each * std::max(tokens, 1), std::max(each, kScoreBytes)) + 256;
}

void kv_blocks_select_run(const RowsView& q, const void* bounds, int num_pages, int H,
                          int page_shift, const SeqTable& sq, int keep_first, int keep_last,
                          int32_t* blocks, int take, void* ws, size_t ws_bytes, int* index_status,
                          int num_sms, cudaStream_t s) {
  BlockArgs a{};
  a.q = q;
  a.bounds = bounds;
  a.seqs = sq;
  a.num_pages = num_pages;
  a.H = H;
  a.G = q.heads / H;
  a.page_shift = page_shift;
  a.keep_first = keep_first;
  a.keep_last = keep_last;
  a.take = take;
  a.blocks = blocks;
  a.index_status = index_status;
  const uintptr_t p = (reinterpret_cast<uintptr_t>(ws) + 255) & ~(uintptr_t)255;
  a.keys = reinterpret_cast<uint64_t*>(p);
  const size_t room = reinterpret_cast<uintptr_t>(ws) + ws_bytes - std::min(p, reinterpret_cast<uintptr_t>(ws) + ws_bytes);
  const bool in_shared = sq.max_pages <= kWarpKeys;
  const size_t held = in_shared ? SIZE_MAX : room / keys_per_token(H, sq.max_pages);  // tokens
  const size_t fit = std::min<size_t>(held, 65535 / H);
  if (fit == 0) fail(ATTNB_ERR_INVALID_ARGUMENT, "workspace too small");
  const int eb = elem_bytes(q.type);
  const bool vec = reinterpret_cast<uintptr_t>(bounds) % 16 == 0 && 2 * q.Dh * eb % 16 == 0;
  ProfScope prof("kv_blocks", s);
  for (a.token0 = 0; a.token0 < sq.total; a.token0 += a.tokens) {
    a.tokens = (int)std::min<size_t>(fit, sq.total - a.token0);
    const int rows = a.tokens * H;
    // f(type, units of 16 bytes a lane).
    auto with_units = [&](auto&& f) {
      with_value_type(q.type, [&](auto tb) {
        constexpr int F = decltype(tb)::value == kF32 ? 2 : 1;
        if (q.Dh <= 64) f(tb, std::integral_constant<int, 2 * F>{});
        else if (q.Dh <= 128) f(tb, std::integral_constant<int, 4 * F>{});
        else f(tb, std::integral_constant<int, 8 * F>{});
      });
    };
    // One CTA a row where rows are short, or so many that they fill the machine; else the
    // blocks of a row are spread over several.  (256 rows of 125-512 blocks 22 us against 25,
    // 1064 rows of 80-310 28 against 41; 4 rows of 4096 88 against 16.)
    if (in_shared || (rows >= 2 * num_sms && sq.max_pages <= kPickKeys)) {
      with_units([&](auto tb, auto nu) {
        ATTNB_CUDA(launch_pdl(select_kernel<decltype(tb)::value, decltype(nu)::value>, dim3(rows),
                              dim3(kScoreThreads), (size_t)sq.max_pages * 8, s, a, vec));
      });
      continue;
    }
    if (sq.max_pages > take) {
      // Four CTAs an SM where there is that much to do.
      const int64_t rounds = (sq.max_pages + kScoreRound - 1) / kScoreRound;
      const int64_t each = (rounds * rows + 4 * num_sms - 1) / (4 * num_sms);
      a.chunk = (int)std::min({rounds, each, (int64_t)kScoreMost / kScoreRound}) * kScoreRound;
      const int chunks = (sq.max_pages + a.chunk - 1) / a.chunk;
      with_units([&](auto tb, auto nu) {
        ATTNB_CUDA(launch_pdl(score_kernel<decltype(tb)::value, decltype(nu)::value>,
                              dim3(chunks, rows), dim3(kScoreThreads), 0, s, a, vec));
      });
    }
    const int hold = std::min(sq.max_pages, kPickKeys);
    ATTNB_CUDA(launch_pdl(pick_kernel, dim3(rows), dim3(kPickThreads), (size_t)hold * 8, s, a, hold));
  }
}

}  // namespace attnb
