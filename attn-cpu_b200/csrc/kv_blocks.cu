// kv_blocks.cu -- K10: choosing the blocks of a long context that a token attends to.
//
// A block is one page of a sequence.  Its bounds are the least and the greatest
// value of its keys in each dimension, so that for a query q
//     q . k <= sum_d max(q_d least_d, q_d greatest_d)     for every key k of the block.
// The score of a block for a token and a KV head is that bound summed over the query
// heads that read the KV head.  It is linear in the positive and the negative part of
// the queries: with q- = sum over heads of min(q, 0) and q+ = sum of max(q, 0),
//     score = q- . least + q+ . greatest,
// one product of 2 Dh numbers for all heads.  Sums are in 64 bits: products of 16-bit or
// fp32 values and their sum are then off by 2^-53 or so, and which of two blocks is
// better does not hang on the order of a sum.
//
// Three kernels: bounds (of the blocks that new tokens complete), scores (as 64-bit keys
// that sort like the scores), and the choice, a radix selection by digits of 8 bits from
// the top.  Equal scores: the lower block.  A NaN counts as greatest.
#include <algorithm>
#include <cmath>
#include <climits>

#include "runtime.h"
#include "seq_elem.cuh"
#include "seq_pages.cuh"

namespace attnb {
namespace {

constexpr int kBoundsThreads = 256;
constexpr int kScoreThreads = 128;
constexpr int kScoreRound = kScoreThreads / 8 * 2;  // blocks of one round of a CTA of the score kernel
constexpr int kPickThreads = 256;
constexpr int kPickKeys = 4096;  // held in shared memory
constexpr size_t kScoreBytes = 64u << 20;  // workspace for scores, at most (or one token's)

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Tokens that sequence b holds, as far as its table goes.
__device__ __forceinline__ int held(const SeqTable& sq, int page_shift, int b, int* index_status) {
  const int len = __ldg(sq.lens + b);
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
      const int b = b0 + tid, len = held(sq, pg.page_shift, b, index_status);
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

// The block that packed token t lies in, of its sequence b; -1 where there is none.
__device__ __forceinline__ int own_block(const SeqTable& sq, int page_shift, int t, int& b,
                                         int* index_status, int* position = nullptr) {
  int first, count;
  b = seq_of(sq, t, first, count);
  if (b < 0) return -1;
  const int pos = held(sq, page_shift, b, index_status) - count + (t - first);
  if (pos < 0) return -1;
  if (position) *position = pos;
  return pos >> page_shift;
}

// Unsigned numbers that sort as the scores do.
__device__ __forceinline__ uint64_t sort_key(double x) {
  if (x != x) return ~0ull;
  if (x == 0.0) x = 0.0;  // -0 is 0
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Eight lanes a block, each with every eighth unit of 16 bytes of its bounds and the same
// part of the queries' sums in registers.  NU: units a lane.
template <int TB, int NU>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const BlockArgs a, const bool vec) {
  using EB = elem_t<TB>;
  constexpr int PER = 16 / sizeof(EB);
  __shared__ double parts[512];  // q-, q+
  const int tid = threadIdx.x, row = blockIdx.y, t = row / a.H, h = row - t * a.H;
  const int Dh = a.q.Dh;
  grid_dep_wait();
  int b;
  const int own = own_block(a.seqs, a.page_shift, a.token0 + t, b, a.index_status);
  if (own + 1 <= a.take) return;  // all of them
  const int from = a.keep_first + blockIdx.x * a.chunk;
  const int to = min(own + 1 - a.keep_last, from + a.chunk);
  if (from >= to) return;
  for (int d = tid; d < Dh; d += kScoreThreads) {
    const EB* q = static_cast<const EB*>(a.q.data) + (int64_t)(a.token0 + t) * a.q.sT +
                  (int64_t)h * a.G * a.q.sH + d;
    double lo = 0.0, hi = 0.0;
    for (int g = 0; g < a.G; ++g) {
      const float x = to_float(q[g * a.q.sH]);
      // (a NaN goes to both)
      lo += (double)(x > 0.f ? 0.f : x);
      hi += (double)(x < 0.f ? 0.f : x);
    }
    parts[d] = lo;
    parts[Dh + d] = hi;
  }
  __syncthreads();
  const int e = tid & 7;
  double q[NU * PER];
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = (u * 8 + e) * PER + i;
      q[u * PER + i] = d < 2 * Dh ? parts[d] : 0.0;
    }
  const int32_t* table = a.seqs.table + b * a.seqs.table_stride;
  uint64_t* keys = a.keys + (int64_t)row * a.seqs.max_pages;
  // Two blocks a group and round, both on their way before the first is summed.
  for (int j0 = from; j0 < to; j0 += kScoreRound) {
    const EB* p[2];
    uint4 x[2][NU];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = j0 + k * (kScoreRound / 2) + (tid >> 3);
      p[k] = nullptr;
      if (j < to) {
        const int page = __ldg(table + j);
        if (page < 0 || page >= a.num_pages) raise_index(a.index_status);  // bounds of zeros
        else p[k] = static_cast<const EB*>(a.bounds) + ((int64_t)page * a.H + h) * 2 * Dh;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int d = (u * 8 + e) * PER;
        x[k][u] = make_uint4(0, 0, 0, 0);
        if (!p[k] || d >= 2 * Dh) continue;
        if (vec) {  // 2 Dh is a multiple of PER
          x[k][u] = *reinterpret_cast<const uint4*>(p[k] + d);
        } else {
          EB* v = reinterpret_cast<EB*>(&x[k][u]);
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (d + i < 2 * Dh) v[i] = p[k][d + i];
        }
      }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      double s = 0.0;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const EB* v = reinterpret_cast<const EB*>(&x[k][u]);
#pragma unroll
        for (int i = 0; i < PER; ++i) s = fma(q[u * PER + i], (double)to_float(v[i]), s);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const int j = j0 + k * (kScoreRound / 2) + (tid >> 3);
      if (e == 0 && j < to) keys[j] = sort_key(s);
    }
  }
}

// ------------------------------------------------------------------ choice
// One CTA for a token and a KV head.  Keys of up to kPickKeys blocks are read once.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const BlockArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sum[kPickThreads / 32];
  __shared__ uint64_t warp_lo[kPickThreads / 32], warp_hi[kPickThreads / 32];
  __shared__ int digit, left;
  __shared__ uint64_t mine[kPickKeys];
  const int tid = threadIdx.x, row = blockIdx.x, t = row / a.H, h = row - t * a.H;
  const int lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  int b;
  const int own = own_block(a.seqs, a.page_shift, a.token0 + t, b, a.index_status);
  if (b < 0) return;  // rows of no sequence stay
  int32_t* out = a.blocks + ((int64_t)(a.token0 + t) * a.H + h) * a.take;
  if (own + 1 <= a.take) {
    for (int i = tid; i < a.take; i += kPickThreads) out[i] = i <= own ? i : -1;
    return;
  }
  const uint64_t* keys = a.keys + (int64_t)row * a.seqs.max_pages + a.keep_first;
  const int n = own + 1 - a.keep_first - a.keep_last;
  const int want = a.take - a.keep_first - a.keep_last;  // < n
  for (int i = tid; i < a.keep_first; i += kPickThreads) out[i] = i;
  for (int i = tid; i < a.keep_last; i += kPickThreads)
    out[a.take - a.keep_last + i] = own + 1 - a.keep_last + i;
  if (want == 0) return;
  // The first bit in which they differ: digits start there.
  uint64_t lo = ~0ull, hi = 0;
#pragma unroll 4
  for (int i = tid; i < n; i += kPickThreads) {
    const uint64_t k = keys[i];
    if (n <= kPickKeys) mine[i] = k;
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
  __syncthreads();
  for (int w = 0; w < kPickThreads / 32; ++w) {
    lo = min(lo, warp_lo[w]);
    hi = max(hi, warp_hi[w]);
  }
  if (n <= kPickKeys) keys = mine;
  // The top digits of the last one taken, until as many keys have them as are wanted.  All keys
  // agree above bit `bits`.
  int bits = 64 - (lo == hi ? 64 : __clzll((long long)(lo ^ hi))), shift = bits;
  uint64_t top = bits == 64 ? 0 : hi >> bits;
  int rest = want;
  while (shift > 0) {
    const int wide = min(8, shift), above = shift;
    shift -= wide;
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPickThreads) {
      const uint64_t k = keys[i];
      if (above == 64 || k >> above == top)
        atomicAdd(&hist[(int)(k >> shift) & ((1 << wide) - 1)], 1);
    }
    __syncthreads();
    // Sums from the greatest digit down: thread i has digit 255 - i.
    const int count = hist[255 - tid];
    int sum = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    for (int i = 0; i < warp; ++i) sum += warp_sum[i];
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
  // Those above, and the first `rest` of those with the same digits, in their order.
  int taken = 0, same = 0;  // before this round
  for (int i0 = 0; i0 < n; i0 += kPickThreads) {
    const int i = i0 + tid;
    const uint64_t k = i < n ? keys[i] >> shift : 0;
    const bool above = i < n && k > top, equal = i < n && k == top;
    const unsigned eq = __ballot_sync(0xffffffffu, equal), ab = __ballot_sync(0xffffffffu, above);
    if (lane == 0) warp_sum[warp] = __popc(eq) | __popc(ab) << 16;
    __syncthreads();
    int eq_before = same + __popc(eq & ((1u << lane) - 1)), ab_before = __popc(ab & ((1u << lane) - 1));
    int eq_all = 0, ab_all = 0;
    for (int w = 0; w < kPickThreads / 32; ++w) {
      const int s = warp_sum[w];
      if (w < warp) {
        eq_before += s & 0xffff;
        ab_before += s >> 16;
      }
      eq_all += s & 0xffff;
      ab_all += s >> 16;
    }
    if (above || (equal && eq_before < rest))
      out[a.keep_first + taken + ab_before + min(eq_before, rest) - min(same, rest)] =
          a.keep_first + i;
    taken += ab_all + min(same + eq_all, rest) - min(same, rest);
    same += eq_all;
    __syncthreads();
  }
}

// ------------------------------------------------ lists to pages, for the attention
// A warp for a token and a KV head: its list up to the first entry that is not above the
// one before it or lies behind the token's own block, as page numbers, and how many keys
// these hold for it.
__global__ void __launch_bounds__(256)
    lists_kernel(const SeqTable sq, const KvPages pg, const int32_t* blocks, int take, int32_t* pages,
                 int32_t* lens, int* index_status) {
  const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  grid_dep_wait();
  if (row >= sq.total * pg.H) return;
  int b, pos = 0;
  const int own = own_block(sq, pg.page_shift, row / pg.H, b, index_status, &pos);
  if (b < 0) {
    if (lane == 0) lens[row] = -1;
    return;
  }
  const int32_t* list = blocks + (int64_t)row * take;
  int last = -1, count = 0;
  for (int i0 = 0; own >= 0 && i0 < take; i0 += 32) {
    const int mine = i0 + lane < take ? __ldg(list + i0 + lane) : -1;
    int prior = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == 0) prior = last;
    const bool good = mine > prior && mine <= own;
    const unsigned bad = __ballot_sync(0xffffffffu, !good);
    const int n = bad ? __ffs(bad) - 1 : 32;
    if (lane < n) {
      const int page = seq_page(sq, pg, b, mine << pg.page_shift, index_status);
      pages[(int64_t)row * take + i0 + lane] = page;
    }
    count += n;
    if (n > 0) last = __shfl_sync(0xffffffffu, mine, n - 1);
    if (n < 32) {
      if (lane == n && i0 + lane < take && mine != -1) raise_index(index_status);
      break;
    }
  }
  if (lane == 0)
    lens[row] = (count << pg.page_shift) -
                (last == own && count > 0 ? (1 << pg.page_shift) - 1 - (pos & ((1 << pg.page_shift) - 1))
                                          : 0);
}

size_t keys_per_token(int H, int max_pages) { return (size_t)H * std::max(max_pages, 1) * 8; }

}  // namespace

void kv_blocks_bounds_launch(const KvPages& pg, void* bounds, int bounds_type, const SeqTable& sq,
                             int* index_status, int num_sms, cudaStream_t s) {
  const bool vec = pg.Dh % 8 == 0 && reinterpret_cast<uintptr_t>(pg.k) % (4 * elem_bytes(pg.type)) == 0;
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
  const size_t fit = std::min<size_t>(room / keys_per_token(H, sq.max_pages), 65535 / H);
  if (fit == 0) fail(ATTNB_ERR_INVALID_ARGUMENT, "workspace too small");
  const int eb = elem_bytes(q.type);
  const bool vec = reinterpret_cast<uintptr_t>(bounds) % 16 == 0 && 2 * q.Dh * eb % 16 == 0;
  for (a.token0 = 0; a.token0 < sq.total; a.token0 += a.tokens) {
    a.tokens = (int)std::min<size_t>(fit, sq.total - a.token0);
    if (sq.max_pages > take) {
      // Four CTAs an SM where there is that much to do.
      const int64_t rounds = (sq.max_pages + kScoreRound - 1) / kScoreRound;
      const int64_t each = std::max<int64_t>(1, rounds * a.tokens * H / (4 * num_sms));
      a.chunk = (int)std::min(rounds, each) * kScoreRound;
      const int chunks = (sq.max_pages + a.chunk - 1) / a.chunk;
      with_value_type(q.type, [&](auto tb) {
        constexpr int TB = decltype(tb)::value;
        constexpr int F = TB == kF32 ? 2 : 1;
        auto go = [&](auto nu) {
          ATTNB_CUDA(launch_pdl(score_kernel<TB, decltype(nu)::value>, dim3(chunks, a.tokens * H),
                                dim3(kScoreThreads), 0, s, a, vec));
        };
        if (q.Dh <= 64) go(std::integral_constant<int, 2 * F>{});
        else if (q.Dh <= 128) go(std::integral_constant<int, 4 * F>{});
        else go(std::integral_constant<int, 8 * F>{});
      });
    }
    ATTNB_CUDA(launch_pdl(pick_kernel, dim3(a.tokens * H), dim3(kPickThreads), 0, s, a));
  }
}

void kv_blocks_lists_launch(const SeqTable& sq, const KvPages& pg, const int32_t* blocks, int take,
                            int32_t* pages, int32_t* lens, int* index_status, cudaStream_t s) {
  const int rows = sq.total * pg.H;
  ATTNB_CUDA(launch_pdl(lists_kernel, dim3((rows + 7) / 8), dim3(256), 0, s, sq, pg, blocks, take,
                        pages, lens, index_status));
}

}  // namespace attnb
