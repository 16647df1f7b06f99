// seq.cuh -- the schedule of the attention kernels over ragged sequences (K6-K9)
// and what they share: bounds of a sequence, the split of all work over the
// CTAs, and the places of partial results.
//
// An item is one KV head of one sequence and up to `rows` of its query rows.
// Row r of a sequence's n * G rows is token r / G, query head (kv head) * G +
// r % G: the query heads that read one KV head lie side by side, so each key is
// read once for all of them.  An item takes the key tiles that its last row
// sees, at least one (a row without keys is written too).  All items' tiles,
// in the order (sequence, KV head, item), form one line that is cut into equal
// pieces, one for each CTA: ragged batches, causal triangles and single long
// contexts all load the CTAs evenly, and nothing about the lengths has to be
// known on the host.  An item counts `extra` tiles more than it has, ahead of
// its first, for what it costs besides (its queries, its output).  An item that a cut falls into is joined afterwards
// (seq_run.cu) from the pieces' running maximum, sum and accumulator; a CTA
// has at most two such pieces, its first and its last, so the workspace does
// not grow with the batch.
//
// Attention to selected blocks runs on the same line, with a "sequence" for each
// token and KV head: the keys of the blocks in its list, one block after the other.  These
// are many and much the same,
// so that each counts for as many tiles as the longest may have: a CTA finds its
// place by one division, where the sum over their own lengths would cost more than
// it evens out.
//
// Lengths and page numbers come from device memory and are clamped here, so
// that wrong ones lead to no access out of range.
#pragma once
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace attnb {

struct SeqInfo {
  int q0, n;   // first query row (packed token) and their count
  int k0, L;   // first packed key (packed keys only) and number of keys
};

// One CTA's first piece, for the merge.
struct SeqSplit {
  long long item0, item1;  // the item's own tiles on the line
  long long quota;         // tiles per CTA
  int extra;
  int row_token, rows;     // the item's first row is row `first_row` of its sequence
  int first_row, kv_head;
  int continues;           // the piece is not the item's first
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Every writer stores the same value.
__device__ __forceinline__ void raise_index(int* index_status) {
  *reinterpret_cast<volatile int*>(index_status) = 1;
  __threadfence_system();
}

// The rows of sequence b among `total` packed ones.
__device__ __forceinline__ void seq_rows(const int32_t* cu, int b, int total, int& first,
                                         int& count) {
  first = clampi(__ldg(cu + b), 0, total);
  count = clampi(__ldg(cu + b + 1), first, total) - first;
}

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

__device__ __forceinline__ SeqInfo seq_info(const SeqAttnArgs& a, int b) {
  SeqInfo i;
  seq_rows(a.seqs.cu, b, a.seqs.total, i.q0, i.n);
  if (a.pages.k) {
    const int len = __ldg(a.seqs.lens + b);
    const long long room = (long long)a.seqs.max_pages << a.pages.page_shift;
    i.L = (int)min((long long)max(len, 0), room);
    if (len < 0 || len > room) raise_index(a.index_status);
    i.k0 = 0;
  } else {
    seq_rows(a.cu_k, b, a.k.tokens, i.k0, i.L);
  }
  return i;
}

// a / b, in 32 bits where they suffice (a 64-bit division costs several times
// one in 32 bits).
__device__ __forceinline__ unsigned long long udiv(unsigned long long a, unsigned long long b) {
  if (((a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
  return a / b;
}

// sum_{i=0}^{n-1} floor((A * i + B) / M), by Euclid's steps on (A, M).
__device__ __forceinline__ long long floor_sum(unsigned long long n, unsigned long long M,
                                               unsigned long long A, unsigned long long B) {
  unsigned long long s = 0;
  while (n > 0) {
    if (A >= M) {
      const unsigned long long d = udiv(A, M);
      s += (n - 1) * n / 2 * d;
      A -= d * M;
    }
    if (B >= M) {
      const unsigned long long d = udiv(B, M);
      s += n * d;
      B -= d * M;
    }
    const unsigned long long top = A * n + B;
    if (top < M) break;
    n = udiv(top, M);
    B = top - n * M;
    const unsigned long long t = M;
    M = A;
    A = t;
  }
  return (long long)s;
}

// Items of one KV head of a sequence.
__device__ __forceinline__ int seq_items(const SeqAttnArgs& a, const SeqInfo& i) {
  return (int)(((unsigned)i.n * a.G + a.rows - 1) / (unsigned)a.rows);  // n * G < 2^30 (host)
}

// Number of keys that the last row of item m sees (<= 0: none).
__device__ __forceinline__ int seq_seen(const SeqAttnArgs& a, const SeqInfo& i, int m) {
  if (!a.causal) return i.L;
  const int end = min(i.n * a.G, (m + 1) * a.rows);
  return i.L - i.n + (end - 1) / a.G + 1;
}

__device__ __forceinline__ int seq_tiles(const SeqAttnArgs& a, const SeqInfo& i, int m) {
  const int seen = seq_seen(a, i, m);
  return max(1, (int)(((long long)max(seen, 0) + (1 << a.kt_shift) - 1) >> a.kt_shift));
}

// Tiles on the line of the items before item m (m <= items) of one KV head.
__device__ __forceinline__ long long seq_own_tiles_before(const SeqAttnArgs& a, const SeqInfo& i,
                                                      int m) {
  if (m <= 0) return 0;
  const int M = seq_items(a, i);
  const long long full =
      max(1ll, ((long long)i.L + (1 << a.kt_shift) - 1) >> a.kt_shift);  // an item that sees all
  if (!a.causal) return full * m;
  long long s = 0;
  int whole = m;
  if (m == M) {  // the last item sees every key
    s = full;
    whole = M - 1;
  }
  // Item k < M - 1 ends with row (k+1) * rows - 1 and takes
  // floor((G * (L - n + kt) + (k+1) * rows - 1) / (G * kt)) tiles, or 1.
  const long long kt = 1ll << a.kt_shift, GK = a.G * kt;
  const long long c = a.G * ((long long)i.L - i.n + kt) + a.rows - 1;
  const long long ones = c >= 2 * GK ? 0 : min((long long)whole, (long long)udiv(2 * GK - c + a.rows - 1, a.rows));
  s += ones;
  if (whole > ones) s += floor_sum(whole - ones, GK, a.rows, c + ones * a.rows);
  return s;
}

__device__ __forceinline__ long long seq_tiles_before(const SeqAttnArgs& a, const SeqInfo& i,
                                                      int m) {
  return seq_own_tiles_before(a, i, m) + (long long)a.extra * max(m, 0);
}

// Where a CTA stands on the line.
struct SeqPlace {
  long long t0, t1, quota;
  long long item0;  // the place of the item that t0 lies in
  int b, h, m, j;   // the item, and how far into it t0 is
};

// Sum over the block (all threads, blockDim.x a multiple of 32); excl: of the
// threads before this one.
__device__ __forceinline__ long long block_scan(long long v, long long& excl, long long* warps) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // `warps` may still be read from the scan before
  if (lane == 31) warps[w] = x;
  __syncthreads();
  long long before = 0, total = 0;
  for (int i = 0; i < nw; ++i) {
    const long long s = warps[i];
    if (i < w) before += s;
    total += s;
  }
  excl = before + x - v;
  return total;
}

struct SeqShared {
  long long warps[32];
  long long rest;
  int b, m;
};

// Items of a KV head, and tiles that one of them counts for, with selected blocks.
__device__ __forceinline__ int sel_items(const SeqAttnArgs& a) {
  return (a.G + a.rows - 1) / a.rows;
}
__device__ __forceinline__ int sel_span(const SeqAttnArgs& a) { return a.sel_tiles + a.extra; }

// What a token and KV head (row v of the lists) attend to.
struct SelRow {
  int b, L;  // sequence (-1: a row of none) and number of keys
};

// All lanes of a warp call.  The list ends at its first entry that is not above the one
// before it or lies behind the token's own block; any but -1 there is told.
__device__ __forceinline__ SelRow sel_row(const SeqAttnArgs& a, int v) {
  const int lane = threadIdx.x & 31, t = v / a.pages.H, shift = a.pages.page_shift;
  // The first entries of the list are on their way while the token's sequence is found.
  const int32_t* list = a.sel_blocks + (int64_t)v * a.sel_take;
  int mine = lane < a.sel_take ? __ldg(list + lane) : -1;
  SelRow r{-1, 0};
  int first = 0, count = 0;
  if (a.seqs.batch <= 64) {  // two sequences a lane at most, all at once
    for (int b0 = 0; b0 < a.seqs.batch && r.b < 0; b0 += 32) {
      int f = 0, c = 0;
      if (b0 + lane < a.seqs.batch) seq_rows(a.seqs.cu, b0 + lane, a.seqs.total, f, c);
      const unsigned hit = __ballot_sync(0xffffffffu, t >= f && t < f + c);
      if (hit) {
        const int src = __ffs(hit) - 1;
        r.b = b0 + src;
        first = __shfl_sync(0xffffffffu, f, src);
        count = __shfl_sync(0xffffffffu, c, src);
      }
    }
  } else {
    r.b = seq_of(a.seqs, t, first, count);
  }
  if (r.b < 0) return r;
  const int len = __ldg(a.seqs.lens + r.b);
  const long long room = (long long)a.seqs.max_pages << shift;
  if (len < 0 || len > room) raise_index(a.index_status);
  const int pos = (int)min((long long)max(len, 0), room) - count + (t - first);
  if (pos < 0) return r;
  const int own = pos >> shift;
  int last = -1, blocks = 0;
  for (int i0 = 0;; ) {
    int prior = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == 0) prior = last;
    const unsigned bad = __ballot_sync(0xffffffffu, !(mine > prior && mine <= own));
    const int n = bad ? __ffs(bad) - 1 : 32;
    blocks += n;
    if (n > 0) last = __shfl_sync(0xffffffffu, mine, n - 1);
    if (n < 32) {
      if (lane == n && i0 + lane < a.sel_take && mine != -1) raise_index(a.index_status);
      break;
    }
    i0 += 32;
    if (i0 >= a.sel_take) break;
    mine = i0 + lane < a.sel_take ? __ldg(list + i0 + lane) : -1;
  }
  r.L = blocks << shift;
  if (blocks > 0 && last == own) r.L -= (1 << shift) - 1 - (pos & ((1 << shift) - 1));
  return r;
}

// All threads of the block; false when the CTA has nothing to do.  SEL here and below: in a
// kernel that selected blocks may come to (K6 and K7 have two forms: their code costs steps over
// all keys 5 us of 61).
template <bool SEL = false>
__device__ inline bool seq_locate(const SeqAttnArgs& a, SeqShared& sh, SeqPlace& p) {
  if (SEL && a.sel_blocks) {
    const int M = sel_items(a), span = sel_span(a);
    const long long total = (long long)a.seqs.total * a.pages.H * M * span;
    p.quota = max((long long)a.min_tiles, (long long)udiv(total + gridDim.x - 1, gridDim.x));
    p.t0 = p.quota * blockIdx.x;
    p.t1 = min(total, p.t0 + p.quota);
    __syncthreads();  // as below: what was set up is seen
    if (p.t0 >= total) return false;
    const long long item = (long long)udiv(p.t0, span);
    p.b = (int)udiv(item, M);
    p.m = (int)(item - (long long)p.b * M);
    p.h = p.b % a.pages.H;
    p.item0 = item * span;
    p.j = (int)(p.t0 - p.item0);
    return true;
  }
  const int tid = threadIdx.x, nt = blockDim.x, batch = a.seqs.batch;
  auto weight = [&](int b) -> long long {
    if (b >= batch) return 0;
    const SeqInfo i = seq_info(a, b);
    return a.pages.H * seq_tiles_before(a, i, seq_items(a, i));
  };
  long long total = 0, excl = 0, w = 0;
  if (batch <= nt) {
    w = weight(tid);
    total = block_scan(w, excl, sh.warps);
  } else {
    long long mine = 0;
    for (int b = tid; b < batch; b += nt) mine += weight(b);
    long long e;
    total = block_scan(mine, e, sh.warps);
  }
  p.quota = max((long long)a.min_tiles, (long long)udiv(total + gridDim.x - 1, gridDim.x));
  p.t0 = p.quota * blockIdx.x;
  p.t1 = min(total, p.t0 + p.quota);
  if (p.t0 >= total) return false;  // the same for every thread
  if (batch <= nt) {
    if (excl <= p.t0 && p.t0 < excl + w) {
      sh.b = tid;
      sh.rest = p.t0 - excl;
    }
  } else {
    long long base = 0;
    for (int b0 = 0; b0 < batch; b0 += nt) {
      w = weight(b0 + tid);
      const long long t = block_scan(w, excl, sh.warps);
      if (base + excl <= p.t0 && p.t0 < base + excl + w) {
        sh.b = b0 + tid;
        sh.rest = p.t0 - (base + excl);
      }
      base += t;
      if (base > p.t0) break;
    }
  }
  if (tid == 0) sh.m = 0;
  __syncthreads();
  p.b = sh.b;
  const SeqInfo i = seq_info(a, p.b);
  const int M = seq_items(a, i);
  const long long per_head = seq_tiles_before(a, i, M);
  p.h = (int)udiv(sh.rest, per_head);
  const long long r = sh.rest - p.h * per_head;
  // The last item that starts at or before tile r: each round, every thread
  // tries one candidate.
  for (int span = M; span > 1;) {
    const int step = (span + nt - 1) / nt;
    const int from = sh.m;
    __syncthreads();
    const int m = from + tid * step;
    if (tid * step < span && m < M && seq_tiles_before(a, i, m) <= r) atomicMax(&sh.m, m);
    __syncthreads();
    span = step;
  }
  p.m = sh.m;
  const long long start = seq_tiles_before(a, i, p.m);
  p.j = (int)(r - start);
  p.item0 = p.t0 - p.j;
  __syncthreads();
  return true;
}

// One piece: tiles [j0, j1) of item (b, h, m), which has nt.
struct SeqPiece {
  SeqInfo s;
  int b, h, m, j0, j1, nt;
  int row0, rows;  // its rows [row0, row0 + rows) of the sequence's n * G
  int v;           // selected blocks: row of the lists
  bool head;       // of the item that the CTA's first tile lies in
};

// Steps through a CTA's pieces; every role of a kernel runs one of its own.
template <bool SEL>
struct SeqIterOf {
  long long t, t1;
  int b, h, m, j;
  bool fresh, head;
  SeqInfo s;
  int items;
  __device__ __forceinline__ void start(const SeqPlace& p) {
    t = p.t0;
    t1 = p.t1;
    b = p.b;
    h = p.h;
    m = p.m;
    j = p.j;
    fresh = head = true;
  }
  __device__ __forceinline__ bool next(const SeqAttnArgs& a, SeqPiece& w) {
    if (SEL && a.sel_blocks) return next_selected(a, w);
    while (t < t1) {
      if (fresh) {
        s = seq_info(a, b);
        items = seq_items(a, s);
        fresh = false;
      }
      w.s = s;
      w.b = b;
      w.h = h;
      w.m = m;
      w.nt = seq_tiles(a, s, m);
      const int end = (int)min((long long)w.nt + a.extra, j + (t1 - t));
      w.j0 = max(0, j - a.extra);
      w.j1 = max(0, end - a.extra);
      w.row0 = m * a.rows;
      w.rows = min(a.rows, s.n * a.G - w.row0);
      w.head = head;
      head = false;
      t += end - j;
      j = 0;
      if (++m == items) {
        m = 0;
        if (++h == a.pages.H) {
          h = 0;
          // The next sequence that has rows.
          while (t < t1 && ++b < a.seqs.batch) {
            s = seq_info(a, b);
            items = seq_items(a, s);
            if (items > 0) break;
          }
        }
      }
      if (w.j1 > w.j0) return true;  // the cut may leave an item's extra alone
    }
    return false;
  }
  __device__ __forceinline__ bool next_selected(const SeqAttnArgs& a, SeqPiece& w) {
    const int span = sel_span(a), M = sel_items(a);
    while (t < t1) {
      const SelRow r = sel_row(a, b);
      w.s = SeqInfo{b / a.pages.H, r.b >= 0 ? 1 : 0, 0, r.L};
      w.b = r.b;
      w.v = b;
      w.h = h;
      w.m = m;
      w.nt = seq_tiles(a, w.s, m);
      const int end = (int)min((long long)span, j + (t1 - t));
      w.j0 = max(0, j - a.extra);
      w.j1 = w.s.n ? min(w.nt, end - a.extra) : 0;
      w.row0 = m * a.rows;
      w.rows = min(a.rows, a.G - w.row0);
      w.head = head;
      head = false;
      t += end - j;
      j = 0;
      if (++m == M) {
        m = 0;
        ++b;
        if (++h == a.pages.H) h = 0;
      }
      if (w.j1 > w.j0) return true;
    }
    return false;
  }
};

using SeqIter = SeqIterOf<false>;

// Number of keys that row r (of the sequence's n * G) sees.
__device__ __forceinline__ int seq_row_seen(const SeqAttnArgs& a, const SeqInfo& s, int r) {
  return a.causal ? s.L - s.n + r / a.G + 1 : s.L;
}

// Which partial a piece writes (-1: none, it is a whole item): one of the item that
// the CTA's first tile lies in goes to its slot 0, a later one to slot 1.
__device__ __forceinline__ int seq_slot(const SeqPiece& w) {
  return w.j0 == 0 && w.j1 == w.nt ? -1 : 2 * (int)blockIdx.x + (w.head ? 0 : 1);
}

// The first warp of every CTA, those without work included.
template <bool SEL = false>
__device__ __forceinline__ void seq_write_split(const SeqAttnArgs& a, bool any,
                                                const SeqPlace& p) {
  SeqSplit d{};
  d.extra = a.extra;
  if (any && p.j > a.extra) {
    SeqInfo s;
    if (SEL && a.sel_blocks) {
      const SelRow r = sel_row(a, p.b);
      s = SeqInfo{p.b / a.pages.H, r.b >= 0 ? 1 : 0, 0, r.L};
    } else {
      s = seq_info(a, p.b);
    }
    d.item0 = p.item0 + a.extra;
    d.item1 = d.item0 + seq_tiles(a, s, p.m);
    d.continues = s.n > 0 && p.t0 < d.item1;
    d.quota = p.quota;
    d.first_row = p.m * a.rows;
    d.rows = min(a.rows, s.n * a.G - d.first_row);
    d.row_token = s.q0;
    d.kv_head = p.h;
  }
  if (threadIdx.x == 0) reinterpret_cast<SeqSplit*>(a.ws_split)[blockIdx.x] = d;
}

// The slot in its sequence's table that slot `i` of the piece's keys is.
__device__ __forceinline__ int piece_slot(const SeqAttnArgs& a, const SeqPiece& w, int i) {
  return a.sel_blocks ? __ldg(a.sel_blocks + (int64_t)w.v * a.sel_take + i) : i;
}

// The page that holds position `pos` of sequence b, or -1.
__device__ __forceinline__ int seq_page(const SeqTable& sq, const KvPages& pg, int b, int pos,
                                        int* index_status) {
  const int slot = pos >> pg.page_shift;
  if (slot >= sq.max_pages) return -1;
  const int page = __ldg(sq.table + b * sq.table_stride + slot);
  if (page < 0 || page >= pg.num_pages) {
    raise_index(index_status);
    return -1;
  }
  return page;
}

}  // namespace attnb
