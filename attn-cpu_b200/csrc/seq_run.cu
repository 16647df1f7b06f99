// seq_run.cu -- choice of kernel and workspace for attention over ragged
// sequences, and the join of the items that several CTAs shared.
#include <algorithm>
#include <cmath>

#include "runtime.h"
#include "seq.cuh"
#include "seq_elem.cuh"

namespace attnb {
namespace {

constexpr int kMergeThreads = 256;

// Joins the pieces of each item that a cut fell into.  The blocks of all the CTAs
// that go on with an item share its rows (an item of a long context has hundreds
// of pieces, and as many blocks).  Few pieces, the usual case: groups of 128
// threads (one per dimension) take a row each.  Many: the block takes a row, its
// threads find the pieces' weights side by side, and each group sums every
// second piece.
template <int T>
__global__ void __launch_bounds__(kMergeThreads) seq_merge_kernel(const SeqAttnArgs a) {
  using E = elem_t<T>;
  constexpr int kChunk = 256;  // pieces whose weights are held at a time
  __shared__ float weight[kChunk];
  __shared__ float red[kMergeThreads];
  grid_dep_wait();
  const int c = blockIdx.x + 1;
  const SeqSplit d = reinterpret_cast<const SeqSplit*>(a.ws_split)[c];
  if (!d.continues) return;
  const int own = (int)udiv(d.item0, d.quota);  // the CTA with the first piece
  const int last = (int)udiv(d.item1 + d.quota - 1, d.quota) - 1, pieces = last - own + 1;
  // It is that CTA's first piece, or a later one.
  const int slot0 = 2 * own + (d.item0 - d.extra <= own * d.quota ? 0 : 1);
  const int worker = (c - own - 1) * gridDim.y + blockIdx.y, workers = (pieces - 1) * gridDim.y;
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml);
  const int Dh = a.q.Dh, tid = threadIdx.x;
  const int wide = Dh <= 128 ? 128 : 256;  // threads per group
  const int group = tid / wide, groups = kMergeThreads / wide, x = tid % wide;
  auto slot = [&](int i) { return (int64_t)(i == 0 ? slot0 : 2 * (own + i)) * a.rows; };
  if (pieces <= 8) {
      for (int r = worker * groups + group; r < d.rows; r += workers * groups) {
        if (x >= Dh) continue;
        float top = -INFINITY, acc = 0.f, sum = 0.f;
        for (int i = 0; i < pieces; ++i) top = fmaxf(top, ml[slot(i) + r].x);
        for (int i = 0; i < pieces; ++i) {
          const float2 p = ml[slot(i) + r];
          const float f = p.x == -INFINITY ? 0.f : fast_exp2(p.x - top);
          sum = fmaf(f, p.y, sum);
          acc = fmaf(f, a.ws_o[(slot(i) + r) * Dh + x], acc);
        }
        const int row = d.first_row + r;
        E* o = static_cast<E*>(a.o.data) + (int64_t)(d.row_token + row / a.G) * a.o.sT +
               (int64_t)(d.kv_head * a.G + row % a.G) * a.o.sH;
        from_float(sum == 0.f ? 0.f : acc / sum, o[x]);
      }
    return;
  }
  for (int r = worker; r < d.rows; r += workers) {
    float top = -INFINITY;
    for (int i = tid; i < pieces; i += kMergeThreads) top = fmaxf(top, ml[slot(i) + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();  // the row before is done with the shared arrays
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    for (int i = 0; i < kMergeThreads / 32; ++i) top = fmaxf(top, red[i]);
    float acc = 0.f, sum = 0.f;
    for (int i0 = 0; i0 < pieces; i0 += kChunk) {
      const int n = min(kChunk, pieces - i0);
      __syncthreads();
      if (tid < n) {
        const float2 p = ml[slot(i0 + tid) + r];
        const float f = p.x == -INFINITY ? 0.f : fast_exp2(p.x - top);
        weight[tid] = f;
        sum = fmaf(f, p.y, sum);
      }
      __syncthreads();
      if (x < Dh) {
#pragma unroll 8
        for (int i = group; i < n; i += groups)
          acc = fmaf(weight[i], a.ws_o[(slot(i0 + i) + r) * Dh + x], acc);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (group > 0) red[x] = acc;  // two groups at most
    if ((tid & 31) == 0) weight[tid >> 5] = sum;
    __syncthreads();
    if (group == 0 && x < Dh) {
      if (groups > 1) acc += red[x];
      sum = 0.f;
      for (int i = 0; i < kMergeThreads / 32; ++i) sum += weight[i];
      const int row = d.first_row + r;
      E* o = static_cast<E*>(a.o.data) + (int64_t)(d.row_token + row / a.G) * a.o.sT +
             (int64_t)(d.kv_head * a.G + row % a.G) * a.o.sH;
      from_float(sum == 0.f ? 0.f : acc / sum, o[x]);
    }
  }
}

// What a kernel takes from the workspace: two partial results and a SeqSplit
// per CTA.
struct Space {
  int rows, ctas;
  size_t bytes(int Dh) const {
    return (size_t)ctas * (2 * rows * ((size_t)Dh * 4 + 8) + sizeof(SeqSplit)) + 64;
  }
};
Space simt_space(int Dh, int64_t rows, int num_sms) {
  if (Dh > 128) return {2, 2 * num_sms};
  return rows == 1 ? Space{1, 3 * num_sms} : Space{4, 2 * num_sms};
}
// Rows of a KV head in one item: 8 for a step of up to 8 query heads, else 16 (32
// sequences of 4096 bf16 keys: 4 rows 91 us against 94, e4m3 59 against 90; 16
// rows 169 us against 103, e4m3 99 against 98).  Over 4-bit pages at head sizes over 64
// always 8, two CTAs an SM, for want of registers (16 rows the same way 101 us
// against 139).
Space mma_space(int type, int Dh, int64_t rows, int num_sms) {
  const bool large = type == kI4 && Dh > 64;
  if (rows > 8 && !large) return {16, 2 * num_sms};
  return {8, (large ? 2 : 3) * num_sms};
}
Space tc_space(int G, int num_sms) { return {seq_tc_rows(G), num_sms}; }
Space tf32_space(int num_sms) { return {128, num_sms}; }

}  // namespace

size_t seq_workspace_bytes(int G, int Dh, int num_sms) {
  size_t n = std::max({simt_space(Dh, 4, num_sms).bytes(Dh), mma_space(kF16, Dh, 16, num_sms).bytes(Dh),
                       mma_space(kF16, Dh, 8, num_sms).bytes(Dh)});
  if (Dh <= 128) n = std::max(n, tf32_space(num_sms).bytes(Dh));
  if (G <= 128 && Dh <= 128) n = std::max(n, tc_space(G, num_sms).bytes(Dh));
  return n + 256;
}

enum Kind { kSimt, kMma, kTc, kTf32 };

// Kernel, then join of what the cuts between CTAs split.  rows: query rows of a KV head and
// sequence, as far as known.
static void run(SeqAttnArgs a, Kind kind, int64_t rows, uintptr_t ws, uintptr_t ws_end, int num_sms,
                cudaStream_t s) {
  const Space sp = kind == kTc     ? tc_space(a.G, num_sms)
                   : kind == kMma  ? mma_space(a.pages.type, a.q.Dh, rows, num_sms)
                   : kind == kTf32 ? tf32_space(num_sms)
                                   : simt_space(a.q.Dh, rows, num_sms);
  a.rows = sp.rows;
  a.kt_shift = kind == kTc ? 7 : kind == kTf32 ? 5 : kind == kMma ? seq_mma_key_shift(a) : 6;
  a.min_tiles = 2;
  a.extra = kind == kTc || kind == kTf32 ? 2 : 1;
  uintptr_t p = (ws + 255) & ~(uintptr_t)255;
  if (p + sp.bytes(a.q.Dh) > ws_end) fail(ATTNB_ERR_INVALID_ARGUMENT, "workspace too small");
  a.ws_split = reinterpret_cast<void*>(p);
  p += sp.ctas * sizeof(SeqSplit);
  a.ws_ml = reinterpret_cast<float*>(p);
  p += (size_t)2 * sp.ctas * sp.rows * 8;
  a.ws_o = reinterpret_cast<float*>(p);
  {
    ProfScope prof("seq_attn", s);
    if (kind == kTc) seq_tc_launch(a, sp.ctas, s);
    else if (kind == kMma) seq_mma_launch(a, sp.ctas, s);
    else if (kind == kTf32) seq_tf32_launch(a, sp.ctas, s);
    else seq_simt_launch(a, sp.ctas, s);
  }
  with_value_type(a.o.type, [&](auto t) {
    ATTNB_CUDA(launch_pdl(seq_merge_kernel<decltype(t)::value>,
                          dim3(sp.ctas - 1, kind == kTc || kind == kTf32 ? 16 : 2), dim3(kMergeThreads), 0, s,
                          a));
  });
}

void seq_attn_run(SeqAttnArgs a, int max_new, void* ws, size_t ws_bytes, int num_sms,
                  cudaStream_t s) {
  if (a.seqs.batch == 0 || a.seqs.total == 0) return;
  // New tokens of one sequence: the caller's bound, or the mean.
  const int64_t rows =
      (int64_t)(max_new > 0 ? max_new : (a.seqs.total + a.seqs.batch - 1) / a.seqs.batch) * a.G;
  // Rows of one KV head and sequence.  16-bit pages: K7 up to 32 rows, K8 beyond (32
  // sequences of 4096 keys, 8 KV heads of 128: 16 rows 102 us against 193, 32 rows
  // 186 against 184, 48 rows 271 against 189); codes, which K8 converts in four
  // warps: up to 48 (e4m3: 48 rows 267 us against 282, 64 rows 347 against 284; 4 bits:
  // 259 against 306, 337 against 307), 4 bits of head sizes up to 64 up to 96 (64 rows
  // 187 us against 268, 96 rows 269 against 273).  In
  // fp32, K9 over 16 rows (8 sequences of 2000 keys, 4 KV heads of 64: 16 rows 53 us
  // both, 64 rows 62 us against K6's 169).
  const int64_t few = a.pages.type == kI4 && a.q.Dh <= 64 ? 96 : elem_coded(a.pages.type) ? 48 : 32;
  Kind kind = kSimt;
  if (seq_mma_supported(a) && rows <= few) kind = kMma;
  else if (seq_tc_supported(a)) kind = kTc;
  else if (seq_mma_supported(a)) kind = kMma;
  else if (a.q.Dh <= 128 && rows > 16) kind = kTf32;
  const uintptr_t at = reinterpret_cast<uintptr_t>(ws);
  run(a, kind, rows, at, at + ws_bytes, num_sms, s);
}

void seq_attn_blocks_run(SeqAttnArgs a, const int32_t* blocks, int take, void* ws, size_t ws_bytes,
                         int num_sms, cudaStream_t s) {
  if (a.seqs.batch == 0 || a.seqs.total == 0) return;
  // K6 or K7 take any number of rows; a token has few.
  const Kind kind = seq_mma_supported(a) ? kMma : kSimt;
  const int kt = kind == kMma ? seq_mma_key_shift(a) : 6;
  a.sel_blocks = blocks;
  a.sel_take = take;
  a.sel_tiles = (int)((((int64_t)take << a.pages.page_shift) + (1 << kt) - 1) >> kt);
  a.causal = 0;  // a list's keys are those that its token sees
  const uintptr_t at = reinterpret_cast<uintptr_t>(ws);
  run(a, kind, a.G, at, at + ws_bytes, num_sms, s);
}

}  // namespace attnb
