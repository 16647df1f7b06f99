// capi_seq.cu -- the C ABI of the operators over ragged sequences and paged KV
// caches (include/attnb.h): validation and dispatch.
#include <algorithm>
#include <cmath>
#include <string>

#include "entry.h"
#include "kernels.h"
#include "runtime.h"

using namespace attnb;

namespace {

constexpr int kMaxDh = 256;
constexpr float kLog2e = 1.44269504f;

void invalid(const std::string& msg) { fail(ATTNB_ERR_INVALID_ARGUMENT, msg); }

bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

void check_rows(const attnb_rows* r, const char* name, bool output) {
  const std::string n(name);
  if (!r) invalid("Null " + n + " descriptor");
  if (r->type != ATTNB_TYPE_F32 && r->type != ATTNB_TYPE_BF16 && r->type != ATTNB_TYPE_F16)
    invalid(n + " must be F32, BF16 or F16");
  if (r->tokens < 0) invalid(n + " has a negative number of tokens");
  if (r->heads <= 0 || r->Dh <= 0 || r->Dh > kMaxDh)
    invalid(n + " has invalid heads/Dh (Dh in [1, 256])");
  if (r->tokens > 0 && !r->data) invalid("Null data pointer (" + n + ")");
  if (reinterpret_cast<uintptr_t>(r->data) % elem_bytes(r->type) != 0)
    invalid(n + " is not aligned to its elements");
  if (output) {
    // One of the two strides steps over whole extents of the other.
    const int64_t t = std::llabs(r->strideT), h = std::llabs(r->strideH);
    const bool heads_inside = (r->heads == 1 || h >= r->Dh) &&
                              (r->tokens <= 1 || t >= (r->heads - 1) * h + r->Dh);
    const bool tokens_inside = (r->tokens <= 1 || t >= r->Dh) &&
                               (r->heads == 1 || h >= (r->tokens - 1) * t + r->Dh);
    if (!heads_inside && !tokens_inside) invalid(n + " has rows that overlap");
  }
}

RowsView rows(const attnb_rows* r) {
  return RowsView{r->data, r->type, r->tokens, r->heads, r->Dh, r->strideT, r->strideH};
}

int page_shift_of(int page_size) {
  int shift = 4;
  while (shift <= 7 && (1 << shift) != page_size) ++shift;
  if (shift > 7) invalid("page_size must be 16, 32, 64 or 128");
  return shift;
}

// keys_only: v and what belongs to it is not looked at.
KvPages pages_of(const attnb_kv_pages* p, int row_type, bool keys_only = false) {
  if (!p) invalid("Null pages descriptor");
  if (p->type != ATTNB_TYPE_I4 && (p->type < ATTNB_TYPE_F32 || p->type > ATTNB_TYPE_I8))
    invalid("unknown page type");
  if (p->num_pages < 0 || p->H <= 0 || p->Dh <= 0 || p->Dh > kMaxDh)
    invalid("pages have an invalid number, H or Dh (Dh in [1, 256])");
  const int shift = page_shift_of(p->page_size);
  const bool i4 = p->type == ATTNB_TYPE_I4;
  void* const v = keys_only ? p->k : p->v;
  float* const v_scale = keys_only ? p->k_scale : p->v_scale;
  uint8_t* const v_group = keys_only || !i4 ? nullptr : p->v_group;
  if (!p->k || !v) invalid("Null page pointer");
  if (!elem_coded(p->type) && p->type != row_type)
    invalid("pages must have the rows' type or be E4M3 or I8 or I4");
  if (reinterpret_cast<uintptr_t>(p->k) % elem_bytes(p->type) != 0 ||
      reinterpret_cast<uintptr_t>(v) % elem_bytes(p->type) != 0)
    invalid("pages are not aligned to their elements");
  if (elem_coded(p->type) && (!p->k_scale || !v_scale))
    invalid("E4M3 and I8 pages need scales, and so do I4 pages");
  if (!aligned4(p->k_scale) || !aligned4(v_scale))
    invalid("scales are not aligned to their elements");
  if (!elem_coded(p->type) && (p->k_scale || v_scale))
    invalid("only E4M3 and I8 pages have scales, and I4 pages");
  if (i4) {
    if (p->Dh % kI4Group != 0) invalid("I4 pages need a Dh that is a multiple of 32");
    if (!p->k_group || (!keys_only && !v_group)) invalid("I4 pages need k_group and v_group");
    if (!aligned4(p->k) || !aligned4(v) || !aligned4(p->k_group) || !aligned4(v_group))
      invalid("I4 pages and factors must start on 4-byte boundaries");
  }
  return KvPages{p->k,         v,     p->k_scale, v_scale, p->type,
                 p->num_pages, p->H,  shift,      p->Dh,   i4 ? p->k_group : nullptr,
                 v_group};
}

SeqTable seqs_of(const attnb_seqs* q, int total) {
  if (!q) invalid("Null sequences descriptor");
  if (q->batch < 0) invalid("batch must be non-negative");
  if (q->max_pages < 0) invalid("max_pages must be non-negative");
  if (q->batch > 0 && (!q->cu || !q->lens || (q->max_pages > 0 && !q->table)))
    invalid("Null cu, lens or table");
  if (!aligned4(q->cu) || !aligned4(q->lens) || !aligned4(q->table))
    invalid("cu, lens or table is not aligned to its elements");
  if (q->batch > 1 && q->table_stride < 0) invalid("table_stride must be non-negative");
  return SeqTable{q->cu, q->batch, total, q->table, q->table_stride, q->max_pages, q->lens};
}

void check_heads(const attnb_rows* Q, const attnb_rows* O, int kv_heads, int kv_dh) {
  if (O->type != Q->type) invalid("O must have Q's type");
  if (O->tokens != Q->tokens || O->heads != Q->heads || O->Dh != Q->Dh)
    invalid("O must be [tokens, heads, Dh] matching Q");
  if (kv_dh != Q->Dh) invalid("Dh mismatch");
  if (Q->heads % kv_heads != 0) invalid("Q heads must be a multiple of the KV heads");
  if ((int64_t)Q->tokens * (Q->heads / kv_heads) >= (1 << 30))
    invalid("tokens times query heads per KV head must be below 2^30");
}

// K and V rows for these pages.
void check_kv(const attnb_rows* K, const attnb_rows* V, const KvPages& pg) {
  if (K->heads != pg.H || K->Dh != pg.Dh || V->heads != pg.H || V->Dh != pg.Dh ||
      V->tokens != K->tokens)
    invalid("K and V must be [tokens, H, Dh] matching the pages");
}

void check_bounds(const attnb_bounds* b) {
  if (!b) invalid("Null bounds descriptor");
  if (b->type != ATTNB_TYPE_F32 && b->type != ATTNB_TYPE_BF16 && b->type != ATTNB_TYPE_F16)
    invalid("bounds must be F32, BF16 or F16");
  if (!b->data) invalid("Null data pointer (bounds)");
  if (reinterpret_cast<uintptr_t>(b->data) % elem_bytes(b->type) != 0)
    invalid("bounds are not aligned to their elements");
}

void check_blocks(const int32_t* blocks, int take, int64_t tokens, int H) {
  if (take <= 0) invalid("take must be positive");
  if (tokens > 0 && !blocks) invalid("Null data pointer (blocks)");
  if (!aligned4(blocks)) invalid("blocks are not aligned to their elements");
  if (tokens * H >= (1 << 30)) invalid("tokens times KV heads must be below 2^30");
}

void check_scale(float scale) {
  if (!std::isfinite(scale) || (scale > 0.f && !std::isfinite(scale * kLog2e)))
    invalid("scale must be finite, times log2(e) too");
}

SeqAttnArgs attn_args(const attnb_rows* Q, const attnb_rows* O, int kv_heads, int causal,
                      float scale, DeviceCtx& c) {
  SeqAttnArgs a{};
  a.q = rows(Q);
  a.o = rows(O);
  a.G = Q->heads / kv_heads;
  a.causal = causal != 0;
  a.scale_log2 =
      (float)((scale > 0.f ? (double)scale : 1.0 / std::sqrt((double)Q->Dh)) * 1.4426950408889634);
  a.pages.H = kv_heads;
  a.index_status = c.index_status;
  a.status = c.status;
  return a;
}

}  // namespace

extern "C" {

int attnb_seq_workspace(int q_heads, int kv_heads, int Dh, size_t* bytes) {
  return guarded(__func__, [&] {
    if (!bytes) invalid("Null data pointer");
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0)
      invalid("Q heads must be a multiple of the KV heads");
    if (Dh <= 0 || Dh > kMaxDh) invalid("Dh must be in [1, 256]");
    *bytes = seq_workspace_bytes(q_heads / kv_heads, Dh, current_ctx().num_sms);
  });
}

int attnb_attn_packed_dev(const attnb_rows* Q, const attnb_rows* K, const attnb_rows* V,
                          const attnb_rows* O, const int32_t* cu_q, const int32_t* cu_k, int batch,
                          int causal, float scale, void* workspace, size_t workspace_bytes,
                          void* stream) {
  return guarded(__func__, [&] {
    check_rows(Q, "Q", false);
    check_rows(K, "K", false);
    check_rows(V, "V", false);
    check_rows(O, "O", true);
    if (K->type != Q->type || V->type != Q->type) invalid("Q, K and V must have one type");
    if (V->tokens != K->tokens || V->heads != K->heads || V->Dh != K->Dh)
      invalid("V must be [tokens, heads, Dh] matching K");
    check_heads(Q, O, K->heads, K->Dh);
    if ((int64_t)K->tokens * (Q->heads / K->heads) >= (1 << 30))
      invalid("tokens times query heads per KV head must be below 2^30");
    if (batch < 0) invalid("batch must be non-negative");
    if (batch > 0 && (!cu_q || !cu_k)) invalid("Null cu_q or cu_k");
    if (!aligned4(cu_q)) invalid("cu_q is not aligned to its elements");
    if (!aligned4(cu_k)) invalid("cu_k is not aligned to its elements");
    check_scale(scale);
    if (batch == 0 || Q->tokens == 0) return;
    if (!workspace) invalid("Null workspace");
    DeviceCtx& c = current_ctx();
    SeqAttnArgs a = attn_args(Q, O, K->heads, causal, scale, c);
    a.k = rows(K);
    a.v = rows(V);
    a.cu_k = cu_k;
    a.seqs.cu = cu_q;
    a.seqs.batch = batch;
    a.seqs.total = Q->tokens;
    seq_attn_run(a, 0, workspace, workspace_bytes, c.num_sms, as_stream(stream));
  });
}

int attnb_attn_paged_dev(const attnb_rows* Q, const attnb_kv_pages* pages, const attnb_rows* O,
                         const attnb_seqs* seqs, int max_new, int causal, float scale,
                         void* workspace, size_t workspace_bytes, void* stream) {
  return guarded(__func__, [&] {
    check_rows(Q, "Q", false);
    check_rows(O, "O", true);
    const KvPages pg = pages_of(pages, Q->type);
    const SeqTable sq = seqs_of(seqs, Q->tokens);
    check_heads(Q, O, pg.H, pg.Dh);
    if (max_new < 0) invalid("max_new must be non-negative");
    if (((int64_t)sq.max_pages << pg.page_shift) * (Q->heads / pg.H) >= (1 << 30))
      invalid("the table's tokens times query heads per KV head must be below 2^30");
    check_scale(scale);
    if (sq.batch == 0 || sq.total == 0) return;
    if (!workspace) invalid("Null workspace");
    DeviceCtx& c = current_ctx();
    SeqAttnArgs a = attn_args(Q, O, pg.H, causal, scale, c);
    a.pages = pg;
    a.seqs = sq;
    seq_attn_run(a, max_new, workspace, workspace_bytes, c.num_sms, as_stream(stream));
  });
}

int attnb_kv_pages_append_dev(const attnb_rows* K, const attnb_rows* V,
                              const attnb_kv_pages* pages, const attnb_seqs* seqs, void* stream) {
  return guarded(__func__, [&] {
    check_rows(K, "K", false);
    check_rows(V, "V", false);
    if (V->type != K->type) invalid("K and V must have one type");
    const KvPages pg = pages_of(pages, K->type);
    check_kv(K, V, pg);
    const SeqTable sq = seqs_of(seqs, K->tokens);
    if (sq.batch == 0 || sq.total == 0) return;
    DeviceCtx& c = current_ctx();
    kv_pages_append_launch(rows(K), rows(V), pg, sq, c.index_status, c.num_sms,
                           as_stream(stream));
  });
}

int attnb_kv_pages_append_rope_dev(const attnb_rows* Q, const attnb_rows* QO, const attnb_rows* K,
                                   const attnb_rows* V, const attnb_kv_pages* pages,
                                   const attnb_seqs* seqs, const attnb_rope* rope, void* stream) {
  return guarded(__func__, [&] {
    check_rows(K, "K", false);
    check_rows(V, "V", false);
    if (V->type != K->type) invalid("K and V must have one type");
    const KvPages pg = pages_of(pages, K->type);
    check_kv(K, V, pg);
    if (!Q != !QO) invalid("Q and QO must both be given or both be NULL");
    if (Q) {
      check_rows(Q, "Q", false);
      check_rows(QO, "QO", true);
      if (Q->type != K->type || QO->type != K->type) invalid("Q and QO must have K's type");
      if (Q->tokens != K->tokens || Q->Dh != K->Dh) invalid("Q must have K's tokens and Dh");
      if (QO->tokens != Q->tokens || QO->heads != Q->heads || QO->Dh != Q->Dh)
        invalid("QO must be [tokens, heads, Dh] matching Q");
      if (Q->data == QO->data && ((Q->tokens > 1 && Q->strideT != QO->strideT) ||
                                  (Q->heads > 1 && Q->strideH != QO->strideH)))
        invalid("QO in the place of Q must have Q's strides");
    }
    if (!rope) invalid("Null rope descriptor");
    if (rope->pairs <= 0 || rope->pairs > K->Dh / 2) invalid("pairs must be in [1, Dh / 2]");
    if (!rope->inv_freq) invalid("Null data pointer (inv_freq)");
    if (!aligned4(rope->inv_freq)) invalid("inv_freq is not aligned to its elements");
    const SeqTable sq = seqs_of(seqs, K->tokens);
    if (sq.batch == 0 || sq.total == 0) return;
    DeviceCtx& c = current_ctx();
    kv_pages_append_rope_launch(Q ? rows(Q) : RowsView{}, Q ? rows(QO) : RowsView{}, rows(K),
                                rows(V), pg, sq,
                                Rope{rope->inv_freq, rope->pairs, rope->interleaved != 0},
                                c.index_status, c.num_sms, as_stream(stream));
  });
}

int attnb_kv_pages_read_dev(const attnb_kv_pages* pages, const attnb_rows* K, const attnb_rows* V,
                            const attnb_seqs* seqs, void* stream) {
  return guarded(__func__, [&] {
    check_rows(K, "K", true);
    check_rows(V, "V", true);
    if (V->type != K->type) invalid("K and V must have one type");
    const KvPages pg = pages_of(pages, K->type);
    check_kv(K, V, pg);
    const SeqTable sq = seqs_of(seqs, K->tokens);
    if (sq.batch == 0 || sq.total == 0) return;
    DeviceCtx& c = current_ctx();
    kv_pages_read_launch(pg, rows(K), rows(V), sq, c.index_status, c.num_sms, as_stream(stream));
  });
}

int attnb_kv_blocks_bounds_dev(const attnb_kv_pages* pages, const attnb_bounds* bounds,
                               const attnb_seqs* seqs, void* stream) {
  return guarded(__func__, [&] {
    check_bounds(bounds);
    const KvPages pg = pages_of(pages, bounds->type, true);
    const SeqTable sq = seqs_of(seqs, 0);
    if ((int64_t)sq.max_pages << pg.page_shift >= (1 << 30))
      invalid("the table's tokens must be below 2^30");
    if (sq.batch == 0 || sq.max_pages == 0) return;
    if ((int64_t)sq.batch * sq.max_pages >= (1ll << 31))
      invalid("sequences times the table's pages must be below 2^31");
    DeviceCtx& c = current_ctx();
    kv_blocks_bounds_launch(pg, bounds->data, bounds->type, sq, c.index_status, c.num_sms,
                            as_stream(stream));
  });
}

int attnb_blocks_workspace(int tokens, int q_heads, int kv_heads, int Dh, int take, int max_pages,
                           size_t* bytes) {
  return guarded(__func__, [&] {
    if (!bytes) invalid("Null data pointer");
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0)
      invalid("Q heads must be a multiple of the KV heads");
    if (Dh <= 0 || Dh > kMaxDh) invalid("Dh must be in [1, 256]");
    if (tokens < 0 || max_pages < 0) invalid("tokens and max_pages must be non-negative");
    if (take <= 0) invalid("take must be positive");
    *bytes = std::max(kv_blocks_workspace_bytes(tokens, kv_heads, max_pages),
                      seq_workspace_bytes(q_heads / kv_heads, Dh, current_ctx().num_sms));
  });
}

int attnb_kv_blocks_select_dev(const attnb_rows* Q, const attnb_bounds* bounds, int num_pages, int H,
                               int page_size, const attnb_seqs* seqs, int keep_first,
                               int keep_last, int32_t* blocks, int take, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return guarded(__func__, [&] {
    check_rows(Q, "Q", false);
    check_bounds(bounds);
    if (Q->type != bounds->type) invalid("Q must have the bounds' type");
    if (num_pages < 0 || H <= 0) invalid("pages have an invalid number or H");
    if (Q->heads % H != 0) invalid("Q heads must be a multiple of the KV heads");
    const int shift = page_shift_of(page_size);
    const SeqTable sq = seqs_of(seqs, Q->tokens);
    check_blocks(blocks, take, Q->tokens, H);
    if (keep_first < 0) invalid("keep_first must be non-negative");
    if (keep_last < 1) invalid("keep_last must be positive: a token's own block is one of them");
    if ((int64_t)keep_first + keep_last > take)
      invalid("keep_first and keep_last must be no more than take");
    if ((int64_t)sq.max_pages << shift >= (1 << 30))
      invalid("the table's tokens must be below 2^30");
    if (sq.batch == 0 || sq.total == 0) return;
    if (!workspace) invalid("Null workspace");
    DeviceCtx& c = current_ctx();
    kv_blocks_select_run(rows(Q), bounds->data, num_pages, H, shift, sq, keep_first, keep_last,
                         blocks, take, workspace, workspace_bytes, c.index_status, c.num_sms,
                         as_stream(stream));
  });
}

int attnb_attn_blocks_dev(const attnb_rows* Q, const attnb_kv_pages* pages, const attnb_rows* O,
                          const attnb_seqs* seqs, const int32_t* blocks, int take, float scale,
                          void* workspace, size_t workspace_bytes, void* stream) {
  return guarded(__func__, [&] {
    check_rows(Q, "Q", false);
    check_rows(O, "O", true);
    const KvPages pg = pages_of(pages, Q->type);
    const SeqTable sq = seqs_of(seqs, Q->tokens);
    check_heads(Q, O, pg.H, pg.Dh);
    check_blocks(blocks, take, Q->tokens, pg.H);
    if (((int64_t)sq.max_pages << pg.page_shift) * (Q->heads / pg.H) >= (1 << 30) ||
        ((int64_t)take << pg.page_shift) * (Q->heads / pg.H) >= (1 << 30))
      invalid("the table's tokens times query heads per KV head must be below 2^30");
    check_scale(scale);
    if (sq.batch == 0 || sq.total == 0) return;
    if (!workspace) invalid("Null workspace");
    DeviceCtx& c = current_ctx();
    SeqAttnArgs a = attn_args(Q, O, pg.H, 1, scale, c);
    a.pages = pg;
    a.seqs = sq;
    seq_attn_blocks_run(a, blocks, take, workspace, workspace_bytes, c.num_sms, as_stream(stream));
  });
}

}  // extern "C"
