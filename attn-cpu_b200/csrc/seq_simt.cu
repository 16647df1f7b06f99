// seq_simt.cu -- K6: attention of packed query rows over packed keys or pages on
// CUDA cores, for every type, stride and head size up to 256 (and all of fp32).
//
// For a query row i and the keys j that it sees,
//     s_j = scale * kscale_j * q . k_j,   o = sum_j 2^(s_j - m) vscale_j v_j / sum_j 2^(s_j - m)
// with s in base-2 units and m the running maximum; the scales are 1 unless the
// pages hold codes.  It follows the online softmax of decode.cu.
//
// A CTA takes up to 4 rows (2 for head sizes over 128) of one KV head and walks
// 64 keys at a time: 16 groups of 8 lanes take 4 keys each, so that a row of K
// is one coalesced read of 8 lanes and a dot product ends after 3 shuffles.
// Each group keeps its own maximum, sum and accumulator in registers; they meet
// in shared memory once per piece.  Four rows are what the registers hold (64
// for q, 64 for the accumulator, 64 for K or V in flight); more rows read the
// keys again, from L2.  For a single row (a step without grouped heads) the
// registers hold V next to K, so that both are in flight at once.
//
// Bound by the loads in flight: 8 sequences x 32 heads x 4096 fp32 keys in pages of
// 16 (1.07 GB) take 295 us, 3.6 TB/s.  The form for a single row of a head size over
// 64 spills (772 bytes stored a thread at 168 registers), a ring of tiles in shared
// memory, as K7 has, would keep more of them going.
#include <cmath>

#include "seq.cuh"
#include "seq_elem.cuh"
#include "runtime.h"

namespace attnb {
namespace {

constexpr int kThreads = 128;
constexpr int kGroups = kThreads / 8;
constexpr int kKeys = 4;  // keys in flight per group; kGroups * kKeys = 64 keys per tile

// Element of the head dimension that lane `e` of a group holds at (c, i).
__device__ __forceinline__ int dim_of(int e, int c, int i) { return (c * 8 + e) * 4 + i; }

// The lane's share of one row.
template <class E, int NC>
__device__ __forceinline__ void load_row(const E* p, int e, int Dh, bool vec, float (&x)[NC * 4]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = dim_of(e, c, 0);
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
      if (d < Dh) load4(p + d, f);  // Dh is a multiple of 4 here
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < Dh) f[i] = to_float(p[d + i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[c * 4 + i] = f[i];
  }
}

template <int TQ, int TK, int R, int NC>
__global__ void __launch_bounds__(kThreads, R == 1 ? 3 : 1) seq_simt_kernel(const SeqAttnArgs a, const bool qvec,
                                                            const bool kvec) {
  using EQ = elem_t<TQ>;
  using EK = elem_t<TK>;
  constexpr bool CODED = TK == kE4M3 || TK == kI8;
  constexpr int D = NC * 32;  // head size padded to the lanes' shares
  __shared__ SeqShared sh;
  __shared__ float sm_acc[kThreads / 32][R][D];
  __shared__ float2 sm_ml[kThreads / 32][R];

  grid_dep_wait();
  SeqPlace place;
  const bool any = seq_locate(a, sh, place);
  if (threadIdx.x == 0) seq_write_split(a, any, place);
  if (!any) return;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = lane & 7, group = threadIdx.x >> 3;
  const int Dh = a.q.Dh;
  const bool paged = a.pages.k != nullptr;
  const int page_mask = (1 << a.pages.page_shift) - 1;

  SeqIter it;
  it.start(place);
  SeqPiece w;
  for (bool first = true; it.next(a, w); first = false) {
    float q[R][NC * 4], acc[R][NC * 4], m[R], l[R];
    int seen[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
      seen[r] = 0;
#pragma unroll
      for (int i = 0; i < NC * 4; ++i) q[r][i] = acc[r][i] = 0.f;
      if (r < w.rows) {
        const int row = w.row0 + r;
        seen[r] = seq_row_seen(a, w.s, row);
        const EQ* p = static_cast<const EQ*>(a.q.data) + (int64_t)(w.s.q0 + row / a.G) * a.q.sT +
                      (int64_t)(w.h * a.G + row % a.G) * a.q.sH;
        load_row<EQ, NC>(p, e, Dh, qvec, q[r]);
      }
    }
    for (int j = w.j0; j < w.j1; ++j) {
      const int key0 = (j << a.kt_shift) + group;
      const EK* kp[kKeys];
      const EK* vp[kKeys];
      float ks[kKeys], vs[kKeys];
#pragma unroll
      for (int u = 0; u < kKeys; ++u) {
        const int key = key0 + u * kGroups;
        kp[u] = vp[u] = nullptr;
        ks[u] = a.scale_log2;
        vs[u] = 1.f;
        if (key < w.s.L) {
          if (paged) {
            const int page = seq_page(a.seqs, a.pages, w.b, key, a.index_status);
            if (page >= 0) {  // a bad page reads as zeros
              const int64_t at =
                  (((int64_t)page * a.pages.H + w.h) << a.pages.page_shift) + (key & page_mask);
              kp[u] = static_cast<const EK*>(a.pages.k) + at * Dh;
              vp[u] = static_cast<const EK*>(a.pages.v) + at * Dh;
              if (CODED) {
                ks[u] = a.scale_log2 * __ldg(a.pages.k_scale + at);
                vs[u] = __ldg(a.pages.v_scale + at);
              }
            }
          } else {
            kp[u] = static_cast<const EK*>(a.k.data) + (int64_t)(w.s.k0 + key) * a.k.sT +
                    (int64_t)w.h * a.k.sH;
            vp[u] = static_cast<const EK*>(a.v.data) + (int64_t)(w.s.k0 + key) * a.v.sT +
                    (int64_t)w.h * a.v.sH;
          }
        }
      }
      float s[R][kKeys];
      float v[R == 1 ? kKeys : 1][NC * 4];
      {
        float x[kKeys][NC * 4];
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
#pragma unroll
          for (int i = 0; i < NC * 4; ++i) x[u][i] = 0.f;
          if (kp[u]) load_row<EK, NC>(kp[u], e, Dh, kvec, x[u]);
        }
        if constexpr (R == 1) {
#pragma unroll
          for (int u = 0; u < kKeys; ++u)
            if (vp[u]) load_row<EK, NC>(vp[u], e, Dh, kvec, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kKeys; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float d = 0.f;
#pragma unroll
            for (int i = 0; i < NC * 4; ++i) d = fmaf(q[r][i], x[u][i], d);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
            const int key = key0 + u * kGroups;
            s[r][u] = key < w.s.L && key < seen[r] ? d * ks[u] : -INFINITY;
          }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int u = 0; u < kKeys; ++u) top = fmaxf(top, s[r][u]);
        const float use = top == -INFINITY ? 0.f : top;
        const float alpha = fast_exp2(m[r] - use);
        m[r] = top;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < NC * 4; ++i) acc[r][i] *= alpha;
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
          s[r][u] = fast_exp2(s[r][u] - use);
          l[r] += s[r][u];
          if (CODED) s[r][u] *= vs[u];
        }
      }
#pragma unroll
      for (int u = 0; u < kKeys; ++u) {
        if (!vp[u]) continue;
        const int at = R == 1 ? u : 0;
        if constexpr (R > 1) load_row<EK, NC>(vp[u], e, Dh, kvec, v[0]);
        const int key = key0 + u * kGroups;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          // A masked value may be anything: it is left out, not multiplied by 0.
          if (key >= seen[r]) continue;
#pragma unroll
          for (int i = 0; i < NC * 4; ++i) acc[r][i] = fmaf(s[r][u], v[at][i], acc[r][i]);
        }
      }
    }
    // The four groups of a warp meet by shuffles, the warps in shared memory.
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float f = top == -INFINITY ? 0.f : fast_exp2(m[r] - top);
      float sum = l[r] * f;
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
      for (int i = 0; i < NC * 4; ++i) {
        float x = acc[r][i] * f;
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (lane < 8) sm_acc[warp][r][dim_of(e, i / 4, i % 4)] = x;
      }
      if (lane == 0) sm_ml[warp][r] = make_float2(top, sum);
    }
    __syncthreads();
    const int slot = seq_slot(w, first);
    for (int r = 0; r < w.rows; ++r) {
      float top = -INFINITY;
      for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, sm_ml[i][r].x);
      float f[kThreads / 32], sum = 0.f;
      for (int i = 0; i < kThreads / 32; ++i) {
        f[i] = top == -INFINITY ? 0.f : fast_exp2(sm_ml[i][r].x - top);
        sum += f[i] * sm_ml[i][r].y;
      }
      const int row = w.row0 + r;
      for (int d = threadIdx.x; d < Dh; d += kThreads) {
        float x = 0.f;
        for (int i = 0; i < kThreads / 32; ++i) x += f[i] * sm_acc[i][r][d];
        if (slot >= 0) {
          a.ws_o[((int64_t)slot * a.rows + r) * Dh + d] = x;
        } else {
          EQ* p = static_cast<EQ*>(a.o.data) + (int64_t)(w.s.q0 + row / a.G) * a.o.sT +
                  (int64_t)(w.h * a.G + row % a.G) * a.o.sH;
          from_float(sum == 0.f ? 0.f : x / sum, p[d]);  // no key: 0
        }
      }
      if (slot >= 0 && threadIdx.x == 0)
        reinterpret_cast<float2*>(a.ws_ml)[(int64_t)slot * a.rows + r] = make_float2(top, sum);
    }
    __syncthreads();
  }
}

bool rows_aligned(const void* p, int64_t sT, int64_t sH, int Dh, int type) {
  const int b = 4 * elem_bytes(type);
  return (reinterpret_cast<uintptr_t>(p) % b) == 0 && sT % 4 == 0 && sH % 4 == 0 && Dh % 4 == 0;
}

}  // namespace

void seq_simt_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  const bool paged = a.pages.k != nullptr;
  const int tk = paged ? a.pages.type : a.k.type;
  const bool qvec = rows_aligned(a.q.data, a.q.sT, a.q.sH, a.q.Dh, a.q.type);
  const bool kvec =
      paged ? rows_aligned(a.pages.k, 0, 0, a.q.Dh, tk) && rows_aligned(a.pages.v, 0, 0, a.q.Dh, tk)
            : rows_aligned(a.k.data, a.k.sT, a.k.sH, a.q.Dh, tk) &&
                  rows_aligned(a.v.data, a.v.sT, a.v.sH, a.q.Dh, tk);
  auto go = [&](auto tq, auto tkc) {
    constexpr int TQ = decltype(tq)::value, TK = decltype(tkc)::value;
    auto run = [&](auto rows, auto nc) {
      constexpr int R = decltype(rows)::value, NC = decltype(nc)::value;
      ATTNB_CUDA(launch_pdl(seq_simt_kernel<TQ, TK, R, NC>, dim3(ctas), dim3(kThreads), 0, s, a,
                            qvec, kvec));
    };
    using std::integral_constant;
    if (a.q.Dh > 128) run(integral_constant<int, 2>{}, integral_constant<int, 8>{});
    else if (a.rows == 1 && a.q.Dh <= 64) run(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (a.rows == 1) run(integral_constant<int, 1>{}, integral_constant<int, 4>{});
    else if (a.q.Dh <= 64) run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else run(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  };
  with_value_type(a.q.type, [&](auto tq) {
    if (tk == kE4M3) go(tq, std::integral_constant<int, kE4M3>{});
    else if (tk == kI8) go(tq, std::integral_constant<int, kI8>{});
    else go(tq, tq);
  });
}

}  // namespace attnb
