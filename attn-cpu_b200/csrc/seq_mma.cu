// seq_mma.cu -- K7: attention of few query rows (16 of a KV head at a time, as in
// generation steps) over pages, 16-bit queries, 16-bit or coded keys.
//
// Bound by memory: every key is read once from HBM for all the query heads of
// its KV head.  With 8 query heads a key of 512 bytes costs 4096 operations, 51
// TFLOP/s at HBM rate and twice that over codes, more than CUDA cores have next
// to the rest of the work: the products go to the tensor cores, in the
// warp-wide form (mma.sync m16n8k16).  A 128-row tile of tcgen05 would hold 8
// useful rows in 128; the 16-row form needs no accumulator outside registers
// and its rate is far above what the memory asks for.
//
// A CTA is four warps and a loader.  The loader streams tiles of 64 keys (K and
// V, and the scales of codes) by TMA into a ring, page by page, across the ends
// of pieces, so that the memory pipe does not drain between items; two CTAs
// share an SM.  Each warp takes 16 of the 64 keys with all rows: Q stays in
// registers, S = Q K^T goes straight into the weights' A fragment, and the
// running maximum, sum and accumulator are the warp's own until the piece ends.
//
// Codes: both products run in f16, where e4m3 and int8 codes are exact.  Q is
// brought to [1, 2) by a power of two per row (bf16 has more range than f16).
// The V scale enters the exponent: with s' = s + log2(vscale) and m the maximum
// of s', the weights 2^(s' - m) lie in [0, 1] whatever the scales are, and the
// sum takes 2^(s' - m) / vscale.  Weights are rounded to the products' type
// once (half a step of 2^-11 in f16, 2^-8 in bf16, of weights at most 1); sums,
// maxima and accumulators are fp32.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "runtime.h"
#include "seq_elem.cuh"
#include "seq_pages.cuh"

namespace attnb {
namespace {

constexpr int kRows = 16;
constexpr int kKeys = 64;
constexpr int kWarps = 4;
constexpr int kThreads = (kWarps + 1) * 32;

template <int TK, int DHP>
struct MmaCfg {
  static constexpr bool CODED = TK == kE4M3 || TK == kI8;
  static constexpr int CHUNKS = CODED ? 1 : DHP / 64;  // 128-byte pieces of a row
  static constexpr int CHUNK = kKeys * 128;
  static constexpr int TILE = CHUNKS * CHUNK;          // K or V
  static constexpr int STAGE = 2 * TILE + (CODED ? 1024 : 0);
  static constexpr int STAGES = CODED ? 5 : (DHP == 128 ? 3 : 6);
  // Exchange at the end of a piece: 32 dimensions of 4 warps x 16 rows.
  static constexpr int XROW = 36;
  static constexpr int OFF_X = STAGES * STAGE;
  static constexpr int OFF_POISON = OFF_X + kWarps * kRows * XROW * 4;
  static constexpr int SMEM = OFF_POISON + 3 * DHP * 4 + 1024;
  static_assert(SMEM <= 112 * 1024, "two CTAs per SM");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// TQ: type of Q and O; TK: TQ or codes; DHP: head size padded to 64 or 128.
template <int TQ, int TK, int DHP>
__global__ void __launch_bounds__(kThreads, 2)
    seq_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ SeqAttnArgs a) {
  using Cfg = MmaCfg<TK, DHP>;
  using EQ = elem_t<TQ>;
  constexpr bool CODED = Cfg::CODED;
  constexpr bool BF16 = TQ == kBF16 && !CODED;  // type of the products
  constexpr int ST = Cfg::STAGES;
  constexpr int KS = DHP / 16;  // steps of the product over the head dimension
  constexpr int NT = DHP / 8;   // 8-wide column tiles of the output

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[ST], empty[ST];
  __shared__ SeqShared sh;
  __shared__ float2 sm_ml[kWarps][kRows];
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t* const mem = smem_raw + (base - smem_addr(smem_raw));
  int* const poison = reinterpret_cast<int*>(mem + Cfg::OFF_POISON);
  volatile int* abort_p = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_addr(&full[i]), 1);
      mbar_init(smem_addr(&empty[i]), kWarps);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  for (int i = threadIdx.x; i < 3 * DHP; i += kThreads) poison[i] = INT_MAX;
  grid_dep_wait();
  SeqPlace place;
  const bool any = seq_locate(a, sh, place);  // synchronises the block
  if (threadIdx.x == 0) seq_write_split(a, any, place);
  if (!any) return;
  __syncthreads();

  SeqIter it;
  it.start(place);
  SeqPiece w;
  if (warp == kWarps) {
    // ---------------------------------------------------------------- loader
    Ring<ST> ring;
    PageWindow win;
    const int shift = a.pages.page_shift;
    const int box = min(1 << shift, kKeys);  // rows per copy
    const int copies = kKeys / box;
    while (it.next(a, w)) {
      const int used = (w.s.L + (1 << shift) - 1) >> shift;
      for (int j = w.j0; j < w.j1; ++j) {
        int got = 0;
        if (lane == 0)
          got = mbar_wait(smem_addr(&empty[ring.stage]), ring.phase ^ 1u, abort_p, a.status);
        if (!__shfl_sync(0xffffffffu, got, 0)) goto drained;
        const uint32_t st = base + ring.stage * Cfg::STAGE;
        const uint32_t bar = smem_addr(&full[ring.stage]);
        int page[kKeys / 16];
        uint32_t bytes = 2 * Cfg::TILE;
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
          if (i >= copies) break;
          const int at = j * kKeys + i * box;
          page[i] = win.get(a, w.b, at >> shift, used);
          if constexpr (CODED) {
            if (page[i] < a.pages.num_pages) {
              bytes += 2 * box * 4;
            } else if (lane < 2) {  // no such page: codes 0 with a scale of 1
              float* sc = reinterpret_cast<float*>(mem + ring.stage * Cfg::STAGE + 2 * Cfg::TILE);
              for (int k = 0; k < box; ++k) sc[lane * kKeys + i * box + k] = 1.f;
              fence_proxy_async_smem();
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
        __syncwarp();
        if (lane < 2) {  // lane 0: K, lane 1: V
          const CUtensorMap* map = lane ? &tmV : &tmK;
          const float* sc = lane ? a.pages.v_scale : a.pages.k_scale;
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i) {
            if (i >= copies) break;
            const int in_page = (j * kKeys + i * box) & ((1 << shift) - 1);
            const uint32_t dst = st + lane * Cfg::TILE + i * box * 128;
#pragma unroll
            for (int c = 0; c < Cfg::CHUNKS; ++c)
              tma_load_4d(dst + c * Cfg::CHUNK, map, bar, c * 64, in_page, w.h, page[i]);
            if (CODED && page[i] < a.pages.num_pages)
              bulk_load(st + 2 * Cfg::TILE + (lane * kKeys + i * box) * 4,
                        sc + ((((int64_t)page[i] * a.pages.H + w.h) << shift) + in_page), box * 4,
                        bar);
          }
        }
        ring.note_issue();
        ring.advance();
      }
    }
  drained:
    // Every copy issued lands before the CTA may exit.
    if (lane == 0)
      for (int i = 0; i < ST; ++i)
        if (ring.issued_mask & (1u << i))
          drain_wait(smem_addr(&full[i]), (ring.issued_parity >> i) & 1u, a.status);
    return;
  }

  // ------------------------------------------------------------------ 16 keys
  const int g = lane >> 2, c = lane & 3;  // fragment row and column group
  Ring<ST> ring;
  bool ok = true;
  for (bool first = true; it.next(a, w); first = false) {
    // Q as A fragments: rows g and g + 8, by step of 16 dimensions.  16-bit keys:
    // dimensions 2c, 2c+1 and 2c+8, 2c+9 of the step; codes: 4c .. 4c+3, as a
    // 4-byte unit of ldmatrix holds them.
    uint32_t q[KS][4];
    int seen[2];
    float qs[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i, row = w.row0 + r;
      seen[i] = 0;
      qs[i] = a.scale_log2;
      float x[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = 0.f;
      if (r < w.rows) {
        seen[i] = seq_row_seen(a, w.s, row);
        const EQ* p = static_cast<const EQ*>(a.q.data) + (int64_t)(w.s.q0 + row / a.G) * a.q.sT +
                      (int64_t)(w.h * a.G + row % a.G) * a.q.sH;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if constexpr (CODED) {
            if (k * 16 + 4 * c < a.q.Dh) load4(p + k * 16 + 4 * c, x[k]);
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = k * 16 + 2 * c + 8 * e;
              if (d < a.q.Dh) {  // Dh is even here
                const uint32_t two = __ldg(reinterpret_cast<const uint32_t*>(p + d));
                q[k][i + 2 * e] = two;
              } else {
                q[k][i + 2 * e] = 0;
              }
            }
          }
        }
      } else if constexpr (!CODED) {
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k][i] = q[k][i + 2] = 0;
      }
      if constexpr (CODED) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[k][e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float f = row_scale(top);
        qs[i] = a.scale_log2 / f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          q[k][i] = pack_f16(x[k][0] * f, x[k][1] * f);
          q[k][i + 2] = pack_f16(x[k][2] * f, x[k][3] * f);
        }
      }
    }
    const int seen_min = seq_row_seen(a, w.s, w.row0);  // of the piece's first row
    float acc[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

    for (int j = w.j0; j < w.j1; ++j) {
      if (ok) ok = mbar_wait(smem_addr(&full[ring.stage]), ring.phase, abort_p, a.status);
      ok = __all_sync(0xffffffffu, ok);
      const uint32_t st = base + ring.stage * Cfg::STAGE;
      const int key0 = j * kKeys + warp * 16;
      const bool masked = key0 + 16 > seen_min;  // warp-uniform
      if (ok && key0 < w.s.L) {
        // ---- S = Q K^T for 16 keys: two column tiles of 8
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
        const int kr = warp * 16 + (lane & 7) + ((lane >> 4) << 3);  // this lane's matrix row
        if constexpr (CODED) {
#pragma unroll
          for (int k = 0; k < KS; k += 2) {
            uint32_t b[4];
            ldsm4(st + sw128(kr, k + ((lane >> 3) & 1)), b);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                uint32_t b0, b1;
                codes_to_f16<TK>(b[2 * t + e], b0, b1);
                mma16816<false>(s[t], q[k + e], b0, b1);
              }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b[4];
            ldsm4(st + (k >> 2) * Cfg::CHUNK + sw128(kr, (k & 3) * 2 + ((lane >> 3) & 1)), b);
            mma16816<BF16>(s[0], q[k], b[0], b[1]);
            mma16816<BF16>(s[1], q[k], b[2], b[3]);
          }
        }
        // ---- weights
        float vinv[2][2];  // codes: 1 / vscale
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + t * 8 + 2 * c + e;
            float k0 = qs[0], k1 = qs[1], add = 0.f;
            if constexpr (CODED) {
              const float* sc = reinterpret_cast<const float*>(
                  mem + ring.stage * Cfg::STAGE + 2 * Cfg::TILE);
              const int at = warp * 16 + t * 8 + 2 * c + e;
              const float ks = sc[at];
              // A vector of zeros has scale 0; any small one does for it.
              const float vs = sc[kKeys + at];
              const float use = vs < 0x1p-60f ? 0x1p-60f : vs;
              k0 *= ks;
              k1 *= ks;
              add = __log2f(use);
              vinv[t][e] = fast_exp2(-add);
            }
            s[t][e] = fmaf(s[t][e], k0, add);
            s[t][e + 2] = fmaf(s[t][e + 2], k1, add);
            if (masked) {
              if (key >= seen[0]) s[t][e] = -INFINITY;
              if (key >= seen[1]) s[t][e + 2] = -INFINITY;
            }
          }
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top, m[i]);
          const float use = top == -INFINITY ? 0.f : top;
          alpha[i] = fast_exp2(m[i] - use);
          m[i] = top;
          float sum = 0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p = fast_exp2(s[t][2 * i + e] - use);
              s[t][2 * i + e] = p;
              // The scale of a masked key may be anything.
              if constexpr (CODED) sum += p != 0.f ? p * vinv[t][e] : 0.f;
              else sum += p;
            }
          l[i] = fmaf(l[i], alpha[i], sum);
        }
        uint32_t p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            p[2 * t + i] = BF16 ? pack_bf16(s[t][2 * i], s[t][2 * i + 1])
                                : pack_f16(s[t][2 * i], s[t][2 * i + 1]);
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[t][0] *= alpha[0];
            acc[t][1] *= alpha[0];
            acc[t][2] *= alpha[1];
            acc[t][3] *= alpha[1];
          }
        }
        // ---- values that a mask hides (written codes are finite)
        if (CODED ? key0 + 16 > w.s.L : masked) {
          uint8_t* v = mem + ring.stage * Cfg::STAGE + Cfg::TILE;
          for (int i = lane; i < 16 * Cfg::CHUNKS * 8; i += 32) {
            const int r = i & 15, u = (i >> 4) & 7, ch = i >> 7;
            const int key = key0 + r;
            uint4* at = reinterpret_cast<uint4*>(v + ch * Cfg::CHUNK + sw128(warp * 16 + r, u));
            if (key >= w.s.L) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (!CODED && key >= seen_min) {
              uint4 x = *at;
              EQ* e = reinterpret_cast<EQ*>(&x);
              bool hit = false;
#pragma unroll
              for (int b = 0; b < 8; ++b) {
                const float f = to_float(e[b]);
                if (fabsf(f) <= 3.402823466e38f) continue;
                hit = true;
                const int kind = f != f ? 0 : (f > 0.f ? 1 : 2);
                atomicMin(&poison[kind * DHP + ch * 64 + u * 8 + b], key);
                from_float(0.f, e[b]);
              }
              if (hit) *at = x;
            }
          }
          fence_proxy_async_smem();  // the next copy into the stage comes after these writes
          __syncwarp();
        }
        // ---- O += P V
        const int vr = warp * 16 + (lane & 15);  // this lane's matrix row
        if constexpr (CODED) {
#pragma unroll
          for (int u = 0; u < KS; u += 2) {  // 16 dimensions each
            uint32_t b[4];
            ldsm4_t(st + Cfg::TILE + sw128(vr, u + (lane >> 4)), b);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // bytes: (key, d), (key, d+1), (key+1, d), (key+1, d+1), brought to
              // pairs of keys: d, then d + 1
              uint32_t lo0, lo1, hi0, hi1;
              codes_to_f16<TK>(__byte_perm(b[2 * e], 0, 0x3120), lo0, lo1);
              codes_to_f16<TK>(__byte_perm(b[2 * e + 1], 0, 0x3120), hi0, hi1);
              mma16816<false>(acc[2 * (u + e)], p, lo0, hi0);
              mma16816<false>(acc[2 * (u + e) + 1], p, lo1, hi1);
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; t += 2) {
            uint32_t b[4];
            ldsm4_t(st + Cfg::TILE + (t >> 3) * Cfg::CHUNK + sw128(vr, (t & 7) + (lane >> 4)), b);
            mma16816<BF16>(acc[t], p, b[0], b[1]);
            mma16816<BF16>(acc[t + 1], p, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&empty[ring.stage]));
      ring.advance();
    }

    // ---- the warps' sums meet, 32 dimensions at a time
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (c == 0) sm_ml[warp][g + 8 * i] = make_float2(m[i], sum);
    }
    named_bar_sync(1, kWarps * 32);
    const int slot = seq_slot(w, first);
    float f[2], total[2], top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      top[i] = -INFINITY;
      for (int k = 0; k < kWarps; ++k) top[i] = fmaxf(top[i], sm_ml[k][r].x);
      const float use = top[i] == -INFINITY ? 0.f : top[i];
      total[i] = 0.f;
      for (int k = 0; k < kWarps; ++k)
        total[i] += fast_exp2(sm_ml[k][r].x - use) * sm_ml[k][r].y;
      f[i] = fast_exp2(m[i] - use);
      if (slot < 0) f[i] = total[i] == 0.f ? 0.f : f[i] / total[i];
      else if (warp == 0 && c == 0 && r < w.rows)
        reinterpret_cast<float2*>(a.ws_ml)[(int64_t)slot * kRows + r] =
            make_float2(top[i], total[i]);
    }
    float* x = reinterpret_cast<float*>(mem + Cfg::OFF_X);
#pragma unroll
    for (int q4 = 0; q4 < DHP / 32; ++q4) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int nt = q4 * 4 + t;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* row = x + (warp * kRows + g + 8 * i) * Cfg::XROW;
          const float v0 = acc[nt][2 * i] * f[i], v1 = acc[nt][2 * i + 1] * f[i];
          if constexpr (CODED) {  // tile nt: dimensions 16 (nt/2) + 4c + (nt & 1), + 2
            row[(t >> 1) * 16 + 4 * c + (t & 1)] = v0;
            row[(t >> 1) * 16 + 4 * c + (t & 1) + 2] = v1;
          } else {
            *reinterpret_cast<float2*>(row + t * 8 + 2 * c) = make_float2(v0, v1);
          }
        }
      }
      named_bar_sync(1, kWarps * 32);
      for (int i = threadIdx.x; i < kRows * 32; i += kWarps * 32) {
        const int r = i >> 5, d = q4 * 32 + (i & 31);
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += x[(k * kRows + r) * Cfg::XROW + (i & 31)];
        if (r < w.rows && d < a.q.Dh) {
          const int row = w.row0 + r;
          if constexpr (!CODED)
            v = poisoned(v, poison, poison + DHP, poison + 2 * DHP, d, seq_row_seen(a, w.s, row));
          if (slot >= 0)
            a.ws_o[((int64_t)slot * kRows + r) * a.q.Dh + d] = v;
          else
            from_float(v, *(static_cast<EQ*>(a.o.data) +
                            (int64_t)(w.s.q0 + row / a.G) * a.o.sT +
                            (int64_t)(w.h * a.G + row % a.G) * a.o.sH + d));
        }
      }
      named_bar_sync(1, kWarps * 32);
    }
    if constexpr (!CODED) {
      for (int i = threadIdx.x; i < 3 * DHP; i += kWarps * 32) poison[i] = INT_MAX;
      named_bar_sync(1, kWarps * 32);
    }
  }
}

template <int TQ, int TK, int DHP>
void launch(const SeqAttnArgs& a, int ctas, const CUtensorMap& k, const CUtensorMap& v,
            cudaStream_t s) {
  using Cfg = MmaCfg<TK, DHP>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  ATTNB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    ATTNB_CUDA(cudaFuncSetAttribute(seq_mma_kernel<TQ, TK, DHP>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    configured.fetch_or(bit);
  }
  ATTNB_CUDA(launch_pdl(seq_mma_kernel<TQ, TK, DHP>, dim3(ctas), dim3(kThreads), Cfg::SMEM, s, k,
                        v, a));
}

}  // namespace

bool seq_pages_tma(const SeqAttnArgs& a) {
  const KvPages& p = a.pages;
  if (!p.k || p.num_pages == 0 || a.q.type == kF32 || p.Dh > 128) return false;
  if ((p.Dh * elem_bytes(p.type)) % 16 != 0) return false;
  auto at16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!at16(p.k) || !at16(p.v)) return false;
  return !elem_coded(p.type) || (at16(p.k_scale) && at16(p.v_scale));
}

CUtensorMap seq_pages_map(const KvPages& p, const void* base, int rows) {
  const uint64_t eb = elem_bytes(p.type), page = 1u << p.page_shift;
  const uint64_t dims[4] = {(uint64_t)p.Dh, page, (uint64_t)p.H, (uint64_t)p.num_pages};
  const uint64_t strides[3] = {p.Dh * eb, p.Dh * page * eb, p.Dh * page * p.H * eb};
  const uint32_t box[4] = {(uint32_t)(128 / eb), (uint32_t)std::min<uint64_t>(page, rows), 1, 1};
  return make_tmap_nd(base, (int)eb, 4, dims, strides, box);
}

// Q is read in units of 2 (16-bit keys) or 4 (codes) elements.
bool seq_mma_supported(const SeqAttnArgs& a) {
  const int unit = elem_coded(a.pages.type) ? 4 : 2;
  return seq_pages_tma(a) && reinterpret_cast<uintptr_t>(a.q.data) % (2 * unit) == 0 &&
         a.q.sT % unit == 0 && a.q.sH % unit == 0;
}

void seq_mma_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  const CUtensorMap k = seq_pages_map(a.pages, a.pages.k, kKeys);
  const CUtensorMap v = seq_pages_map(a.pages, a.pages.v, kKeys);
  auto go = [&](auto tq, auto tk) {
    constexpr int TQ = decltype(tq)::value, TK = decltype(tk)::value;
    if constexpr (TQ != kF32) {
      if (a.q.Dh <= 64) launch<TQ, TK, 64>(a, ctas, k, v, s);
      else launch<TQ, TK, 128>(a, ctas, k, v, s);
    }
  };
  with_value_type(a.q.type, [&](auto tq) {
    if (a.pages.type == kE4M3) go(tq, std::integral_constant<int, kE4M3>{});
    else if (a.pages.type == kI8) go(tq, std::integral_constant<int, kI8>{});
    else go(tq, tq);
  });
}

}  // namespace attnb
