// seq_mma.cu -- K7: attention of few query rows (8 or 16 of a KV head at a time, as
// in generation steps) over pages, 16-bit queries, 16-bit or coded keys.
//
// Bound by memory: every key is read once from HBM for all the query heads of
// its KV head.  With 8 query heads a key of 512 bytes costs 4096 operations, 51
// TFLOP/s at HBM rate and twice that over codes, more than CUDA cores have next
// to the rest of the work: the products go to the tensor cores, in the
// warp-wide form (mma.sync m16n8k16).  A 128-row tile of tcgen05 would hold 8
// useful rows in 128; here the 16 rows of the instruction are keys (S^T = K Q^T)
// and dimensions (O^T = V^T P^T), and the 8 columns are query rows, so that a
// step of 4 or 8 query heads wastes little of either product, and a thread holds
// half the weights and accumulators that rows of queries would take.
//
// A CTA is four warps and a loader.  The loader streams tiles of 64 keys (K and
// V, and the scales of codes) by TMA into a ring, page by page, across the ends
// of pieces, so that the memory pipe does not drain between items; two or three
// CTAs share an SM.  Each warp takes 16 of the 64 keys with all rows: Q stays in
// registers, S^T becomes the weights' B fragment by one transposition of 8 x 8
// values, and the running maximum, sum and accumulator are the warp's own until
// the piece ends.
//
// Codes: both products run in f16, where e4m3 and int8 codes are exact.  Q is
// brought to [1, 2) by a power of two per row (bf16 has more range than f16).
// The V scale enters the exponent of a weight, which keeps a reference of its
// own: with m the running maximum of the scores, the sum takes 2^(s - m) and the
// product 2^(s - m + log2(vscale) - rho), rho a running bound of that exponent
// (which may pass it by 8: f16 holds 2^8).  So neither overflows or vanishes whatever
// the scales are, and a vector of zeros (scale 0) weighs nothing; 2^rho goes
// into the output.  Weights are rounded to the products' type once (half a step
// of 2^-11 in f16, 2^-8 in bf16); sums, maxima and accumulators are fp32.
//
// Measured: 32 sequences of 500-4096 bf16 keys, 32/8 heads (296 MB) 58 us, 64 of
// 1000-8192 keys in e4m3 (622 MB) 126 us, 5 TB/s with the join; one context of
// 100001 keys (205 MB) 52 us.  With query rows as the instruction's 16 rows and two
// CTAs an SM the e4m3 case took 165 us.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "runtime.h"
#include "seq_elem.cuh"
#include "seq_pages.cuh"

namespace attnb {
namespace {

constexpr int kKeys = 64;
constexpr int kWarps = 4;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr float kRhoGap = 8.f;
constexpr float kNoRho = -1e30f;  // no weight so far: any exponent is above it

// NR: query rows / 8.
template <int TK, int DHP, int NR>
struct MmaCfg {
  static constexpr bool CODED = TK == kE4M3 || TK == kI8;
  static constexpr int ROWS = 8 * NR;
  static constexpr int CTAS = NR == 1 ? 3 : 2;         // per SM
  static constexpr int CHUNKS = CODED ? 1 : DHP / 64;  // 128-byte pieces of a row
  static constexpr int CHUNK = kKeys * 128;
  static constexpr int TILE = CHUNKS * CHUNK;          // K or V
  static constexpr int STAGE = 2 * TILE + (CODED ? 1024 : 0);
  // Together the CTAs of an SM have about 190 KB of copies in flight.
  static constexpr int STAGES = CODED ? (NR == 1 ? 3 : 5)
                                      : (DHP == 128 ? (NR == 1 ? 2 : 3) : (NR == 1 ? 4 : 6));
  // Exchange at the end of a piece: 32 dimensions of 4 warps' rows.
  static constexpr int XROW = 36;
  static constexpr int OFF_X = STAGES * STAGE;
  static constexpr int OFF_POISON = OFF_X + kWarps * ROWS * XROW * 4;
  static constexpr int SMEM = OFF_POISON + 3 * DHP * 4 + 1024;
  static_assert(SMEM + 2048 <= 227 * 1024 / CTAS, "CTAs per SM");
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
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 tile of 16-bit values, transposed across the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// TQ: type of Q and O; TK: TQ or codes; DHP: head size padded to 64 or 128.
template <int TQ, int TK, int DHP, int NR>
__global__ void __launch_bounds__(kThreads, (MmaCfg<TK, DHP, NR>::CTAS))
    seq_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ SeqAttnArgs a) {
  using Cfg = MmaCfg<TK, DHP, NR>;
  using EQ = elem_t<TQ>;
  constexpr bool CODED = Cfg::CODED;
  constexpr bool BF16 = TQ == kBF16 && !CODED;  // type of the products
  constexpr int ST = Cfg::STAGES;
  constexpr int ROWS = Cfg::ROWS;
  constexpr int KS = DHP / 16;  // 16 dimensions each

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[ST], empty[ST];
  __shared__ SeqShared sh;
  __shared__ float2 sm_ml[kWarps][ROWS];
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
            } else if (lane < 2) {  // no such page: codes 0 with a scale of 0
              float* sc = reinterpret_cast<float*>(mem + ring.stage * Cfg::STAGE + 2 * Cfg::TILE);
              for (int k = 0; k < box; ++k) sc[lane * kKeys + i * box + k] = 0.f;
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
    // Q^T as B fragments: row 8 r + g, by step of 16 dimensions.  16-bit keys:
    // dimensions 2c, 2c+1 and 2c+8, 2c+9 of the step; codes: 4c .. 4c+3, as a
    // 4-byte unit of ldmatrix holds them.
    uint32_t q[NR][KS][2];
    float mulq[NR][2];  // score to exponent, of this thread's rows 8 r + 2c, + 1
    int seen[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = w.row0 + 8 * r + g;
      const bool there = 8 * r + g < w.rows;
      const EQ* p = static_cast<const EQ*>(a.q.data) + (int64_t)(w.s.q0 + row / a.G) * a.q.sT +
                    (int64_t)(w.h * a.G + row % a.G) * a.q.sH;
      if constexpr (CODED) {
        float x[KS][4], top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][e] = 0.f;
          if (there && k * 16 + 4 * c < a.q.Dh) load4(p + k * 16 + 4 * c, x[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[k][e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float f = row_scale(top);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          q[r][k][0] = pack_f16(x[k][0] * f, x[k][1] * f);
          q[r][k][1] = pack_f16(x[k][2] * f, x[k][3] * f);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          mulq[r][i] = a.scale_log2 / __shfl_sync(0xffffffffu, f, (2 * c + i) * 4);
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = k * 16 + 2 * c + 8 * e;  // Dh is even here
            q[r][k][e] =
                there && d < a.q.Dh ? __ldg(reinterpret_cast<const uint32_t*>(p + d)) : 0u;
          }
        mulq[r][0] = mulq[r][1] = a.scale_log2;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = 8 * r + 2 * c + i;
        seen[r][i] = rr < w.rows ? seq_row_seen(a, w.s, w.row0 + rr) : 0;
      }
    }
    const int seen_min = seq_row_seen(a, w.s, w.row0);  // of the piece's first row
    float acc[KS][NR][4], m[NR][2], l[NR][2];
    float rho[NR][2];  // codes: the product's reference, relative to m
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r][0] = m[r][1] = -INFINITY;
      l[r][0] = l[r][1] = 0.f;
      rho[r][0] = rho[r][1] = kNoRho;
#pragma unroll
      for (int u = 0; u < KS; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][r][e] = 0.f;
    }

    for (int j = w.j0; j < w.j1; ++j) {
      if (ok) ok = mbar_wait_quick(smem_addr(&full[ring.stage]), ring.phase, abort_p, a.status);
      ok = __all_sync(0xffffffffu, ok);
      const uint32_t st = base + ring.stage * Cfg::STAGE;
      const int key0 = j * kKeys + warp * 16;
      const bool masked = key0 + 16 > seen_min;  // warp-uniform
      if (ok && key0 < w.s.L) {
        // ---- S^T = K Q^T: keys g, g + 8 by rows 2c, 2c + 1
        float s[NR][4];
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[r][e] = 0.f;
        const int kr = warp * 16 + (lane & 15);  // this lane's matrix row
        if constexpr (CODED) {
#pragma unroll
          for (int k = 0; k < KS; k += 2) {
            uint32_t b[4];
            ldsm4(st + sw128(kr, k + (lane >> 4)), b);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a0, a1, a2, a3;
              codes_to_f16<TK>(b[2 * e], a0, a2);
              codes_to_f16<TK>(b[2 * e + 1], a1, a3);
#pragma unroll
              for (int r = 0; r < NR; ++r)
                mma16816<false>(s[r], a0, a1, a2, a3, q[r][k + e][0], q[r][k + e][1]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b[4];
            ldsm4(st + (k >> 2) * Cfg::CHUNK + sw128(kr, (k & 3) * 2 + (lane >> 4)), b);
#pragma unroll
            for (int r = 0; r < NR; ++r)
              mma16816<BF16>(s[r], b[0], b[1], b[2], b[3], q[r][k][0], q[r][k][1]);
          }
        }
        // ---- weights
        float mulk[2] = {1.f, 1.f}, lv[2] = {0.f, 0.f};  // of keys g, g + 8
        if constexpr (CODED) {
          const float* sc =
              reinterpret_cast<const float*>(mem + ring.stage * Cfg::STAGE + 2 * Cfg::TILE);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = warp * 16 + g + 8 * i;
            mulk[i] = sc[at];
            lv[i] = __log2f(sc[kKeys + at]);  // -inf for a vector of zeros
          }
        }
        uint32_t p[NR][2];
        bool moved = false;
        float alpha[NR][2];  // what acc is multiplied by
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (CODED) s[r][e] *= mulq[r][e & 1] * mulk[e >> 1];
            else s[r][e] *= mulq[r][e & 1];
            if (masked && key0 + g + 8 * (e >> 1) >= seen[r][e & 1]) s[r][e] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[r][i], s[r][i + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[r][i]);
            const float use = top == -INFINITY ? 0.f : top;
            const float beta = fast_exp2(m[r][i] - use);
            if constexpr (CODED) {
              if (m[r][i] != -INFINITY) rho[r][i] -= top - m[r][i];
            } else {
              alpha[r][i] = beta;
              moved |= beta != 1.f;
            }
            m[r][i] = top;
            l[r][i] *= beta;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float x = s[r][i + 2 * k] - use;
              const float weight = fast_exp2(x);
              l[r][i] += weight;
              if constexpr (CODED) {
                // The scale of a masked key may be anything.
                s[r][i + 2 * k] = x == -INFINITY ? x : x + lv[k];
                moved |= s[r][i + 2 * k] - rho[r][i] > kRhoGap;
              } else {
                s[r][i + 2 * k] = weight;
              }
            }
          }
        }
        moved = __any_sync(0xffffffffu, moved);
        if constexpr (CODED) {
          if (moved) {
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float top = fmaxf(s[r][i], s[r][i + 2]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                top = fmaxf(top, rho[r][i]);
                alpha[r][i] = fast_exp2(rho[r][i] - top);
                rho[r][i] = top;
              }
          }
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[r][e] = fast_exp2(s[r][e] - rho[r][e & 1]);
        }
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            p[r][k] = transposed(BF16 ? pack_bf16(s[r][2 * k], s[r][2 * k + 1])
                                      : pack_f16(s[r][2 * k], s[r][2 * k + 1]));
        if (moved) {
#pragma unroll
          for (int u = 0; u < KS; ++u)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[u][r][e] *= alpha[r][e & 1];
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
        // ---- O^T += V^T P^T, 16 dimensions at a time
        if constexpr (CODED) {
#pragma unroll
          for (int u = 0; u < KS; u += 2) {
            uint32_t b[4];
            ldsm4_t(st + Cfg::TILE + sw128(kr, u + (lane >> 4)), b);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // bytes: (key, d), (key, d+1), (key+1, d), (key+1, d+1), brought to
              // pairs of keys: d = 2g, then 2g + 1
              uint32_t a0, a1, a2, a3;
              codes_to_f16<TK>(__byte_perm(b[2 * e], 0, 0x3120), a0, a1);
              codes_to_f16<TK>(__byte_perm(b[2 * e + 1], 0, 0x3120), a2, a3);
#pragma unroll
              for (int r = 0; r < NR; ++r)
                mma16816<false>(acc[u + e][r], a0, a1, a2, a3, p[r][0], p[r][1]);
            }
          }
        } else {
          const int vr = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
          for (int u = 0; u < KS; ++u) {
            uint32_t b[4];
            ldsm4_t(st + Cfg::TILE + (u >> 2) * Cfg::CHUNK +
                        sw128(vr, (u & 3) * 2 + ((lane >> 3) & 1)), b);
#pragma unroll
            for (int r = 0; r < NR; ++r)
              mma16816<BF16>(acc[u][r], b[0], b[1], b[2], b[3], p[r][0], p[r][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&empty[ring.stage]));
      ring.advance();
    }

    // ---- the warps' sums meet, 32 dimensions at a time
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[r][i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) sm_ml[warp][8 * r + 2 * c + i] = make_float2(m[r][i], sum);
      }
    named_bar_sync(1, kWarps * 32);
    const int slot = seq_slot(w, first);
    float f[NR][2], fr[NR][2];  // two factors: 2^rho may lie below the smallest fp32 number
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = 8 * r + 2 * c + i;
        float top = -INFINITY, total = 0.f;
        for (int k = 0; k < kWarps; ++k) top = fmaxf(top, sm_ml[k][rr].x);
        const float use = top == -INFINITY ? 0.f : top;
        for (int k = 0; k < kWarps; ++k)
          total += fast_exp2(sm_ml[k][rr].x - use) * sm_ml[k][rr].y;
        fr[r][i] = CODED ? fast_exp2(0.5f * (m[r][i] - use + rho[r][i])) : 1.f;
        f[r][i] = CODED ? fr[r][i] : fast_exp2(m[r][i] - use);
        if (slot < 0) f[r][i] = total == 0.f ? 0.f : f[r][i] / total;
        else if (warp == 0 && g == 0 && rr < w.rows)
          reinterpret_cast<float2*>(a.ws_ml)[(int64_t)slot * ROWS + rr] = make_float2(top, total);
      }
    float* x = reinterpret_cast<float*>(mem + Cfg::OFF_X);
#pragma unroll
    for (int q4 = 0; q4 < DHP / 32; ++q4) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = t * 16 + (CODED ? 2 * g + (e >> 1) : g + 8 * (e >> 1));
            x[(warp * ROWS + 8 * r + 2 * c + (e & 1)) * Cfg::XROW + d] =
                (CODED ? acc[q4 * 2 + t][r][e] * fr[r][e & 1] : acc[q4 * 2 + t][r][e]) * f[r][e & 1];
          }
      named_bar_sync(1, kWarps * 32);
      for (int i = threadIdx.x; i < ROWS * 32; i += kWarps * 32) {
        const int r = i >> 5, d = q4 * 32 + (i & 31);
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += x[(k * ROWS + r) * Cfg::XROW + (i & 31)];
        if (r < w.rows && d < a.q.Dh) {
          const int row = w.row0 + r;
          if constexpr (!CODED)
            v = poisoned(v, poison, poison + DHP, poison + 2 * DHP, d, seq_row_seen(a, w.s, row));
          if (slot >= 0)
            a.ws_o[((int64_t)slot * ROWS + r) * a.q.Dh + d] = v;
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

template <int TQ, int TK, int DHP, int NR>
void launch(const SeqAttnArgs& a, int ctas, const CUtensorMap& k, const CUtensorMap& v,
            cudaStream_t s) {
  using Cfg = MmaCfg<TK, DHP, NR>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  ATTNB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    ATTNB_CUDA(cudaFuncSetAttribute(seq_mma_kernel<TQ, TK, DHP, NR>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    configured.fetch_or(bit);
  }
  ATTNB_CUDA(launch_pdl(seq_mma_kernel<TQ, TK, DHP, NR>, dim3(ctas), dim3(kThreads), Cfg::SMEM, s,
                        k, v, a));
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
      if (a.rows == 8) {
        if (a.q.Dh <= 64) launch<TQ, TK, 64, 1>(a, ctas, k, v, s);
        else launch<TQ, TK, 128, 1>(a, ctas, k, v, s);
      } else {
        if (a.q.Dh <= 64) launch<TQ, TK, 64, 2>(a, ctas, k, v, s);
        else launch<TQ, TK, 128, 2>(a, ctas, k, v, s);
      }
    }
  };
  with_value_type(a.q.type, [&](auto tq) {
    if (a.pages.type == kE4M3) go(tq, std::integral_constant<int, kE4M3>{});
    else if (a.pages.type == kI8) go(tq, std::integral_constant<int, kI8>{});
    else go(tq, tq);
  });
}

}  // namespace attnb
