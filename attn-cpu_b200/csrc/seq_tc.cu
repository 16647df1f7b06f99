// seq_tc.cu -- K8: attention of packed query rows over packed keys or pages with
// tcgen05, for 16-bit queries and 16-bit or coded keys: whole prompts and chunks
// of new tokens.
//
// Bound by the tensor cores (4 * Dh operations per visible key and query head)
// and, next to them, by the exponentials: a 128 x 128 tile of weights takes 1024
// cycles of the SM's 16 exponentials a cycle, as many as its two products.
//
//   A CTA takes two tiles A, B of up to 128 rows of one KV head (the query heads
//   that share it lie side by side) and streams tiles of 128 keys by TMA; each
//   K and V tile serves both.  The two tiles run as chains, so that one's
//   products run under the other's softmax:
//       S = Q K^T (TMEM)  ->  softmax writes P over S (16 bits, TMEM)  ->  O += P V
//   with O in TMEM as well: 2 x (128 + 128) columns.  The chain goes in steps of
//   64 keys through two halves of its S columns, so that the scores of a step
//   are there before the softmax of the one before has ended.  V is read as it
//   lies in memory, keys by rows (an N-major operand).
//   Warp 0 loads; warps 1 and 2 issue the chains' scores and two others their
//   P V (a thread that waits for the one would hold up the other); warps 4-7 and
//   8-11 own one row of A or B per thread; one warp clears masked V values.
//   With codes, warps 12-15 turn them into f16 tiles and warp 17 looks at their
//   scales.
//   CTAs are persistent and walk the pieces of the schedule in seq.cuh.
//   Measured: prompts of 5000 and 8000 tokens, 32/8 heads, bf16, 750 us (970
//   TFLOP/s of visible work); chunks of 1024-2048 tokens over 6000-16000 int8 keys
//   1.03 ms (578 TFLOP/s: the conversion of codes shares the SM's issue slots; with
//   the scales in the f16 tiles 0.98 ms, and two roundings of every K and V more).
//
// 4-bit codes come as r (code - 8) 2^-19, exact in f16, 32 at a time of one group, with the
// dimensions of each eight in the order (0, 4, 1, 5, 2, 6, 3, 7), which Q follows on its way in
// and O on its way out.  The same chunks over 4-bit pages take 1.04 ms.
//
// The running maximum moves only when it grows by more than 8 (weights stay
// below 2^8, which f16 and bf16 hold); O and the sum are rescaled then.  Weights
// are rounded to 16 bits once, to nearest; maxima, sums and O are fp32.
//
// Codes: both products run in f16, over the codes as they are (exact).  Q is
// brought to [1, 2) by a power of two per row; a score is multiplied in fp32 by its
// key's K scale, and a weight by its V scale before it is rounded to f16.
// 64 keys share a power of two 2^E of their K scales, which goes into the row's
// scale, and 2^F of their V scales, which goes into the weights' exponent.
// The weights of the product have a reference rho of their own beside the sum's
// maximum m, 2^(s - m + F - rho), so that V may have any size and change it from
// block to block; 2^rho goes into the output.  The sum is theirs times 2^(rho - F).
// Some steps go key by key, scales of V in the exponent as in seq_mma.cu and a sum
// with exponentials of its own: where V scales are more than 2^6 apart (weights
// would lose bits to the larger ones) or V was much larger earlier in the piece, and
// where one is zero, not finite or next to the ends of fp32.  So a key that a row
// does not see changes nothing for it, whatever its scales are.  (Where all steps go
// so, chunks of 1024-2048 tokens over 6000-16000 keys take 1.6 to 1.8 ms.)
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "runtime.h"
#include "seq_elem.cuh"
#include "seq_pages.cuh"

namespace attnb {
namespace {

constexpr int BM = 128;
constexpr int BN = 128;  // keys of a tile in shared memory
constexpr int BS = 64;   // keys of a step
constexpr float kRescaleGap = 8.f;
constexpr float kNoRho = -1e30f;  // no weight so far: any exponent is above it
// How much larger V of an earlier step may be (in powers of two) where a step takes
// its sum from the product's weights.  With hi the greatest F so far rho <= hi + 8
// (no score is more than 8 above m), so the factor 2^(rho - F) stays below 2^40
// and no weight that counts has vanished.  (A small factor is harmless: the sum holds
// the 1 of the row's best key.)
constexpr int kSpread = 24;
constexpr int kPoison = 6;  // pieces that warp 3 may be ahead of the outputs, and more

template <bool CODED, int DHP>
struct TcCfg {
  static constexpr int THREADS = CODED ? 576 : 448;
  static constexpr int PV_A = CODED ? 3 : 12, PV_B = CODED ? 16 : 13;  // warps that issue P V
  static constexpr int SCALER = 17;              // codes: warp that looks at the scales
  static constexpr int CHUNKS = DHP / 64;        // 128-byte pieces of a 16-bit row
  static constexpr int CHUNK = BN * 128;         // 16 KB: 128 rows x 64 columns
  static constexpr int TILE = CHUNKS * CHUNK;    // Q, K or V
  static constexpr int K_ST = DHP == 128 ? 2 : 4;
  static constexpr int V_ST = DHP == 128 ? 2 : 4;
  static constexpr int RAW_ST = 3;               // codes: half tiles of 64 keys
  static constexpr int RAW = 64 * 128 + 1024;    // codes, then K and V scales
  static constexpr int OFF_K = 2 * TILE;
  static constexpr int OFF_V = OFF_K + K_ST * TILE;
  static constexpr int OFF_RAW = OFF_V + V_ST * TILE;
  static constexpr int OFF_X = OFF_RAW + (CODED ? RAW_ST * RAW : 0);
  // Codes: what the softmax needs of a tile, by half: E's and F's powers of two and
  // the keys' scales over them; where the keys go one by one both are NaN and K
  // scales and logarithms of V scales follow.  Else poison.  When a tile's raw half is
  // there, V of the tile before the last has been converted, so the softmax is at
  // most V_ST tiles behind that one.
  static constexpr int SCALES = V_ST + 2;
  static constexpr int XHEAD = 4;  // floats
  static constexpr int XTILE = XHEAD * 4 + 2 * 128 * 4;
  // 2 KB per softmax warp to write outputs through; with codes Q's place serves.
  static constexpr int OFF_OUT = OFF_X + (CODED ? SCALES * XTILE : kPoison * 3 * DHP * 4);
  static constexpr int SMEM = OFF_OUT + (CODED ? 0 : 8 * 2048) + 1024;
  static_assert(SMEM <= 227 * 1024 - 1024, "shared memory budget");
};

template <int TQ>
__device__ __forceinline__ bool any_not_finite(const uint4& x) {
  constexpr uint32_t mask = TQ == kBF16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t unit = TQ == kBF16 ? 0x00800080u : 0x04000400u;
  return ((((x.x & mask) + unit) | ((x.y & mask) + unit) | ((x.z & mask) + unit) |
           ((x.w & mask) + unit)) &
          0x80008000u) != 0;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A step of the softmax over codes whose keys go by scales of their own (`keys`:
// K scales, logarithms of V scales): largest exponent of the step.  Rare, so
// that it may take three passes over the scores in TMEM; a call keeps it from
// costing the other steps registers.
struct RowState {
  float m, l, rho, alpha;
  bool need;
};
__device__ __noinline__ float step_by_key(RowState& st, uint32_t sb, int kb0, int seen,
                                          float scale, const float4* keys) {
  float m = st.m, l = st.l, rho = st.rho, top = -INFINITY, best = -INFINITY;
  uint32_t s[32];
  // Exponents of 32 keys in place of their scores.
  auto load = [&](int k0) {
    tmem_ld32(sb + k0, s);
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      const float4 x = keys[(k0 + k) >> 2];
      const float ks[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[k + e] = kb0 + k0 + k + e >= seen
                       ? __float_as_uint(-INFINITY)
                       : __float_as_uint(__uint_as_float(s[k + e]) * (scale * ks[e]));
    }
  };
#pragma unroll 1
  for (int k0 = 0; k0 < BS; k0 += 32) {
    load(k0);
#pragma unroll
    for (int k = 0; k < 32; k += 2)
      top = max3_nan(top, __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
    tmem_st32(sb + k0, s);
  }
  tmem_wait_st();
  if (top - m > kRescaleGap) {
    if (m != -INFINITY) rho -= top - m;
    l *= fast_exp2(m - top);
    m = top;
  }
  const float ref = m == -INFINITY ? 0.f : m;
  // The product's exponents but for rho; the scale of a masked key may be anything.
  auto product = [&](int k0, int k, float (&u)[4]) {
    const float4 x = keys[(BS + k0 + k) >> 2];
    const float lv[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = __uint_as_float(s[k + e]);
      u[e] = t == -INFINITY ? t : t - ref + lv[e];
    }
  };
#pragma unroll 1
  for (int k0 = 0; k0 < BS; k0 += 32) {
    tmem_ld32(sb + k0, s);
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      float u[4];
      product(k0, k, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l += fast_exp2(__uint_as_float(s[k + e]) - ref);
        best = fmaxf(best, u[e]);
      }
    }
  }
  st.need = best - rho > kRescaleGap;
  if (st.need) {
    st.alpha = fast_exp2(rho - best);
    rho = best;
  }
#pragma unroll 1
  for (int k0 = 0; k0 < BS; k0 += 32) {
    tmem_ld32(sb + k0, s);
    uint32_t p[16];
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      float u[4];
      product(k0, k, u);
      p[k >> 1] = pack_f16(fast_exp2(u[0] - rho), fast_exp2(u[1] - rho));
      p[(k >> 1) + 1] = pack_f16(fast_exp2(u[2] - rho), fast_exp2(u[3] - rho));
    }
    tmem_st16(sb + (k0 >> 1), p);  // over scores that have been read
  }
  st.m = m;
  st.l = l;
  st.rho = rho;
  return top;
}

template <int TQ, int TK, int DHP>
__global__ void __launch_bounds__(TcCfg<elem_coded(TK), DHP>::THREADS, 1)
    seq_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ SeqAttnArgs a,
                  const bool qtma, const bool qvec, const bool ovec) {
  constexpr bool CODED = elem_coded(TK), I4 = TK == kI4;
  using Cfg = TcCfg<CODED, DHP>;
  using EQ = elem_t<TQ>;
  constexpr bool BF16 = TQ == kBF16 && !CODED;  // type of the products
  constexpr int KST = Cfg::K_ST, VST = Cfg::V_ST, RST = Cfg::RAW_ST;
  constexpr uint32_t IDESC_S = idesc_f16(BM, BS, BF16, false);
  constexpr uint32_t IDESC_PV = idesc_f16(BM, DHP, BF16, true);

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t kfull[KST], kempty[KST], vfull[VST], vempty[VST], vfix[VST];
  __shared__ __align__(8) uint64_t rfull[RST], rempty[RST];
  __shared__ __align__(8) uint64_t q_bar[2], q_free[2], s_bar[2][2], p_bar[2][2], pv_bar[2][2],
      done_bar[4];
  __shared__ SeqShared sh;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int poison_set[kPoison];
  __shared__ int outputs[2];  // warps' outputs written, per chain

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t* const mem = smem_raw + (base - smem_addr(smem_raw));
  volatile int* abort_p = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    outputs[0] = outputs[1] = 0;
    for (int i = 0; i < KST; ++i) {
      mbar_init(smem_addr(&kfull[i]), CODED ? 5 : 1);
      mbar_init(smem_addr(&kempty[i]), 2);
    }
    for (int i = 0; i < VST; ++i) {
      mbar_init(smem_addr(&vfull[i]), CODED ? 4 : 1);
      mbar_init(smem_addr(&vempty[i]), 2);
      mbar_init(smem_addr(&vfix[i]), 1);
    }
    for (int i = 0; i < RST; ++i) {
      mbar_init(smem_addr(&rfull[i]), 1);
      mbar_init(smem_addr(&rempty[i]), 5);
    }
    for (int c = 0; c < 2; ++c) {
      mbar_init(smem_addr(&q_bar[c]), qtma ? 1 : 4);
      mbar_init(smem_addr(&q_free[c]), 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_addr(&s_bar[c][i]), 1);
        mbar_init(smem_addr(&p_bar[c][i]), 4);
        mbar_init(smem_addr(&pv_bar[c][i]), 1);
      }
      mbar_init(smem_addr(&done_bar[c]), 1);
      mbar_init(smem_addr(&done_bar[2 + c]), 1);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (threadIdx.x < kPoison) poison_set[threadIdx.x] = 0;
  if constexpr (!CODED) {
    int* ps = reinterpret_cast<int*>(mem + Cfg::OFF_X);
    for (int i = threadIdx.x; i < kPoison * 3 * DHP; i += Cfg::THREADS) ps[i] = INT_MAX;
  }
  grid_dep_wait();
  SeqPlace place;
  const bool any = seq_locate(a, sh, place);  // synchronises the block
  if (threadIdx.x < 32) seq_write_split(a, any, place);
  if (!any) return;
  if (warp == 1) {
    tmem_alloc(smem_addr(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  const int half = a.rows >> 1;  // rows of chain A's tile
  SeqIter it;
  it.start(place);
  SeqPiece w{};
  // Steps of the piece that chain c takes: the first ones.
  auto steps_of = [&](int c) {
    const int rows = min(w.rows - c * half, half);
    if (rows <= 0) return 0;
    int seen = w.s.L;
    if (a.causal) seen = seq_row_seen(a, w.s, w.row0 + c * half + rows - 1);
    const int n = max(1, (max(seen, 0) + BS - 1) / BS);
    return min(n, 2 * w.j1) - min(n, 2 * w.j0);
  };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) {
    const bool got = mbar_wait_quick(smem_addr(bar), parity, abort_p, a.status);
    return __all_sync(0xffffffffu, got) != 0;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- loader
    const bool paged = a.pages.k != nullptr;
    const int shift = a.pages.page_shift, mask = (1 << shift) - 1;
    PageWindow win;
    bool ok = true;
    if constexpr (CODED) {
      Ring<RST> ring;
      const int box = min(1 << shift, 64), copies = 64 / box;
      const int row = I4 ? a.q.Dh / 2 : 128;  // bytes of a key as it comes
      while (ok && it.next(a, w)) {
        const int used = (w.s.L + mask) >> shift;
        for (int hj = 4 * w.j0; ok && hj < 4 * w.j1; ++hj) {
          // Half tiles: K, K, V, V of each tile.
          const bool is_v = (hj & 2) != 0;
          ok = warp_wait(&rempty[ring.stage], ring.phase ^ 1u);
          if (!ok) break;
          const uint32_t st = base + Cfg::OFF_RAW + ring.stage * Cfg::RAW;
          const uint32_t bar = smem_addr(&rfull[ring.stage]);
          const int key0 = (hj >> 2) * BN + (hj & 1) * 64;
          int page = 0;  // of this lane's copy
          uint32_t bytes = 64 * row;
          for (int i = 0; i < copies; ++i) {
            const int p = win.get<false>(a, w, (key0 + i * box) >> shift, used);
            if (lane == i) page = p;
            if (p < a.pages.num_pages) bytes += ((is_v ? 0 : 2) + (I4 ? 1 : 0)) * box * 4;
          }
          const int my_key = key0 + lane * box;
          const bool there = page < a.pages.num_pages;
          if (lane < copies && !is_v && !there) {  // no such page: codes 0 with scales of 0
            float* sc = reinterpret_cast<float*>(mem + Cfg::OFF_RAW + ring.stage * Cfg::RAW +
                                                 64 * 128);
            for (int k = 0; k < box; ++k) sc[lane * box + k] = sc[64 + lane * box + k] = 0.f;
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
          __syncwarp();
          if (lane < copies) {
            const int in_page = my_key & mask;
            tma_load_4d(st + lane * box * row, is_v ? &tmV : &tmK, bar, 0,
                        I4 ? in_page * row / 128 : in_page, w.h, page);
            const int64_t at = (((int64_t)page * a.pages.H + w.h) << shift) + (my_key & mask);
            if (I4 && there)
              bulk_load(st + 64 * 128 + 512 + lane * box * 4,
                        (is_v ? a.pages.v_group : a.pages.k_group) + at * 4, box * 4, bar);
            if (!is_v && there) {
              bulk_load(st + 64 * 128 + lane * box * 4, a.pages.k_scale + at, box * 4, bar);
              bulk_load(st + 64 * 128 + 256 + lane * box * 4, a.pages.v_scale + at, box * 4, bar);
            }
          }
          ring.note_issue();
          ring.advance();
        }
      }
      if (lane == 0)
        for (int i = 0; i < RST; ++i)
          if (ring.issued_mask & (1u << i))
            drain_wait(smem_addr(&rfull[i]), (ring.issued_parity >> i) & 1u, a.status);
    } else {
      Ring<KST> rk;
      Ring<VST> rv;
      const int box = paged ? min(1 << shift, BN) : BN, copies = BN / box;
      // One tile of K or V: `copies` lanes issue their copies.
      auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int j, int used) {
        int page = 0;
        if (paged)
          for (int i = 0; i < copies; ++i) {
            const int p = win.get<false>(a, w, (j * BN + i * box) >> shift, used);
            if (lane == i) page = p;
          }
        if (lane == 0) mbar_arrive_expect_tx(bar, Cfg::TILE);
        __syncwarp();
        if (lane < copies) {
          const int key = j * BN + lane * box;
#pragma unroll
          for (int c = 0; c < Cfg::CHUNKS; ++c) {
            const uint32_t to = dst + c * Cfg::CHUNK + lane * box * 128;
            if (paged) tma_load_4d(to, map, bar, c * 64, key & mask, w.h, page);
            else tma_load_3d(to, map, bar, c * 64, w.h, w.s.k0 + key);
          }
        }
      };
      // Q of chain c, once the products of the piece before are done with it.
      uint32_t qloads[2] = {0, 0};
      auto load_q = [&](int c) {
        if (!warp_wait(&q_free[c], (qloads[c] & 1) ^ 1)) return false;
        ++qloads[c];
        if (lane == 0) {
          const uint32_t bar = smem_addr(&q_bar[c]);
          mbar_arrive_expect_tx(bar, Cfg::CHUNKS * half * 128);
          const int token = w.s.q0 + (w.row0 + c * half) / a.G;
#pragma unroll
          for (int k = 0; k < Cfg::CHUNKS; ++k)
            tma_load_3d(base + c * Cfg::TILE + k * Cfg::CHUNK, &tmQ, bar, k * 64, w.h * a.G, token);
        }
        return true;
      };
      while (ok && it.next(a, w)) {
        const int used = paged ? (w.s.L + mask) >> shift : 0;
        for (int j = w.j0; ok && j < w.j1; ++j) {
          ok = warp_wait(&kempty[rk.stage], rk.phase ^ 1u);
          if (!ok) break;
          load(&tmK, base + Cfg::OFF_K + rk.stage * Cfg::TILE, smem_addr(&kfull[rk.stage]), j, used);
          rk.note_issue();
          rk.advance();
          if (qtma && j == w.j0) {
            for (int c = 0; ok && c < 2; ++c)
              if (steps_of(c) > 0) ok = load_q(c);
            if (!ok) break;
          }
          ok = warp_wait(&vempty[rv.stage], rv.phase ^ 1u);
          if (!ok) break;
          load(&tmV, base + Cfg::OFF_V + rv.stage * Cfg::TILE, smem_addr(&vfull[rv.stage]), j, used);
          rv.note_issue();
          rv.advance();
        }
      }
      // Every copy issued lands before the CTA may exit.
      if (lane == 0) {
        for (int i = 0; i < KST; ++i)
          if (rk.issued_mask & (1u << i))
            drain_wait(smem_addr(&kfull[i]), (rk.issued_parity >> i) & 1u, a.status);
        for (int i = 0; i < VST; ++i)
          if (rv.issued_mask & (1u << i))
            drain_wait(smem_addr(&vfull[i]), (rv.issued_parity >> i) & 1u, a.status);
        for (int c = 0; c < 2; ++c)
          if (qloads[c] > 0) drain_wait(smem_addr(&q_bar[c]), (qloads[c] - 1) & 1u, a.status);
      }
    }
  } else if (warp <= 2) {
    // ------------------------------------ scores of chain c: the whole warp keeps
    // step, one lane issues
    const int c = warp - 1;
    const uint32_t sbuf = tmem + c * BN;
    Ring<KST> rk;
    uint32_t g = 0, qphase = 0;  // step g uses half g & 1 of S
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && warp_wait(bar, parity);
      return ok;
    };
    const uint64_t qd = sdesc_kmajor_sw128(base + c * Cfg::TILE);
    while (ok && it.next(a, w)) {
      const int n = steps_of(c);
      if (n > 0) {
        if (!wait(&q_bar[c], qphase)) break;
        qphase ^= 1;
      }
      for (int i = 0; i < n; ++i, ++g) {
        if (!(i & 1) && !wait(&kfull[rk.stage], rk.phase)) break;
        // They overwrite the weights of step g - 2, whose product has to be done.
        if (g >= 2 && !wait(&pv_bar[c][g & 1], ((g >> 1) - 1) & 1)) break;
        tc_fence_after();
        const uint64_t kd = sdesc_kmajor_sw128(base + Cfg::OFF_K + rk.stage * Cfg::TILE +
                                               (i & 1) * BS * 128);
        const bool tile_end = (i & 1) || i == n - 1;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < DHP / 16; ++k) {
            const uint64_t at = ((k >> 2) * Cfg::CHUNK + (k & 3) * 32) >> 4;
            mma_f16(sbuf + (g & 1) * BS, qd + at, kd + at, IDESC_S, k != 0 ? 1u : 0u);
          }
          mma_commit(smem_addr(&s_bar[c][g & 1]));
          if (tile_end) mma_commit(smem_addr(&kempty[rk.stage]));
          if (i == n - 1) mma_commit(smem_addr(&q_free[c]));
        }
        __syncwarp();
        if (tile_end) rk.advance();
      }
      // Tiles that only the other chain takes.
      for (int j = (n + 1) / 2; ok && j < w.j1 - w.j0; ++j) {
        if (!wait(&kfull[rk.stage], rk.phase)) break;
        if (lane == 0) mbar_arrive(smem_addr(&kempty[rk.stage]));
        rk.advance();
      }
    }
    // Every product issued completes before TMEM is released.
    __syncwarp();
    if (elect_one()) mma_commit(smem_addr(&done_bar[c]));
    __syncwarp();
    drain_wait(smem_addr(&done_bar[c]), 0, a.status);
  } else if (warp == Cfg::PV_A || warp == Cfg::PV_B) {
    // ------------------------------------------------------- P V of chain c
    const int c = warp == Cfg::PV_A ? 0 : 1;
    const uint32_t sbuf = tmem + c * BN;
    const uint32_t obuf = tmem + 2 * BN + c * 128;
    Ring<VST> rv;
    uint32_t g = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && warp_wait(bar, parity);
      return ok;
    };
    while (ok && it.next(a, w)) {
      const int n = steps_of(c);
      const int seen_max = seq_row_seen(a, w.s, w.row0 + w.rows - 1);
      for (int i = 0; i < n; ++i, ++g) {
        if (!(i & 1)) {
          if (!wait(&vfull[rv.stage], rv.phase)) break;
          if (!CODED && !wait(&vfix[rv.stage], rv.phase)) break;
        }
        if (!wait(&p_bar[c][g & 1], (g >> 1) & 1)) break;
        tc_fence_after();
        const uint64_t vd = sdesc_mnmajor_sw128(
            base + Cfg::OFF_V + rv.stage * Cfg::TILE + (i & 1) * BS * 128, Cfg::CHUNK);
        const bool tile_end = (i & 1) || i == n - 1;
        // Keys behind the last one that a row of the item sees are not read.
        const int left = seen_max - w.j0 * BN - i * BS;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < BS / 16; ++k)
            if (k == 0 || k * 16 < left) mma_f16_ts(obuf, sbuf + (g & 1) * BS + k * 8, vd + k * (2048 >> 4), IDESC_PV,
                       (i | k) != 0 ? 1u : 0u);
          mma_commit(smem_addr(&pv_bar[c][g & 1]));
          if (tile_end) mma_commit(smem_addr(&vempty[rv.stage]));
        }
        __syncwarp();
        if (tile_end) rv.advance();
      }
      for (int j = (n + 1) / 2; ok && j < w.j1 - w.j0; ++j) {
        if (!wait(&vfull[rv.stage], rv.phase)) break;
        if (!CODED && !wait(&vfix[rv.stage], rv.phase)) break;
        if (lane == 0) mbar_arrive(smem_addr(&vempty[rv.stage]));
        rv.advance();
      }
    }
    __syncwarp();
    if (elect_one()) mma_commit(smem_addr(&done_bar[2 + c]));
    __syncwarp();
    drain_wait(smem_addr(&done_bar[2 + c]), 0, a.status);
  } else if (warp == 3) {
    // ------------------------------------------ values of V that a mask hides
    if constexpr (!CODED) {
      Ring<VST> rv;
      bool ok = true;
      int piece = 0;
      while (ok && it.next(a, w)) {
        const int at = piece % kPoison;
        int* ps = reinterpret_cast<int*>(mem + Cfg::OFF_X) + at * 3 * DHP;
        // Piece - kPoison had the place before; its outputs come first.
        auto settle = [&] {
          const uint64_t t0 = globaltimer();
          const int want = 4 * (piece - kPoison + 1);
          while (*(volatile int*)&outputs[0] < want || *(volatile int*)&outputs[1] < want) {
            if (*abort_p) break;
            if (globaltimer() - t0 > ATTNB_WAIT_LIMIT_NS) {
              *abort_p = 1;
              raise_timeout(a.status);
              break;
            }
          }
          __syncwarp();
        };
        if (*(volatile int*)&poison_set[at]) {
          settle();
          for (int i = lane; i < 3 * DHP; i += 32) ps[i] = INT_MAX;
          if (lane == 0) poison_set[at] = 0;
          __syncwarp();
        }
        const int seen_min = seq_row_seen(a, w.s, w.row0);
        for (int j = w.j0; j < w.j1; ++j) {
          ok = warp_wait(&vfull[rv.stage], rv.phase);
          if (!ok) break;
          const int key0 = j * BN;
          if (key0 + BN > seen_min) {
            uint8_t* v = mem + Cfg::OFF_V + rv.stage * Cfg::TILE;
            // Rows that some row of the item does not see, up to the last one
            // that the products read (16 at a time).
            const int from = max(0, seen_min - key0);
            const int seen_max = max(seq_row_seen(a, w.s, w.row0 + w.rows - 1), 1);
            const int last = min(BN, ((seen_max + 15) & ~15) - key0);
            const int units = max(0, last - from) * 8;  // per chunk
            const int gone = w.s.L - key0;  // rows from here on are not the sequence's
            bool found = false;
            for (int i0 = lane; i0 < units; i0 += 128) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * 32, r = from + (i >> 3), u = i & 7;
                if (i >= units) continue;
#pragma unroll
                for (int ch = 0; ch < Cfg::CHUNKS; ++ch) {
                  uint4* p = reinterpret_cast<uint4*>(v + ch * Cfg::CHUNK + sw128(r, u));
                  if (r >= gone) *p = make_uint4(0, 0, 0, 0);
                  else found |= any_not_finite<TQ>(*p);
                }
              }
            }
            const bool hit = __any_sync(0xffffffffu, found);
            if (hit) settle();
            if (hit)
              for (int i = lane; i < units; i += 32) {
                const int r = from + (i >> 3), u = i & 7;
                for (int ch = 0; ch < Cfg::CHUNKS; ++ch) {
                  uint4* p = reinterpret_cast<uint4*>(v + ch * Cfg::CHUNK + sw128(r, u));
                  uint4 x = *p;
                  EQ* e = reinterpret_cast<EQ*>(&x);
#pragma unroll
                  for (int b = 0; b < 8; ++b) {
                    const float f = to_float(e[b]);
                    if (fabsf(f) <= 3.402823466e38f) continue;
                    const int kind = f != f ? 0 : (f > 0.f ? 1 : 2);
                    atomicMin(&ps[kind * DHP + ch * 64 + u * 8 + b], key0 + r);
                    from_float(0.f, e[b]);
                  }
                  *p = x;
                }
              }
            if (hit) poison_set[at] = 1;
            fence_proxy_async_smem();  // the products read V through the async proxy
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&vfix[rv.stage]));
          rv.advance();
        }
        ++piece;
      }
    }
  } else if (warp == Cfg::SCALER) {
    // ------------------------------------ scales of 64 keys: what they share
    if constexpr (CODED) {
      Ring<RST> ring;
      Ring<KST> rk;
      bool ok = true;
      uint32_t tile = 0;
      while (ok && it.next(a, w)) {
        int hi = INT_MIN;  // V's greatest power of two in the piece so far
        for (int j = w.j0; ok && j < w.j1; ++j, ++tile) {
#pragma unroll 1
          for (int part = 0; part < 4; ++part) {  // as the loader: K, K, V, V
            ok = warp_wait(&rfull[ring.stage], ring.phase);
            if (!ok) break;
            if (part < 2) {
              const float* sc = reinterpret_cast<const float*>(mem + Cfg::OFF_RAW +
                                                               ring.stage * Cfg::RAW + 64 * 128);
              float* xt = reinterpret_cast<float*>(mem + Cfg::OFF_X +
                                                   (tile % Cfg::SCALES) * Cfg::XTILE);
              const int left = w.s.L - j * BN - part * 64;
              const bool in0 = lane < left, in1 = lane + 32 < left;
              // Scales past the sequence may be anything, and do not count.
              const float k0 = in0 ? sc[lane] : 0.f, k1 = in1 ? sc[lane + 32] : 0.f;
              const float v0 = in0 ? sc[lane + 64] : 0.f, v1 = in1 ? sc[lane + 96] : 0.f;
              // Largest and smallest by their bits: those of an infinity or a NaN (and
              // of a negative number) are above all others.  K scales of 0 take no part.
              auto bits = [](float x) { return __float_as_uint(x); };
              const uint32_t kmax = __reduce_max_sync(0xffffffffu, max(bits(k0), bits(k1)));
              const uint32_t vmax = __reduce_max_sync(0xffffffffu, max(bits(v0), bits(v1)));
              const uint32_t kmin = __reduce_min_sync(0xffffffffu, min(bits(k0) - 1u, bits(k1) - 1u));
              const uint32_t vmin =
                  __reduce_min_sync(0xffffffffu, min(in0 ? bits(v0) : ~0u, in1 ? bits(v1) : ~0u));
              constexpr uint32_t kLow = 0x0d800000u, kHigh = 0x71800000u;  // 2^-100, 2^100
              bool wide = false;
              if (left > 0) {
                const int e = (int)(vmax >> 23);
                hi = max(hi, e);
                wide = kmax > kHigh || kmin < kLow || vmax > kHigh || vmin < kLow ||
                       vmax - vmin > (6u << 23) || hi - e > kSpread;
              }
              // The largest scales' powers of two (as in row_scale), inverted.
              const float ke = row_scale(__uint_as_float(kmax)), ve = row_scale(__uint_as_float(vmax));
              if (lane == 0) {
                const float own = __int_as_float(0x7fffffff);
                xt[part] = wide ? own : 1.f / ke;
                xt[2 + part] = wide ? own : (float)(127 - (int)(bits(ve) >> 23));
              }
              float* keys = xt + Cfg::XHEAD + part * 128;
              // (No factor of 0: a masked -inf stays one.)
              auto kscale = [&](float x) { return wide ? x : fmaxf(x * ke, 0x1p-126f); };
              auto vscale = [&](float x) { return wide ? __log2f(x) : x * ve; };
              keys[lane] = kscale(k0);
              keys[lane + 32] = kscale(k1);
              keys[lane + 64] = vscale(v0);
              keys[lane + 96] = vscale(v1);
            }
            __syncwarp();
            if (lane == 0) {
              if (part == 1) mbar_arrive(smem_addr(&kfull[rk.stage]));
              mbar_arrive(smem_addr(&rempty[ring.stage]));
            }
            ring.advance();
          }
          rk.advance();
        }
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------ codes to f16 tiles
    if constexpr (CODED) {
      const int t = threadIdx.x - 384, row = t & 63, part = t >> 6;  // half the row's units
      Ring<RST> ring;
      Ring<KST> rk;
      Ring<VST> rv;
      bool ok = true;
      uint32_t tile = 0;
      while (ok && it.next(a, w)) {
        for (int j = w.j0; ok && j < w.j1; ++j, ++tile) {
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            ok = ok && (kv ? warp_wait(&vempty[rv.stage], rv.phase ^ 1u)
                           : warp_wait(&kempty[rk.stage], rk.phase ^ 1u));
            uint8_t* to = mem + (kv ? Cfg::OFF_V + rv.stage * Cfg::TILE
                                    : Cfg::OFF_K + rk.stage * Cfg::TILE);
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
              ok = ok && warp_wait(&rfull[ring.stage], ring.phase);
              if (!ok) break;
              const uint8_t* from = mem + Cfg::OFF_RAW + ring.stage * Cfg::RAW;
              const int r = hf * 64 + row;
              const bool gone = row >= w.s.L - j * BN - hf * 64;  // stale
              if constexpr (I4) {
                // 32 codes of one group; pairs of dimensions (0, 4), (1, 5), (2, 6), (3, 7) of
                // each eight, the order that Q and the outputs follow.
                const uint32_t factors =
                    gone ? 0u : reinterpret_cast<const uint32_t*>(from + 64 * 128 + 512)[row];
#pragma unroll 1
                for (int i = 0; i < DHP / 64; ++i) {
                  const int u = part * (DHP / 64) + i;
                  const uint4 x = *reinterpret_cast<const uint4*>(from + i4_unit(row * (a.q.Dh / 32) + u));
                  const I4Factors f = i4_factors(__byte_perm(factors >> (8 * u), 0, 0x4040));
                  const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                  uint8_t* ch = to + (u >> 1) * Cfg::CHUNK;
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const uint32_t lo = xs[k], hi = xs[k] >> 8;
                    *reinterpret_cast<uint4*>(ch + sw128(r, (u & 1) * 4 + k)) =
                        make_uint4(fma_f16x2(lo & kI4Low, f.low, f.add),
                                   fma_f16x2(lo & kI4High, f.high, f.add),
                                   fma_f16x2(hi & kI4Low, f.low, f.add),
                                   fma_f16x2(hi & kI4High, f.high, f.add));
                  }
                }
              } else
#pragma unroll 1  // (the instruction cache, see the softmax)
              for (int i = 0; i < DHP / 32; ++i) {
                const int u = part * (DHP / 32) + i;  // 16 codes
                uint4 x = *reinterpret_cast<const uint4*>(from + sw128(row, u));
                if (gone) x = make_uint4(0, 0, 0, 0);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                uint32_t y[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) codes_to_f16<TK>(xs[k], y[2 * k], y[2 * k + 1]);
                uint8_t* ch = to + (u >> 2) * Cfg::CHUNK;
                *reinterpret_cast<uint4*>(ch + sw128(r, (u & 3) * 2)) =
                    make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(ch + sw128(r, (u & 3) * 2 + 1)) =
                    make_uint4(y[4], y[5], y[6], y[7]);
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_addr(&rempty[ring.stage]));
              ring.advance();
            }
            if (!ok) break;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(kv ? smem_addr(&vfull[rv.stage]) : smem_addr(&kfull[rk.stage]));
            if (kv) rv.advance();
            else rk.advance();
          }
        }
      }
    }
  } else {
    // ------------------------------------------------ softmax / output, chain c
    const int c = warp >= 8 ? 1 : 0;
    const int quarter = warp & 3;  // TMEM lanes [32 * quarter, +32)
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t srow = tmem + lane_off + c * BN;
    const uint32_t orow = tmem + lane_off + 2 * BN + c * 128;
    uint32_t g = 0, tile0 = 0;  // steps of this chain; tiles of the CTA
    bool ok = true;
    int piece = 0;
    for (; it.next(a, w); ++piece) {
      const int n = steps_of(c);
      const int rows = min(w.rows - c * half, half);  // of this chain, <= 0: none
      const bool mine = r < rows;
      const int row = w.row0 + c * half + r;
      const int seen = mine ? seq_row_seen(a, w.s, row) : 0;
      const int64_t token = w.s.q0 + row / a.G;
      const int head = w.h * a.G + row % a.G;
      float m = -INFINITY, l = 0.f, scale = a.scale_log2;
      float mraw = 0.f;    // 16-bit keys: m as a score, 0 while there is none
      float rho = kNoRho;  // codes: the product's reference, relative to m
      if (ok && n > 0 && !qtma) {
        // ---- Q: this thread's row into its tile (the products that read the
        // row before are done: the last S of the piece before has been seen)
        uint8_t* qt = mem + c * Cfg::TILE;
        const EQ* p = static_cast<const EQ*>(a.q.data) + token * a.q.sT + (int64_t)head * a.q.sH;
        auto unit = [&](int u) {  // 8 values
          uint4 x = make_uint4(0, 0, 0, 0);
          if (mine) {
            if (qvec) {
              if (u * 8 < a.q.Dh) x = __ldg(reinterpret_cast<const uint4*>(p) + u);
            } else {
              EQ* e = reinterpret_cast<EQ*>(&x);
#pragma unroll
              for (int b = 0; b < 8; ++b)
                if (u * 8 + b < a.q.Dh) e[b] = p[u * 8 + b];
            }
          }
          return x;
        };
        float f = 1.f;
        if constexpr (CODED) {
          float top = 0.f;
#pragma unroll 4
          for (int u = 0; u < DHP / 8; ++u) {
            const uint4 x = unit(u);
            const EQ* e = reinterpret_cast<const EQ*>(&x);
#pragma unroll
            for (int b = 0; b < 8; ++b) top = fmaxf(top, fabsf(to_float(e[b])));
          }
          f = I4 ? i4_row_scale(top) : row_scale(top);
          scale = I4 ? a.scale_log2 * (kI4Unit / kI4Rows) / (f / kI4Rows) : a.scale_log2 / f;
        }
#pragma unroll 4
        for (int u = 0; u < DHP / 8; ++u) {
          uint4 x = unit(u);
          if constexpr (CODED) {
            const EQ* e = reinterpret_cast<const EQ*>(&x);
            auto two = [&](int b) {  // 4-bit codes: dimensions b / 2 and b / 2 + 4
              return pack_f16(to_float(e[I4 ? b / 2 : b]) * f,
                              to_float(e[I4 ? b / 2 + 4 : b + 1]) * f);
            };
            x = make_uint4(two(0), two(2), two(4), two(6));
          }
          *reinterpret_cast<uint4*>(qt + (u >> 3) * Cfg::CHUNK + sw128(r, u & 7)) = x;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&q_bar[c]));
      }
      for (int i = 0; i < n; ++i, ++g) {
        if (ok) ok = warp_wait(&s_bar[c][g & 1], (g >> 1) & 1);
        if (!ok) continue;
        tc_fence_after();
        const uint32_t sb = srow + (g & 1) * BS;
        const int kb0 = w.j0 * BN + i * BS;
        // Masks only occur in some steps; a warp applies them only there.
        const bool masked = __any_sync(0xffffffffu, kb0 + BS > seen);
        const float* xt = reinterpret_cast<const float*>(
            mem + Cfg::OFF_X + (CODED ? ((tile0 + (i >> 1)) % Cfg::SCALES) * Cfg::XTILE : 0));
        float top, alpha = 1.f;  // largest exponent of the step; what O is multiplied by
        bool rescale;            // in some row of the warp
        if constexpr (CODED) {
          // The code of this loop and of the conversion share the schedulers'
          // instruction caches and are bound by them (unrolled, 4.4 of the 13 cycles a warp
          // took for an instruction were waits for the instruction): so 32 scores at a
          // time in loops, read from TMEM twice, and masks in a pass of their own.
          uint32_t s[32];
          const float f = xt[2 + (i & 1)];
          const float4* keys = reinterpret_cast<const float4*>(xt + Cfg::XHEAD + (i & 1) * 128);
          if (f == f) {
            if (masked) {
#pragma unroll 1
              for (int k0 = 0; k0 < BS; k0 += 32) {
                tmem_ld32(sb + k0, s);
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (kb0 + k0 + k >= seen) s[k] = __float_as_uint(-INFINITY);
                tmem_st32(sb + k0, s);
              }
              tmem_wait_st();
            }
            auto two = [&](int k) {
              return pack_f32x2(__uint_as_float(s[k]), __uint_as_float(s[k + 1]));
            };
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
            for (int k0 = 0; k0 < BS; k0 += 32) {
              tmem_ld32(sb + k0, s);
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 ks = keys[(k0 + k) >> 2];
                float s0, s1, s2, s3;
                unpack_f32x2(mul_f32x2(two(k), pack_f32x2(ks.x, ks.y)), s0, s1);
                unpack_f32x2(mul_f32x2(two(k + 2), pack_f32x2(ks.z, ks.w)), s2, s3);
                mx[0] = max3_nan(mx[0], s0, s1);
                mx[1] = max3_nan(mx[1], s2, s3);
                s[k] = __float_as_uint(s0);
                s[k + 1] = __float_as_uint(s1);
                s[k + 2] = __float_as_uint(s2);
                s[k + 3] = __float_as_uint(s3);
              }
              tmem_st32(sb + k0, s);
            }
            tmem_wait_st();
            const float smax = max_nan(mx[0], mx[1]);
            // (No factor below the smallest normal number: a masked -inf stays one.)
            const float mul = fmaxf(scale * xt[i & 1], 0x1p-126f);
            top = smax * mul;
            if (top - m > kRescaleGap) {
              if (m != -INFINITY) rho -= top - m;
              l *= fast_exp2(m - top);
              m = top;
            }
            const float best = top == -INFINITY ? top : top - m + f;
            const bool need = best - rho > kRescaleGap;
            rescale = __any_sync(0xffffffffu, need);
            if (need) {
              alpha = fast_exp2(rho - best);
              rho = best;
            }
            // Score to exponent: (s - smax) * mul + shift; the maximum's own is exact
            // whatever its magnitude.
            const float sref = smax == -INFINITY ? 0.f : smax, shift = best - rho;
            const uint64_t mul2 = pack_f32x2(mul, mul), ref2 = pack_f32x2(-sref, -sref);
            const uint64_t shift2 = pack_f32x2(shift, shift);
            uint64_t ls[2] = {0, 0};
#pragma unroll 1
            for (int k0 = 0; k0 < BS; k0 += 32) {
              tmem_ld32(sb + k0, s);
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 vs = keys[(BS + k0 + k) >> 2];
                auto weights = [&](uint64_t t, float x, float y, uint64_t& sum) {
                  float p0, p1;
                  unpack_f32x2(fma_f32x2(add_f32x2(t, ref2), mul2, shift2), p0, p1);
                  const uint64_t p = pack_f32x2(fast_exp2(p0), fast_exp2(p1));
                  sum = add_f32x2(sum, p);
                  unpack_f32x2(mul_f32x2(p, pack_f32x2(x, y)), p0, p1);
                  return pack_f16(p0, p1);
                };
                const uint64_t t0 = two(k), t1 = two(k + 2);  // (the first is written over)
                s[k >> 1] = weights(t0, vs.x, vs.y, ls[0]);
                s[(k >> 1) + 1] = weights(t1, vs.z, vs.w, ls[1]);
              }
              // Over scores that have been read.
              tmem_st16(sb + (k0 >> 1), *reinterpret_cast<const uint32_t(*)[16]>(s));
            }
            float l0, l1;
            unpack_f32x2(add_f32x2(ls[0], ls[1]), l0, l1);
            l = fmaf(l0 + l1, fast_exp2(rho - f), l);
          } else {
            RowState st{m, l, rho, alpha, false};
            top = step_by_key(st, sb, kb0, seen, scale, keys);
            m = st.m;
            l = st.l;
            rho = st.rho;
            alpha = st.alpha;
            rescale = __any_sync(0xffffffffu, st.need);
          }
        } else {
          uint32_t s[BS];
          tmem_ld64(sb, s);
          if (masked) {
#pragma unroll
            for (int k = 0; k < BS; ++k)
              if (kb0 + k >= seen) s[k] = __float_as_uint(-INFINITY);
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < BS; k += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              mx[u] = max3_nan(mx[u], __uint_as_float(s[k + 2 * u]), __uint_as_float(s[k + 2 * u + 1]));
          const float smax = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          top = smax * scale;
          // (m + 8 would round, next to 2^27; beyond 2^26 a new maximum always moves m.)
          const bool need =
              top - m > kRescaleGap || (top >= m && fabsf(top) > 0x1p26f && top != -INFINITY);
          rescale = __any_sync(0xffffffffu, need);
          if (need) {
            alpha = m == -INFINITY ? 0.f : fast_exp2(m - top);
            l *= alpha;
            m = top;
            mraw = smax;
          }
          // Exponents from the difference to the maximum's score: the maximum's own
          // is 0 whatever its magnitude, where s * scale - m would be off by the last
          // place of m (32 for scores of 2^28).
          const uint64_t mul2 = pack_f32x2(scale, scale), ref2 = pack_f32x2(-mraw, -mraw);
          uint64_t ls[2] = {0, 0};
#pragma unroll
          for (int k = 0; k < BS; k += 2) {
            const uint64_t x = mul_f32x2(
                add_f32x2(pack_f32x2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), ref2), mul2);
            float p0, p1;
            unpack_f32x2(x, p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            ls[(k >> 1) & 1] = add_f32x2(ls[(k >> 1) & 1], pack_f32x2(p0, p1));
            s[k >> 1] = BF16 ? pack_bf16(p0, p1) : pack_f16(p0, p1);
          }
          tmem_st32(sb, *reinterpret_cast<const uint32_t(*)[32]>(s));
          float l0, l1;
          unpack_f32x2(add_f32x2(ls[0], ls[1]), l0, l1);
          l += l0 + l1;
        }
        // A score that is NaN or +inf makes the whole row NaN.
        if (!(top < INFINITY)) l = __int_as_float(0x7fffffff);
        if (rescale && i > 0) {
          // O holds the products up to the step before, which has to be done.
          ok = warp_wait(&pv_bar[c][(g - 1) & 1], ((g - 1) >> 1) & 1);
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; ok && d < DHP; d += 32) {
            uint32_t o[32];
            tmem_ld32(orow + d, o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st32(orow + d, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&p_bar[c][g & 1]));
      }
      tile0 += w.j1 - w.j0;
      if (ok && n > 0) ok = warp_wait(&pv_bar[c][(g - 1) & 1], ((g - 1) >> 1) & 1);
      // ---- output: O / l, or the piece's partial result
      const int slot = seq_slot(w);
      if (ok && rows > 0) {
        tc_fence_after();
        float mulo = slot >= 0 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        // Two factors: 2^rho may lie below the smallest fp32 number.
        const float half_rho = CODED ? fast_exp2(0.5f * rho) : 1.f;
        mulo *= half_rho;
        if constexpr (I4) mulo *= kI4Unit;
        const int* ps = reinterpret_cast<const int*>(mem + Cfg::OFF_X) + (piece % kPoison) * 3 * DHP;
        const bool hit = !CODED && *(volatile int*)&poison_set[piece % kPoison] != 0;
        const int64_t prow = (int64_t)slot * a.rows + c * half + r;
        if (slot >= 0 && mine)
          reinterpret_cast<float2*>(a.ws_ml)[prow] = make_float2(m, l);
        // Through shared memory, 64 bytes of each row at a time, so that four
        // lanes write one row's piece side by side.
        uint8_t* stage = CODED ? mem + c * Cfg::TILE + quarter * 4096
                               : mem + Cfg::OFF_OUT + (warp - 4) * 2048;
        const int64_t out = token * a.o.sT + (int64_t)head * a.o.sH;
        const int row0 = quarter * 32;  // of the chain
#pragma unroll 1
        for (int d = 0; d < DHP; d += 32) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld32(orow + d, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = __uint_as_float(o[i]);
            o[i] = __float_as_uint((CODED ? x * half_rho : x) * mulo);
          }
          if constexpr (I4) {  // in the order of the dimensions
            uint32_t t[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) t[i] = o[(i & ~7) + (i & 3) * 2 + ((i >> 2) & 1)];
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = t[i];
          }
          if (hit) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint(poisoned(__uint_as_float(o[i]), ps, ps + DHP, ps + 2 * DHP,
                                              d + i, seen));
          }
          const int unit = lane & 3;
          if (slot >= 0) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {  // 16 values are 64 bytes
              __syncwarp();
#pragma unroll
              for (int u = 0; u < 4; ++u)
                *reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(o[hf * 16 + u * 4], o[hf * 16 + u * 4 + 1], o[hf * 16 + u * 4 + 2],
                               o[hf * 16 + u * 4 + 3]);
              __syncwarp();
              const int dd = d + hf * 16 + unit * 4;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int rr = k * 8 + (lane >> 2);
                const uint4 x = *reinterpret_cast<const uint4*>(
                    stage + rr * 64 + ((unit ^ ((rr >> 1) & 3)) << 4));
                if (row0 + rr < rows && dd < a.q.Dh)  // Dh is a multiple of 8
                  *reinterpret_cast<uint4*>(
                      a.ws_o + ((int64_t)slot * a.rows + c * half + row0 + rr) * a.q.Dh + dd) = x;
              }
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint4 x;
              EQ* e = reinterpret_cast<EQ*>(&x);
#pragma unroll
              for (int b = 0; b < 8; ++b) from_float(__uint_as_float(o[u * 8 + b]), e[b]);
              *reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) = x;
            }
            __syncwarp();
            const int dd = d + unit * 8;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int rr = k * 8 + (lane >> 2);
              const uint4 x = *reinterpret_cast<const uint4*>(
                  stage + rr * 64 + ((unit ^ ((rr >> 1) & 3)) << 4));
              EQ* to = static_cast<EQ*>(a.o.data) + __shfl_sync(0xffffffffu, out, rr) + dd;
              if (row0 + rr >= rows || dd >= a.q.Dh) continue;
              if (ovec) {
                *reinterpret_cast<uint4*>(to) = x;
              } else {
                const EQ* e = reinterpret_cast<const EQ*>(&x);
#pragma unroll
                for (int b = 0; b < 8; ++b) to[b] = e[b];
              }
            }
          }
        }
        tc_fence_before();
      }
      if constexpr (!CODED) {
        __syncwarp();
        if (lane == 0) atomicAdd(&outputs[c], 1);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int TQ, int TK, int DHP>
void launch(const SeqAttnArgs& a, int ctas, const CUtensorMap& q, const CUtensorMap& k,
            const CUtensorMap& v, bool qtma, bool qvec, bool ovec, cudaStream_t s) {
  using Cfg = TcCfg<elem_coded(TK), DHP>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  ATTNB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    ATTNB_CUDA(cudaFuncSetAttribute(seq_tc_kernel<TQ, TK, DHP>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    configured.fetch_or(bit);
  }
  ATTNB_CUDA(launch_pdl(seq_tc_kernel<TQ, TK, DHP>, dim3(ctas), dim3(Cfg::THREADS), Cfg::SMEM, s, q,
                        k, v, a, qtma, qvec, ovec));
}

bool aligned16(const RowsView& r) {
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.sT % 8 == 0 && r.sH % 8 == 0;
}

// Packed rows [tokens, heads, Dh] as (Dh, heads, tokens), copied `heads` by
// `tokens` rows at a time.
bool map_allowed(const RowsView& r) {
  return r.tokens > 0 && aligned16(r) && (r.tokens == 1 || r.sT > 0) &&
         (r.heads == 1 || r.sH > 0) && r.sT < (1ll << 38) && r.sH < (1ll << 38);
}
CUtensorMap rows_map(const RowsView& r, int heads, int tokens) {
  const uint64_t dims[3] = {(uint64_t)r.Dh, (uint64_t)r.heads, (uint64_t)r.tokens};
  const uint64_t any = ((uint64_t)r.Dh * 2 + 15) / 16 * 16;  // of a dimension of one
  const uint64_t strides[2] = {r.heads > 1 ? (uint64_t)r.sH * 2 : any,
                               r.tokens > 1 ? (uint64_t)r.sT * 2 : any * r.heads};
  const uint32_t box[3] = {64, (uint32_t)heads, (uint32_t)tokens};
  return make_tmap_nd(r.data, 2, 3, dims, strides, box);
}

}  // namespace

bool seq_tc_supported(const SeqAttnArgs& a) {
  if (a.q.type == kF32 || a.G > BM || a.q.Dh > 128 || a.q.Dh % 8 != 0) return false;
  if (a.pages.k) return seq_pages_tma(a);
  return map_allowed(a.k) && map_allowed(a.v);
}

int seq_tc_rows(int G) { return 2 * (BM / G) * G; }

void seq_tc_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  const bool paged = a.pages.k != nullptr, coded = paged && elem_coded(a.pages.type);
  const int box = coded ? 64 : BN;
  const CUtensorMap k = paged ? seq_pages_map(a.pages, a.pages.k, box) : rows_map(a.k, 1, BN);
  const CUtensorMap v = paged ? seq_pages_map(a.pages, a.pages.v, box) : rows_map(a.v, 1, BN);
  // Over codes Q is scaled on its way in, by threads.
  const bool qtma = !coded && map_allowed(a.q);
  const CUtensorMap q = qtma ? rows_map(a.q, a.G, BM / a.G) : k;
  const bool qvec = aligned16(a.q), ovec = aligned16(a.o);
  auto go = [&](auto tq, auto tk) {
    constexpr int TQ = decltype(tq)::value, TK = decltype(tk)::value;
    if constexpr (TQ != kF32) {
      if (a.q.Dh <= 64) launch<TQ, TK, 64>(a, ctas, q, k, v, qtma, qvec, ovec, s);
      else launch<TQ, TK, 128>(a, ctas, q, k, v, qtma, qvec, ovec, s);
    }
  };
  with_value_type(a.q.type, [&](auto tq) {
    if (a.pages.k && a.pages.type == kE4M3) go(tq, std::integral_constant<int, kE4M3>{});
    else if (a.pages.k && a.pages.type == kI8) go(tq, std::integral_constant<int, kI8>{});
    else if (a.pages.k && a.pages.type == kI4) go(tq, std::integral_constant<int, kI4>{});
    else go(tq, tq);
  });
}

}  // namespace attnb
