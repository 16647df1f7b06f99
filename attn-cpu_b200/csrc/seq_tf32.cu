// seq_tf32.cu -- K9: attention of many query rows in fp32, over packed keys or
// pages of any type (and of 16-bit rows that TMA cannot read), on tensor cores.
//
// Every product is three tf32 products of split operands, big.big + big.small +
// small.big, as in the 3xTF32 kernels of this library: an fp32 value is the sum
// of two tf32 values but for 2^-22 of it.  The instruction cuts its fp32 sums off
// instead of rounding them, so long sums through it come out short: scores of 64
// dimensions and outputs of 450 keys were off by 2.2e-6.  So the cross terms of a
// score have a sum of their own, its large terms go in sums of 32 dimensions, and a
// tile's P V starts at 0 and meets O in a rounded fma: 4.0e-7 (fp32 products and sums
// of torch: 5.4e-7), in the same time.
// Bound by the warp-wide tensor instruction (mma.sync m16n8k8) and the plain loads
// that feed it.  tcgen05, over tiles that are split in shared memory as K3's are,
// has more room; that form is not built for ragged sequences.
//
// A CTA of eight warps takes 128 rows of one KV head, 16 a warp, and walks 32
// keys at a time.  K and V are read by all threads while the tile before is
// being multiplied, split once and kept in shared memory as (big, small) pairs,
// so that a fragment element is one 8-byte read; row lengths are padded so that
// these reads touch every bank once.  The weights go from the accumulator layout
// into the A operand without a shuffle: the sum over keys may run in any order,
// so column 2c of the scores serves as column c of A, 2c + 1 as c + 4, and V's
// rows are picked accordingly.
//
// Measured: three sequences of 101-901 fp32 tokens, 16/4 heads of 64, 127 us where
// K6 takes 440.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "runtime.h"
#include "seq.cuh"
#include "seq_elem.cuh"

namespace attnb {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;
constexpr int kKeys = 32;

template <int DH>  // head size padded to 64 or 128
struct Tf32Cfg {
  static constexpr int QROW = DH + 4;   // floats
  static constexpr int KROW = DH + 4;   // pairs; 4 modulo 16
  static constexpr int VROW = DH + 2;   // pairs; 2 modulo 8
  static constexpr int OFF_K = kRows * QROW * 4;
  static constexpr int OFF_V = OFF_K + kKeys * KROW * 8;
  static constexpr int SMEM = OFF_V + kKeys * VROW * 8;
  static constexpr int EACH = kKeys * DH / kThreads;  // elements of K per thread
};

__device__ __forceinline__ float2 split_tf32(float x) {
  const float big = tf32_round(x);
  return make_float2(big, tf32_round(x - big));
}
// The same where x may be next to the largest fp32 number.  That rounds to
// infinity; there both parts are cut off, so that their sum stays below it.
__device__ __forceinline__ float2 split_tf32_any(float x) {
  const float2 s = split_tf32(x);
  if (fabsf(s.x) != INFINITY) return s;
  const float big = __uint_as_float(__float_as_uint(x) & 0xFFFFE000u);
  return make_float2(big, __uint_as_float(__float_as_uint(x - big) & 0xFFFFE000u));
}

// tf32_round adds to the bits, which takes a NaN with a full payload (what CUDA's
// arithmetic returns) to -0 and one with a small payload to infinity.  Operands
// therefore hold a NaN as this one, which is rounded to itself; its small part
// becomes -0.
__device__ __forceinline__ float plain_nan(float x) {
  return x != x ? __int_as_float(0x7fc00000) : x;
}

__device__ __forceinline__ void mma_tf32_sync(float (&d)[4], const float (&a)[4], float b0,
                                              float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
        "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

template <int TQ, int TK, int DH>
__global__ void __launch_bounds__(kThreads, 1)
    seq_tf32_kernel(const __grid_constant__ SeqAttnArgs a, const bool kvec) {
  using Cfg = Tf32Cfg<DH>;
  using EQ = elem_t<TQ>;
  using EK = elem_t<TK>;
  constexpr bool CODED = TK == kE4M3 || TK == kI8;
  constexpr int QUADS = Cfg::EACH / 4;  // 4-element reads of K (and of V) per thread
  extern __shared__ uint8_t mem[];
  __shared__ SeqShared sh;
  float* const qs = reinterpret_cast<float*>(mem);
  float2* const kp = reinterpret_cast<float2*>(mem + Cfg::OFF_K);
  float2* const vp = reinterpret_cast<float2*>(mem + Cfg::OFF_V);

  grid_dep_wait();
  SeqPlace place;
  const bool any = seq_locate(a, sh, place);
  if (threadIdx.x == 0) seq_write_split(a, any, place);
  if (!any) return;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int Dh = a.q.Dh;
  const bool paged = a.pages.k != nullptr;
  SeqIter it;
  it.start(place);
  SeqPiece w;
  for (bool first = true; it.next(a, w); first = false) {
    // ---- Q, with the scale
    for (int i = tid; i < kRows * DH; i += kThreads) {
      const int r = i / DH, d = i % DH;
      float x = 0.f;
      if (r < w.rows && d < Dh) {
        const int row = w.row0 + r;
        x = to_float(static_cast<const EQ*>(a.q.data)[(int64_t)(w.s.q0 + row / a.G) * a.q.sT +
                                                      (int64_t)(w.h * a.G + row % a.G) * a.q.sH + d]) *
            a.scale_log2;
      }
      qs[r * Cfg::QROW + d] = plain_nan(x);
    }
    // K and V of a tile as they come, times their scales.
    float kr[QUADS][4], vr[QUADS][4];
    auto fetch = [&](int j) {
#pragma unroll
      for (int u = 0; u < QUADS; ++u) {
        const int i = tid + u * kThreads, key = j * kKeys + i / (DH / 4), d = i % (DH / 4) * 4;
        const EK *kx = nullptr, *vx = nullptr;
        float ks = 1.f, vs = 1.f;
        if (key < w.s.L) {
          if (paged) {
            const int page = seq_page(a.seqs, a.pages, w.b, key, a.index_status);
            if (page >= 0) {  // a bad page reads as zeros
              const int64_t at = (((int64_t)page * a.pages.H + w.h) << a.pages.page_shift) +
                                 (key & ((1 << a.pages.page_shift) - 1));
              kx = static_cast<const EK*>(a.pages.k) + at * Dh;
              vx = static_cast<const EK*>(a.pages.v) + at * Dh;
              if (CODED) {
                ks = __ldg(a.pages.k_scale + at);
                vs = __ldg(a.pages.v_scale + at);
              }
            }
          } else {
            const int64_t t = w.s.k0 + key;
            kx = static_cast<const EK*>(a.k.data) + t * a.k.sT + (int64_t)w.h * a.k.sH;
            vx = static_cast<const EK*>(a.v.data) + t * a.v.sT + (int64_t)w.h * a.v.sH;
          }
        }
        float k4[4] = {0.f, 0.f, 0.f, 0.f}, v4[4] = {0.f, 0.f, 0.f, 0.f};
        if (kx) {
          if (kvec) {
            if (d < Dh) {  // Dh is a multiple of 4
              load4(kx + d, k4);
              load4(vx + d, v4);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < Dh) {
                k4[e] = to_float(kx[d + e]);
                v4[e] = to_float(vx[d + e]);
              }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[u][e] = CODED ? k4[e] * ks : k4[e];
          vr[u][e] = CODED ? v4[e] * vs : v4[e];
        }
      }
    };
    const int seen_min = seq_row_seen(a, w.s, w.row0);
    int seen[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = warp * 16 + g + 8 * i;
      seen[i] = r < w.rows ? seq_row_seen(a, w.s, w.row0 + r) : 0;
    }
    float acc[DH / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < DH / 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    const bool rows_here = warp * 16 < w.rows;

    fetch(w.j0);
    for (int j = w.j0; j < w.j1; ++j) {
      __syncthreads();  // the tile before has been read
      const bool masked = (j + 1) * kKeys > seen_min;
      bool finite = true;
#pragma unroll
      for (int u = 0; u < QUADS; ++u) {
        const int i = tid + u * kThreads, r = i / (DH / 4), d = i % (DH / 4) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          finite = finite && fabsf(vr[u][e]) <= 3.402823466e38f;
          kp[r * Cfg::KROW + d + e] = split_tf32_any(plain_nan(kr[u][e]));
          vp[r * Cfg::VROW + d + e] = split_tf32_any(plain_nan(vr[u][e]));
        }
      }
      // A V that is not finite cannot be split, and must not reach the rows that
      // do not see it: the keys of such a tile are then added one by one.
      const bool plain = __syncthreads_and(finite);
      if (j + 1 < w.j1) fetch(j + 1);
      if (!rows_here) continue;
      // ---- scores: four column tiles of 8 keys
      float s[4][4], cross[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = cross[t][e] = 0.f;
      const float* qr = qs + (warp * 16 + g) * Cfg::QROW + c;
#pragma unroll
      for (int k0 = 0; k0 < DH / 8; k0 += 4) {
        float part[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[t][e] = 0.f;
#pragma unroll
        for (int k = k0; k < k0 + 4; ++k) {
          float big[4], small[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = split_tf32(qr[(e & 1) * 8 * Cfg::QROW + k * 8 + (e >> 1) * 4]);
            big[e] = x.x;
            small[e] = x.y;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const float2 b0 = kp[(t * 8 + g) * Cfg::KROW + k * 8 + c];
            const float2 b1 = kp[(t * 8 + g) * Cfg::KROW + k * 8 + c + 4];
            mma_tf32_sync(cross[t], small, b0.x, b1.x);
            mma_tf32_sync(cross[t], big, b0.y, b1.y);
            mma_tf32_sync(part[t], big, b0.x, b1.x);
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] += part[t][e];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] += cross[t][e];
      // ---- weights
      if (masked) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j * kKeys + t * 8 + 2 * c + (e & 1) >= seen[e >> 1]) s[t][e] = -INFINITY;
      }
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = m[i];
#pragma unroll
        for (int t = 0; t < 4; ++t) top = fmaxf(top, fmaxf(s[t][2 * i], s[t][2 * i + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float use = top == -INFINITY ? 0.f : top;
        alpha[i] = fast_exp2(m[i] - use);
        m[i] = top;
        l[i] *= alpha[i];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[t][2 * i + e] = fast_exp2(s[t][2 * i + e] - use);
            l[i] += s[t][2 * i + e];
          }
      }
      if (!plain) {
#pragma unroll
        for (int t = 0; t < DH / 8; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] *= alpha[e >> 1];
        // Every key's row by itself: p of key k lies with lane (g, k / 2 % 4).
        for (int k = 0; k < kKeys; ++k) {
          const int src = (lane & ~3) | ((k >> 1) & 3);
          float p[2] = {0.f, 0.f};
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float x = __shfl_sync(0xffffffffu, s[t][2 * i + e], src);
                if (t == k >> 3 && e == (k & 1)) p[i] = x;
              }
          const int key = j * kKeys + k;
#pragma unroll
          for (int t = 0; t < DH / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = vp[k * Cfg::VROW + t * 8 + 2 * c + (e & 1)];
              // The small part of an infinity is a NaN, of no use here.
              const float x = fabsf(v.x) <= 3.402823466e38f ? v.x + v.y : v.x;
              if (key < seen[e >> 1]) acc[t][e] = fmaf(p[e >> 1], x, acc[t][e]);
            }
        }
        continue;
      }
      // ---- O = alpha O + P V
      float big[4][4], small[4][4];
#pragma unroll
      for (int t8 = 0; t8 < 4; ++t8)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // A's column c is key 2c, its column c + 4 key 2c + 1.
          const float2 x = split_tf32(s[t8][(e & 1) * 2 + (e >> 1)]);
          big[t8][e] = x.x;
          small[t8][e] = x.y;
        }
#pragma unroll
      for (int t = 0; t < DH / 8; ++t) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t8 = 0; t8 < 4; ++t8) {
          const float2 b0 = vp[(t8 * 8 + 2 * c) * Cfg::VROW + t * 8 + g];
          const float2 b1 = vp[(t8 * 8 + 2 * c + 1) * Cfg::VROW + t * 8 + g];
          mma_tf32_sync(part, small[t8], b0.x, b1.x);
          mma_tf32_sync(part, big[t8], b0.y, b1.y);
          mma_tf32_sync(part, big[t8], b0.x, b1.x);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(acc[t][e], alpha[e >> 1], part[e]);
      }
    }
    // ---- output
    const int slot = seq_slot(w, first);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int r = warp * 16 + g + 8 * i;
      if (r >= w.rows) continue;
      const int row = w.row0 + r;
      const int64_t prow = (int64_t)slot * kRows + r;
      if (slot >= 0 && c == 0) reinterpret_cast<float2*>(a.ws_ml)[prow] = make_float2(m[i], sum);
      EQ* o = static_cast<EQ*>(a.o.data) + (int64_t)(w.s.q0 + row / a.G) * a.o.sT +
              (int64_t)(w.h * a.G + row % a.G) * a.o.sH;
#pragma unroll
      for (int t = 0; t < DH / 8; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = t * 8 + 2 * c + e;
          if (d >= Dh) continue;
          const float x = acc[t][2 * i + e];
          if (slot >= 0) a.ws_o[prow * Dh + d] = x;
          else from_float(sum == 0.f ? 0.f : x / sum, o[d]);  // no key: 0
        }
    }
    __syncthreads();  // Q is replaced next
  }
}

bool quads(const void* p, int64_t sT, int64_t sH, int Dh, int type) {
  return reinterpret_cast<uintptr_t>(p) % (4 * elem_bytes(type)) == 0 && sT % 4 == 0 &&
         sH % 4 == 0 && Dh % 4 == 0;
}

template <int TQ, int TK, int DH>
void launch(const SeqAttnArgs& a, int ctas, bool kvec, cudaStream_t s) {
  using Cfg = Tf32Cfg<DH>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  ATTNB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    ATTNB_CUDA(cudaFuncSetAttribute(seq_tf32_kernel<TQ, TK, DH>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    configured.fetch_or(bit);
  }
  ATTNB_CUDA(launch_pdl(seq_tf32_kernel<TQ, TK, DH>, dim3(ctas), dim3(kThreads), Cfg::SMEM, s, a,
                        kvec));
}

}  // namespace

void seq_tf32_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  const bool paged = a.pages.k != nullptr;
  const int tk = paged ? a.pages.type : a.k.type;
  const bool kvec = paged ? quads(a.pages.k, 0, 0, a.q.Dh, tk) && quads(a.pages.v, 0, 0, a.q.Dh, tk)
                          : quads(a.k.data, a.k.sT, a.k.sH, a.q.Dh, tk) &&
                                quads(a.v.data, a.v.sT, a.v.sH, a.q.Dh, tk);
  auto go = [&](auto tq, auto tkc) {
    constexpr int TQ = decltype(tq)::value, TK = decltype(tkc)::value;
    if (a.q.Dh <= 64) launch<TQ, TK, 64>(a, ctas, kvec, s);
    else launch<TQ, TK, 128>(a, ctas, kvec, s);
  };
  with_value_type(a.q.type, [&](auto tq) {
    if (tk == kE4M3) go(tq, std::integral_constant<int, kE4M3>{});
    else if (tk == kI8) go(tq, std::integral_constant<int, kI8>{});
    else go(tq, tq);
  });
}

}  // namespace attnb
