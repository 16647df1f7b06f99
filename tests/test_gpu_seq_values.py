"""Values at the edges of their range in attention over ragged sequences: NaN as the GPU computes it,
vectors that are not finite behind a causal mask, and scales of coded pages that are tiny, huge, zero
or far apart.  One sequence and one pool throughout; the kernel follows from the type and from the
number of new tokens."""
from __future__ import annotations

import pytest
import torch

import seq_ref
from attn_cpu import capi
from test_gpu_seq_ops import BF16, E4M3, F16, F32, I8, Pool, _gen, _randn

pytestmark = pytest.mark.gpu

HALF_F16 = seq_ref.HALF[F16]


def _reference(q, k, v, causal=True, scale=None):
    """q [n, heads, D] over k, v [L, H, D] in 64 bits: outputs, sum_j p_j |v_j|, the largest
    p_j max|v_j| of each row, the largest |scale q.k| that the norms allow, and the largest
    scale * sqrt(sum_d (q_d k_d)^2)."""
    n, heads, D = q.shape
    L, H = k.shape[:2]
    q, k, v = (x.double().cpu() for x in (q, k, v))
    qq = q.permute(1, 0, 2)
    kk = k.permute(1, 2, 0).repeat_interleave(heads // H, 0)
    vv = v.permute(1, 0, 2).repeat_interleave(heads // H, 0)
    f = D ** -0.5 if scale is None else scale
    seen = torch.ones(n, L, dtype=torch.bool)
    if causal:
        seen = seen.tril(L - n)
    p = torch.softmax(torch.where(seen, (qq @ kk) * f, -torch.inf), -1)
    out, mag = (p @ vv).permute(1, 0, 2), (p @ vv.abs()).permute(1, 0, 2)
    most = (p * vv.abs().amax(-1)[:, None, :]).amax(-1).permute(1, 0)[..., None]
    smax = float(q.norm(dim=-1).max() * k.norm(dim=-1).max()) * f
    s2 = float(((qq ** 2) @ (kk ** 2)).max()) ** 0.5 * f
    return out, mag, most, smax, s2


def _bound(rows, coded, ref, L, exact_k=False):
    """|error| per element.  fp32 arithmetic as in seq_ref.attention_bound, and the output's rounding.

    16-bit rows over codes: weights in f16, half a step of 2^-11; K and V as code * factor in f16,
    two roundings of half a step each.  Those of V are 2 * 2^-11 of sum p |v|.  Those of K are off by
    at most 2^-11 each, so by 0.82 * 2^-11 in the root mean square of both, which add up over the
    dimensions to 0.82 * 2^-11 * s2 in a score; three times that for the largest of many, and twice
    since the sum of the weights is off as well: 5 * 2^-11 * s2 of sum p |v| (nothing where the
    factors are powers of two).  Weights below 2^-14 of the row's largest p_j v_j have f16's steps
    of 2^-24 and are off by 2^-25 of it each; where keys share one power of two, their scales may
    differ by 2^6 and the reference is up to 2^7 above the largest p_j v_j."""
    out, mag, most, smax, s2 = ref
    rel = seq_ref.HALF[F32] * (40 * smax + 4 * out.shape[-1] ** 0.5 + 2 * L ** 0.5 + 16)
    floor = 0.0
    if coded and rows != F32:
        rel += HALF_F16 * (3 + (0 if exact_k else 5 * s2))
        floor = 2.0 ** -25 * 2.0 ** 7 * L * most
    elif rows != F32:
        rel += seq_ref.HALF[rows]
    return mag * rel + out.abs() * 1.01 * seq_ref.HALF[rows] + floor


def _check(o, ref, bound):
    o = o.double().cpu()
    bad = ~((o - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((o - ref).abs() / bound).nan_to_num(1e9).max()))


def _attend(p, q, causal=True):
    o = torch.full_like(q, 7.0)
    capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts([len(q)]), p.table, p.lens, len(q), causal,
                        None, p.ks, p.vs)
    return o


def _pool(L, H, D, rows, cache, seed, k=None, v=None, page=64):
    """A sequence of L tokens in pages, written from k and v (functions of the drawn values)."""
    p = Pool([L], H, D, page, rows, cache, seed)
    p.x = [x if f is None else f(x).to(rows).contiguous() for x, f in zip(p.x, (k, v))]
    p.append()
    return p


def _nan(bits):
    x = torch.tensor([bits], dtype=torch.int32, device="cuda").view(F32)
    assert torch.isnan(x).all()
    return x


# What CUDA's arithmetic returns, what torch writes, and one with the lowest bit of the payload.
NANS = [0x7fffffff, 0x7fc00000, 0x7f800001, -1]


@pytest.mark.parametrize("bits", NANS)
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("n", [3, 300])
def test_nan_in_fp32(cuda, bits, paged, n):
    """A NaN in a query is that row's, one in a key every row's that sees it, one in a value those
    rows' in its dimension."""
    D, L = 64, 300
    g = _gen(40)
    q, k, v = _randn(g, n, 4, D), _randn(g, L, 2, D), _randn(g, L, 2, D)
    ref = _reference(q, k, v)
    bound = _bound(F32, False, ref, L)
    row, key, value = n - 2, L - 1, L - n + n // 3
    q[row, 1, 5] = _nan(bits)
    k[key, 1, 7] = _nan(bits)
    v[value, 0, 9] = _nan(bits)
    want = torch.zeros(n, 4, D, dtype=torch.bool)
    want[row, 1] = True
    want[key - L + n:, 2:] = True
    want[value - L + n:, :2, 9] = True
    if paged:
        p = _pool(L, 2, D, F32, F32, 41, lambda x: k, lambda x: v)
        o = _attend(p, q)
    else:
        o = torch.full_like(q, 7.0)
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        capi.attn_packed_dev(q, k, v, o, cu, seq_ref.starts([L]), causal=True)
    assert torch.equal(torch.isnan(o).cpu(), want)
    _check(torch.where(want, 0.0, o.cpu()), torch.where(want, 0.0, ref[0]), bound)


@pytest.mark.parametrize("n", [3, 300])
def test_largest_fp32_values(cuda, n):
    """The largest and the lowest fp32 number among the values stay finite numbers."""
    D, L = 64, 300
    g = _gen(42)
    q, k, v = _randn(g, n, 4, D), _randn(g, L, 2, D), _randn(g, L, 2, D)
    v[0, :, 3] = torch.finfo(F32).max
    v[0, :, 4] = torch.finfo(F32).min
    ref = _reference(q, k, v)
    o = torch.empty_like(q)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    capi.attn_packed_dev(q, k, v, o, cu, seq_ref.starts([L]), causal=True)
    _check(o, ref[0], _bound(F32, False, ref, L))


@pytest.mark.parametrize("rows,cache", [(F32, E4M3), (F32, I8)])
@pytest.mark.parametrize("n", [3, 300])
@pytest.mark.parametrize("bad", ["k", "v"])
def test_vectors_that_are_not_finite_in_pages(cuda, rows, cache, n, bad):
    """A vector with a NaN or an infinity makes the rows that see it NaN, and no others."""
    D, L = 64, 400
    late, later = L - n + n // 2, L - 1
    q = _randn(_gen(43), n, 4, D, dtype=rows)
    p = _pool(L, 2, D, rows, cache, 44)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    x = p.x["kv".index(bad)]
    x[late, 0, 11] = float("inf")
    x[later, 1, 0] = float("nan")
    p.append()
    o = _attend(p, q)
    want = torch.zeros(n, 4, D, dtype=torch.bool)
    want[late - L + n:, :2] = True
    want[later - L + n:, 2:] = True
    assert torch.equal(torch.isnan(o).cpu(), want)
    o = torch.where(want, 0.0, o.double().cpu())
    _check(o, torch.where(want, 0.0, ref[0]), _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", [(BF16, E4M3), (BF16, I8), (F32, E4M3), (F32, I8)])
@pytest.mark.parametrize("n", [1, 12])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 1e-20, 1e-5, 1e25, 2.0 ** 80])
def test_values_of_any_size(cuda, rows, cache, n, size):
    D, L = 64, 400
    q = _randn(_gen(48), n, 4, D, dtype=rows)
    p = _pool(L, 2, D, rows, cache, 49, v=lambda x: x.float() * size)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))
