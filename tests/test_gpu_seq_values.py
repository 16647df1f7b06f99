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
    differ by 2^6 and the reference is up to 2^7 above the largest p_j v_j.  Outputs in f16 have
    steps of 2^-24 below 2^-14 as well: their rounding is off by up to 2^-25."""
    out, mag, most, smax, s2 = ref
    rel = seq_ref.HALF[F32] * (40 * smax + 4 * out.shape[-1] ** 0.5 + 2 * L ** 0.5 + 16)
    floor = 0.0
    if coded and rows != F32:
        rel += HALF_F16 * (3 + (0 if exact_k else 5 * s2))
        floor = 2.0 ** -25 * 2.0 ** 7 * L * most
    elif rows != F32:
        rel += seq_ref.HALF[rows]
    return mag * rel + out.abs() * 1.01 * seq_ref.HALF[rows] + floor + (2.0 ** -25 if rows == F16 else 0.0)


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


CODED = [(BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, I8), (F16, I8), (F32, I8)]


@pytest.mark.parametrize("rows,cache", CODED)
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


@pytest.mark.parametrize("rows,cache", CODED)
@pytest.mark.parametrize("n", [3, 300])
@pytest.mark.parametrize("big", ["k", "v"])
def test_huge_vectors_behind_the_mask(cuda, rows, cache, n, big):
    """A large finite vector at the end changes nothing for the rows that do not see it."""
    D, L = 64, 400
    q = _randn(_gen(45), n, 4, D, dtype=rows)
    p = _pool(L, 2, D, rows, cache, 46)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    p.x["kv".index(big)][L - 1] = _randn(_gen(47), 2, D) * (3e4 if rows == F16 else 1e30)
    p.x["kv".index(big)][L - 1].clamp_(*((-6e4, 6e4) if rows == F16 else (-1e31, 1e31)))
    p.append()
    o = _attend(p, q)[:n - 1]
    ref = tuple(x[:n - 1] if torch.is_tensor(x) else x for x in ref)
    _check(o, ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", [(BF16, E4M3), (BF16, I8), (F32, E4M3), (F32, I8)])
@pytest.mark.parametrize("n", [1, 12, 60, 300])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 1e-20, 1e-5, 1e25, 2.0 ** 80])
def test_values_of_any_size(cuda, rows, cache, n, size):
    D, L = 64, 400
    q = _randn(_gen(48), n, 4, D, dtype=rows)
    p = _pool(L, 2, D, rows, cache, 49, v=lambda x: x.float() * size)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


def _blocks(L, sizes):
    """A factor for each token: 64 of one size, then 64 of the next."""
    s = torch.tensor(sizes, device="cuda").repeat(-(-L // (64 * len(sizes))))
    return s.repeat_interleave(64)[:L, None, None]


@pytest.mark.parametrize("rows,cache", CODED)
@pytest.mark.parametrize("n", [1, 60, 300])
@pytest.mark.parametrize("sizes", [(0.0, 1e-4), (1e-4, 0.0, 1.0), (0.0, 2e-5), (2e-5, 1.0, 300.0)])
def test_value_sizes_that_change_between_blocks(cuda, rows, cache, n, sizes):
    """Whole blocks of zeros or of other sizes beside small values.  Each block's share of an output
    is held to its own size: where one block's values are large they set the bound's floor."""
    D, L = 64, 400
    q = _randn(_gen(50), n, 4, D, dtype=rows)
    p = _pool(L, 2, D, rows, cache, 51, v=lambda x: x.float() * _blocks(L, sizes))
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", [(BF16, E4M3), (BF16, I8), (F32, I8)])
@pytest.mark.parametrize("n", [1, 60, 300])
def test_value_sizes_that_no_f16_holds_together(cuda, rows, cache, n):
    """Rows whose weight lies on small values alone: the keys of the large ones score low."""
    D, L = 64, 400
    q = _randn(_gen(52), n, 4, D, dtype=rows)
    q[..., 0] = 8.0

    def keys(x):
        x = x.clone()
        x[..., 0] = 4.0
        x[::3, :, 0] = -60.0  # with q_0 = 8 a score of -64 less than the others: 2^-92
        return x

    def values(x):
        x = x.float() * 1e-6
        x[::3] *= 1e20
        return x

    p = _pool(L, 2, D, rows, cache, 53, keys, values)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    assert float(ref[1].max()) < 1e-4
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", CODED)
@pytest.mark.parametrize("n", [3, 300])
def test_key_sizes_that_differ_in_a_block(cuda, rows, cache, n):
    """Some keys 2^15 times the others, all with very low scores: the others' scores keep their
    bits."""
    D, L = 64, 400
    q = _randn(_gen(54), n, 4, D, dtype=rows)
    q[..., 0] = 1.0

    def keys(x):
        x = x.clone()
        x[::5] = 0
        x[::5, :, 0] = -30000.0  # a score of -3750
        return x

    p = _pool(L, 2, D, rows, cache, 55, keys)
    k, v = p.held(0)[0], p.held(1)[0]
    out, mag, most, _, _ = _reference(q, k, v)
    rest = torch.arange(L) % 5 != 0  # the weights of the large keys are 0 in 64 bits too
    _, _, _, smax, s2 = _reference(q, k[rest], v[rest], causal=False)
    ref = out, mag, most, smax, s2
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", [(BF16, E4M3), (BF16, I8), (F32, E4M3)])
@pytest.mark.parametrize("n", [3, 300])
@pytest.mark.parametrize("qsize,ksize", [(1e-18, 1e-18), (2.0 ** -100, 2.0 ** -40), (2.0 ** -126, 2.0 ** -100),
                                         (2.0 ** 100, 2.0 ** -100)])
def test_tiny_queries_and_keys(cuda, rows, cache, n, qsize, ksize):
    """Scores next to 0 over values whose size changes from block to block."""
    D, L = 64, 400
    q = (_randn(_gen(56), n, 4, D) * qsize).to(rows)
    p = _pool(L, 2, D, rows, cache, 57, lambda x: x.float() * ksize,
              lambda x: x.float() * _blocks(L, (1.0, 2.0 ** -12)))
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("rows,cache", CODED)
@pytest.mark.parametrize("n,L", [(1, 3), (3, 3), (1, 65), (3, 65), (30, 65), (1, 300), (3, 300),
                                 (30, 300), (300, 300)])
def test_weights_over_codes_have_the_bits_of_f16(cuda, rows, cache, n, L):
    """Key scales that are powers of two, so that what is left is the rounding of weights and
    values: bf16 weights, 2^-8, would not pass for rows in f16."""
    D = 64
    q = _randn(_gen(58), n, 4, D, dtype=rows)

    def keys(x):
        x = x.float().clamp(-1.7, 1.7)
        x[..., 0] = seq_ref.TOP[cache] * 2.0 ** -8 * (4 if cache == I8 else 1)
        return x

    p = _pool(L, 2, D, rows, cache, 59, keys)
    assert torch.equal(torch.frexp(p.ks[p.table[0, :1].long(), :, 0])[0].cpu(), torch.full((1, 2), 0.5))
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L, exact_k=True))


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("n", [1, 60])
def test_one_key_takes_all(cuda, cache, n):
    """Scores of 2^28: the output is the value of the key with the largest score."""
    D, L = 64, 200
    q = (_randn(_gen(60), n, 4, D).sign() * 1.5 * 2.0 ** 127).to(BF16)
    p = _pool(L, 1, D, BF16, cache, 61, lambda x: x.float() * 2.0 ** -100)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    k = p.held(0)[0][:, 0]
    s = torch.einsum("nhd,ld->nhl", q.double().cpu(), k) * D ** -0.5
    s = torch.where(torch.arange(L) <= (L - n + torch.arange(n))[:, None, None], s, -torch.inf)
    two = s.topk(2, -1).values
    # Rows whose two best scores are nearer than the roundings of K (5 * 2^-11 * s2, as in _bound) and
    # of fp32 sums allow are left out; there are few.
    clear = two[..., 0] - two[..., 1] > 5 * HALF_F16 * ref[4] + 2.0 ** -19 * ref[3]
    assert clear.float().mean() > 0.8
    out = ref[0] * clear[..., None]
    o = _attend(p, q).double().cpu() * clear[..., None]
    # V as code * factor in f16 (two roundings) and the output in bf16.
    _check(o, out, out.abs() * (2 * HALF_F16 + 1.01 * seq_ref.HALF[BF16]) + 2.0 ** -24 * ref[1].max())


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_chunks_over_codes(cuda, cache, D):
    """Chunks of one and a few steps, with fewer keys than rows or more, whose tiles have scales of
    their own: each tile's belong to it for as long as both row tiles of an item need them."""
    keys = [(b * 37) % 260 + 1 for b in range(70)]
    new = [(b * 53) % 200 + 40 for b in range(70)]
    new = [min(n, 2 * k + 30) for n, k in zip(new, keys)]
    p = Pool(keys, 2, D, 32, BF16, cache, 63)
    size = torch.tensor([2.0 ** ((b * 7) % 11 - 5) for b in range(70)], device="cuda")
    p.x[1] = (p.x[1] * size.repeat_interleave(torch.tensor(keys, device="cuda"))[:, None, None]).to(BF16)
    p.append()
    q = _randn(_gen(64), sum(new), 4, D, dtype=BF16)
    o = torch.full_like(q, 7.0)
    capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts(new), p.table, p.lens, max(new), True, None,
                        p.ks, p.vs)
    first = 0
    for n, k, v in zip(new, *(p.held(i) for i in (0, 1))):
        there = min(n, len(k))  # the rows before see no key
        rows = slice(first + n - there, first + n)
        ref = _reference(q[rows], k, v)
        _check(o[rows], ref[0], _bound(BF16, True, ref, len(k)))
        assert (o[first:first + n - there] == 0).all()
        first += n
    capi.stream_status()


@pytest.mark.parametrize("rows,cache", [(BF16, E4M3), (F16, I8), (F32, E4M3)])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("n", [1, 200])
def test_long_context_of_changing_sizes(cuda, rows, cache, D, n):
    """A context that many CTAs share: their pieces have references of their own, some of them over
    values of one size, some over several, zeros among them, and keys of several sizes too."""
    L = 20011
    q = _randn(_gen(66), n, 8, D, dtype=rows)
    sizes = (1.0, 1.0, 1.0, 2.0 ** -10, 0.0, 2.0 ** -10, 30.0) if rows == F16 else \
        (1.0, 1.0, 1.0, 1e-9, 0.0, 1e-9, 1e-9, 1e5)

    def keys(x):
        return x.float() * torch.where(torch.arange(L, device="cuda") % 97 == 0, 2.0 ** -9, 1.0)[:, None, None]

    p = _pool(L, 2, D, rows, cache, 67, keys, lambda x: x.float() * _blocks(L, sizes))
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))
    capi.stream_status()


@pytest.mark.parametrize("rows,cache", CODED)
@pytest.mark.parametrize("n", [1, 12, 300])
def test_first_key_takes_the_weight_and_has_no_value(cuda, rows, cache, n):
    """The first key's weight is 1 but for 2^-20 or so and its value is 0: what is left of the
    others comes out with its bits."""
    D, L = 64, 400
    q = _randn(_gen(68), n, 4, D, dtype=rows)
    q[..., 0] = 4.0

    def keys(x):
        x = x.clone()
        x[..., 0] = 0
        x[0] = 0
        x[0, :, 0] = 40.0
        return x

    def values(x):
        x = x.clone()
        x[0] = 0
        return x

    p = _pool(L, 2, D, rows, cache, 69, keys, values)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])
    _check(_attend(p, q), ref[0], _bound(rows, True, ref, L))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("paged", [False, True])
def test_fp32_sums_are_rounded(cuda, D, paged):
    """Root mean square of the error relative to the outputs'.  A product of split operands is off by
    2^-22 of its largest terms; sums that are rounded are off at random, by 2^-24 a step: for scores
    of up to 4 or so in units of log2 some 20 steps make 2^-24 * 4 * sqrt(20), and the outputs' own
    sums as much again, 1.2e-6 at worst and half of it in the mean square.  Sums that are cut off are
    off by half of 2^-23 at every one of 3 D / 8 steps, all to one side: 2e-6 and more."""
    n = 900
    g = _gen(70)
    q, k, v = _randn(g, n, 4, D) * 1.5, _randn(g, n, 2, D), _randn(g, n, 2, D)
    k *= _randn(g, 1, 2, D).abs() + 0.5
    ref = _reference(q, k, v)[0]
    if paged:
        p = _pool(n, 2, D, F32, F32, 71, lambda x: k, lambda x: v)
        o = _attend(p, q)
    else:
        o = torch.empty_like(q)
        capi.attn_packed_dev(q, k, v, o, seq_ref.starts([n]), causal=True)
    err = float((o.double().cpu() - ref).norm() / ref.norm())
    assert err <= 1e-6, err


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("n,L", [(1, 1500), (10, 1500), (200, 300), (300, 3000)])
@pytest.mark.parametrize("D", [64, 128])
def test_f16_over_codes_rounds_weights_and_outputs_only(cuda, cache, n, L, D):
    """Root mean square of the error relative to the outputs'.  A rounding to f16 is off by 2^-11 at
    most and evenly spread, 2^-11 / sqrt(3) * 0.75 in the mean square over a binade (values spread
    over it), 2.1e-4: one of the outputs, one of the weights, together 3.0e-4.  A third and fourth of
    keys or values, or any of scores, would pass 3.3e-4 by far: scores are several units large."""
    q = _randn(_gen(72), n, 8, D, dtype=F16) * 1.5
    p = _pool(L, 2, D, F16, cache, 73, lambda x: x.float() * 1.5)
    ref = _reference(q, p.held(0)[0], p.held(1)[0])[0]
    o = _attend(p, q).double().cpu()
    err = float((o - ref).norm() / ref.norm())
    assert err <= 3.3e-4, err
