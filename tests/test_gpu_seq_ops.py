"""Attention over packed prompts, the paged KV cache and attention over it, against 64-bit forms:
ragged lengths from none to thousands, every type, grouped heads, odd head sizes and strides, pages
in any order, stale NaN in what no query may see, bad page numbers, streams, graphs and replays."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import seq_ref
from attn_cpu import capi

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3, I8 = (torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn,
                            torch.int8)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _smax(q, k, scale=None):
    D = q.shape[-1]
    s = D ** -0.5 if scale is None else scale
    return float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * s if q.numel() and k.numel() else 1.0


def _check(o, ref, mag, dtype, smax, coded=False, L=1, floor=0.0):
    o = o.double().cpu()
    bound = seq_ref.attention_bound(dtype, mag, ref, smax, coded, ref.shape[-1], L) + floor
    bad = ~((o - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((o - ref).abs() / bound).nan_to_num(1e9).max()))


def _split(x, counts):
    return list(torch.split(x, counts)) if sum(counts) else [x[:0] for _ in counts]


# ------------------------------------------------------------------ packed prompts
LENGTHS = {
    "one": [1],
    "ragged": [5, 0, 64, 129, 1, 0, 300],
    "edges": [127, 128, 129, 255, 256, 257],
    "long": [1500, 3, 700],
}


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (6, 2, 33),
                                              (4, 1, 256), (20, 4, 96)])
@pytest.mark.parametrize("name", list(LENGTHS))
def test_packed(cuda, dtype, heads, kv_heads, D, name):
    new = LENGTHS[name]
    g = _gen(len(name) * 1000 + heads * 10 + D)
    n = sum(new)
    q = _randn(g, n, heads, D, dtype=dtype)
    k, v = (_randn(g, n, kv_heads, D, dtype=dtype) for _ in range(2))
    o = torch.full_like(q, float("nan"))
    cu = seq_ref.starts(new)
    for causal in (True, False):
        capi.attn_packed_dev(q, k, v, o, cu, causal=causal)
        ref, mag = seq_ref.attention(q, _split(k, new), _split(v, new), new, causal)
        _check(o, ref, mag, dtype, _smax(q, k), L=max(new))
    capi.stream_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_other_key_lengths(cuda, dtype, causal):
    """Keys that are more, fewer or none: rows without a key give zeros."""
    new, keys = [3, 130, 7, 40, 0, 200], [0, 500, 4, 40, 9, 61]
    g = _gen(5)
    q = _randn(g, sum(new), 4, 64, dtype=dtype)
    k, v = (_randn(g, sum(keys), 2, 64, dtype=dtype) for _ in range(2))
    o = torch.full_like(q, float("nan"))
    capi.attn_packed_dev(q, k, v, o, seq_ref.starts(new), seq_ref.starts(keys), causal=causal,
                         scale=0.2)
    ref, mag = seq_ref.attention(q, _split(k, keys), _split(v, keys), new, causal, 0.2)
    _check(o, ref, mag, dtype, _smax(q, k, 0.2), L=500)
    assert (o[:3] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_packed_strides_and_rows_behind(cuda, dtype):
    """q, k, v as slices of one projection, an output with gaps; rows of no sequence stay."""
    new, heads, kv, D = [70, 200], 8, 2, 64
    g = _gen(6)
    n = sum(new)
    qkv = _randn(g, n + 9, heads + 2 * kv, D, dtype=dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = torch.full((heads, n + 9, 2 * D), 7.0, dtype=dtype, device="cuda")
    o = out[:, :, :D].transpose(0, 1)
    capi.attn_packed_dev(q, k, v, o, seq_ref.starts(new), causal=True)
    ref, mag = seq_ref.attention(q[:n], _split(k[:n], new), _split(v[:n], new), new)
    _check(o[:n], ref, mag, dtype, _smax(q, k), L=200)
    assert (out[:, n:] == 7).all() and (out[:, :, D:] == 7).all()
    # misaligned rows: the same numbers one element further on
    flat = torch.empty(qkv.numel() + 1, dtype=dtype, device="cuda")
    odd = flat[1:].view_as(qkv).copy_(qkv)
    o2 = torch.empty(n + 9, heads, D, dtype=dtype, device="cuda")
    capi.attn_packed_dev(odd[:, :heads], odd[:, heads:heads + kv], odd[:, heads + kv:], o2,
                         seq_ref.starts(new), causal=True)
    _check(o2[:n], ref, mag, dtype, _smax(q, k), L=200)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_does_not_see_other_sequences(cuda, dtype):
    """NaN and infinities in the next sequence and behind the last one stay out of the others."""
    new, D = [50, 130, 20], 128
    g = _gen(7)
    n = sum(new)
    q = _randn(g, n + 5, 8, D, dtype=dtype)
    k, v = (_randn(g, n + 5, 2, D, dtype=dtype) for _ in range(2))
    ref, mag = seq_ref.attention(q[:n], _split(k[:n], new), _split(v[:n], new), new)
    smax = _smax(q, k)
    k[50:180], v[50:180], k[n:], v[n:] = float("nan"), float("inf"), float("nan"), float("nan")
    o = torch.zeros_like(q)
    capi.attn_packed_dev(q, k, v, o, seq_ref.starts(new), causal=True)
    for a, b in ((0, 50), (180, 200)):
        _check(o[a:b], ref[a:b], mag[a:b], dtype, smax, L=50)
    assert torch.isnan(o[50:180].float()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_future_values_stay_out(cuda, dtype):
    """A NaN or infinity in a later key of the same sequence does not reach earlier rows."""
    n, D = 300, 64
    g = _gen(8)
    q = _randn(g, n, 4, D, dtype=dtype)
    k, v = (_randn(g, n, 2, D, dtype=dtype) for _ in range(2))
    ref, mag = seq_ref.attention(q, [k], [v], [n])
    smax = _smax(q, k)
    k[200], v[230], v[290] = float("nan"), float("nan"), float("inf")
    o = torch.zeros_like(q)
    capi.attn_packed_dev(q, k, v, o, seq_ref.starts([n]), causal=True)
    _check(o[:200], ref[:200], mag[:200], dtype, smax, L=n)
    assert torch.isnan(o[200:].float()).all()


def test_packed_scores_of_any_size(cuda):
    """Scores far apart (one weight takes all), equal scores, and infinite keys."""
    n, D = 200, 64
    g = _gen(9)
    for dtype in (F32, BF16):
        q = _randn(g, n, 2, D, dtype=dtype) * 30
        k, v = (_randn(g, n, 1, D, dtype=dtype) * 20 for _ in range(2))
        o = torch.empty_like(q)
        capi.attn_packed_dev(q, k, v, o, seq_ref.starts([n]), causal=True)
        assert torch.isfinite(o.float()).all()
        ref, mag = seq_ref.attention(q, [k], [v], [n])
        _check(o, ref, mag, dtype, _smax(q, k), L=n)
        capi.attn_packed_dev(torch.zeros_like(q), k, v, o, seq_ref.starts([n]), causal=False)
        mean = v.double().cpu().mean(0, keepdim=True).expand(n, 2, D)
        _check(o, mean, v.double().cpu().abs().mean(0, keepdim=True).expand(n, 2, D), dtype, 1.0,
               L=n)


def test_packed_many_sequences(cuda):
    """More sequences than a CTA has threads, most of them tiny, some empty."""
    rng = np.random.default_rng(3)
    new = [int(x) for x in rng.integers(0, 9, 1500)]
    new[700] = 400
    g = _gen(10)
    for dtype in (F32, BF16):
        q = _randn(g, sum(new), 4, 64, dtype=dtype)
        k, v = (_randn(g, sum(new), 2, 64, dtype=dtype) for _ in range(2))
        o = torch.full_like(q, float("nan"))
        capi.attn_packed_dev(q, k, v, o, seq_ref.starts(new), causal=True)
        ref, mag = seq_ref.attention(q, _split(k, new), _split(v, new), new)
        _check(o, ref, mag, dtype, _smax(q, k), L=400)


# -------------------------------------------------------------- paged cache
def _fill(shape, dtype, g):
    """What earlier sequences and the allocator left in a pool: NaN among it."""
    if dtype == I8:
        return torch.randint(-128, 128, shape, device="cuda", generator=g, dtype=I8)
    return torch.full(shape, float("nan"), device="cuda").to(dtype)


class Pool:
    """Sequences of `keys` tokens in pages; what they hold, in 64 bits, in .k and .v."""

    def __init__(self, keys, H, D, page, rows_type, cache_type, seed, spare=3):
        gen = torch.Generator().manual_seed(seed)
        g = _gen(seed)
        need = sum(-(-n // page) for n in keys)
        self.page, self.keys = page, keys
        width = max(1, max(-(-n // page) for n in keys) + 1)
        self.table = seq_ref.random_pages(keys, page, need + spare, width, gen).cuda()
        self.lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
        self.kp, self.vp = (_fill((need + spare, H, page, D), cache_type, g) for _ in range(2))
        self.ks = self.vs = None
        if cache_type in seq_ref.TOP:
            self.ks, self.vs = (torch.full((need + spare, H, page), float("nan"), device="cuda")
                                for _ in range(2))
        n = sum(keys)
        self.x = [_randn(g, n, H, D, dtype=rows_type) * 1.5, _randn(g, n, H, D, dtype=rows_type)]

    def append(self, **kw):
        capi.kv_pages_append_dev(*self.x, self.kp, self.vp, seq_ref.starts(self.keys), self.table,
                                 self.lens, self.ks, self.vs, **kw)

    def held(self, i):
        """Token values per sequence as the pages hold them, read by indexing."""
        pages, scale = ((self.kp, self.ks), (self.vp, self.vs))[i]
        out = []
        for b, n in enumerate(self.keys):
            pos = torch.arange(n, device="cuda")
            pg, at = self.table[b].long()[pos // self.page], pos % self.page
            x = pages.float()[pg, :, at].double()
            if scale is not None:
                x = x * scale[pg, :, at].double()[..., None]
            out.append(x.cpu())
        return out


CACHES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, I8),
          (F16, I8), (F32, I8)]


@pytest.mark.parametrize("rows_type,cache_type", CACHES)
@pytest.mark.parametrize("H,D,page", [(2, 64, 16), (1, 128, 64), (3, 40, 32), (2, 33, 128),
                                      (1, 256, 16)])
def test_append_and_read(cuda, rows_type, cache_type, H, D, page):
    keys = [1, 0, 17, 64, 200]
    p = Pool(keys, H, D, page, rows_type, cache_type, D + page)
    x = p.x[0]
    x[3] = 0  # a vector of zeros
    x[5, 0, :] = x[5, 0, 0]  # equal values
    x[6] *= 1e-3
    p.x[1][7] *= 1000
    p.append()
    for i in (0, 1):
        src = p.x[i]
        if cache_type in seq_ref.TOP:
            codes, scale = seq_ref.quantise(src, cache_type)
            pages, scales = ((p.kp, p.ks), (p.vp, p.vs))[i]
            first = 0
            for b, n in enumerate(keys):
                pos = torch.arange(n, device="cuda")
                pg, at = p.table[b].long()[pos // page], pos % page
                assert torch.equal(pages.float()[pg, :, at].double().cpu(), codes[first:first + n])
                assert torch.equal(scales[pg, :, at].cpu(), scale[first:first + n])
                first += n
        else:
            assert torch.equal(torch.cat(p.held(i)), src.double().cpu())
    out = [torch.full_like(x, 5.0) for x in p.x]
    capi.kv_pages_read_dev(p.kp, p.vp, *out, seq_ref.starts(keys), p.table, p.lens, p.ks, p.vs)
    for i in (0, 1):
        want = torch.cat(p.held(i)).float().to(rows_type)
        assert torch.equal(out[i].cpu(), want)
    # the last tokens only, into strided rows with some of no sequence behind
    some = [0, 0, 3, 64, 190]
    wide = [torch.full((sum(some) + 4, H, 2 * D), 5.0, dtype=rows_type, device="cuda")
            for _ in range(2)]
    capi.kv_pages_read_dev(p.kp, p.vp, *(w[..., :D] for w in wide), seq_ref.starts(some), p.table,
                           p.lens, p.ks, p.vs)
    for i in (0, 1):
        want = torch.cat([h[len(h) - n:] for h, n in zip(p.held(i), some)]).float().to(rows_type)
        assert torch.equal(wide[i][:sum(some), :, :D].cpu(), want)
        assert (wide[i][sum(some):] == 5).all() and (wide[i][..., D:] == 5).all()
    capi.stream_status()


@pytest.mark.parametrize("cache_type", [E4M3, I8])
@pytest.mark.parametrize("rows_type", [F32, BF16, F16])
def test_codes_at_borders(cuda, rows_type, cache_type):
    """Values on and next to the borders between codes, and a range of magnitudes."""
    top = seq_ref.TOP[cache_type]
    g = _gen(4)
    x = _randn(g, 512, 1, 128)
    x[:128] = (torch.randint(-253, 254, (128, 1, 128), device="cuda", generator=g) / 2.0)
    x[:128, 0, 0] = top  # scale 1: halves are ties
    x[128:256] = torch.exp2(torch.randint(-12, 9, (128, 1, 128), device="cuda", generator=g).float()) * 1.0625
    x[128:256, 0, 0] = top
    if rows_type == F32:  # one fp32 step to either side of a tie
        x[256:384] = torch.nextafter(x[:128], torch.full_like(x[:128], 1e9))
        x[256:384, 0, 0] = top
        x[384:] *= 1e30
    elif rows_type == BF16:
        x[384:] *= 1e37
    else:
        x[384:] *= 1e-5
    x = x.to(rows_type)
    p = Pool([512], 1, 128, 32, rows_type, cache_type, 4)
    p.x = [x, x.clone()]
    p.append()
    codes, scale = seq_ref.quantise(x, cache_type)
    pos = torch.arange(512, device="cuda")
    pg, at = p.table[0].long()[pos // 32], pos % 32
    got = p.kp.float()[pg, :, at].double().cpu()
    assert torch.equal(got, codes), int((got != codes).sum())
    assert torch.equal(p.vs[pg, :, at].cpu(), scale)


@pytest.mark.parametrize("cache_type", [E4M3, I8])
def test_not_finite_vectors(cuda, cache_type):
    p = Pool([40], 2, 64, 16, BF16, cache_type, 5)
    p.x[0][3, 1, 5] = float("nan")
    p.x[1][9, 0, 63] = float("-inf")
    p.append()
    out = [torch.empty_like(x) for x in p.x]
    capi.kv_pages_read_dev(p.kp, p.vp, *out, seq_ref.starts([40]), p.table, p.lens, p.ks, p.vs)
    assert torch.isnan(out[0][3, 1].float()).all() and torch.isnan(out[1][9, 0].float()).all()
    assert int(torch.isnan(out[0].float()).sum()) == 64 == int(torch.isnan(out[1].float()).sum())


@pytest.mark.parametrize("rows_type,cache_type", CACHES)
@pytest.mark.parametrize("heads,H,D,page", [(8, 2, 128, 16), (8, 8, 64, 64), (10, 2, 80, 128),
                                            (3, 1, 33, 32), (4, 1, 256, 16), (32, 1, 64, 32)])
def test_paged(cuda, rows_type, cache_type, heads, H, D, page):
    keys = [1, 300, 17, 0, 64, 1100, 128, 5]
    p = Pool(keys, H, D, page, rows_type, cache_type, heads + D)
    p.append()
    ks, vs = p.held(0), p.held(1)
    coded = cache_type in seq_ref.TOP
    g = _gen(D)
    for new in ([1, 1, 1, 0, 1, 1, 1, 1], [1, 5, 17, 0, 30, 300, 128, 2], [0, 0, 0, 3, 0, 1, 2, 9]):
        q = _randn(g, sum(new), heads, D, dtype=rows_type)
        smax = float(q.double().norm(dim=-1).max() * torch.cat(ks).norm(dim=-1).max()) * D ** -0.5
        for causal in (True, False):
            o = torch.full_like(q, float("nan"))
            capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts(new), p.table, p.lens, max(new),
                                causal, None, p.ks, p.vs)
            ref, mag = seq_ref.attention(q, ks, vs, new, causal)
            _check(o, ref, mag, rows_type, smax, coded, max(keys))
    capi.stream_status()


@pytest.mark.parametrize("rows_type,cache_type", [(BF16, BF16), (F16, I8), (BF16, E4M3), (F32, F32)])
@pytest.mark.parametrize("new", [1, 3, 77, 600])
def test_paged_one_long_context(cuda, rows_type, cache_type, new):
    """A context that is split over all CTAs; max_new unknown and known alike."""
    n = 20011
    p = Pool([n], 2, 128, 64, rows_type, cache_type, new)
    p.append()
    q = _randn(_gen(1), new, 8, 128, dtype=rows_type)
    ks, vs = p.held(0), p.held(1)
    ref, mag = seq_ref.attention(q, ks, vs, [new])
    smax = float(q.double().norm(dim=-1).max() * ks[0].norm(dim=-1).max()) * 128 ** -0.5
    for most in (0, new, 1):
        o = torch.empty_like(q)
        capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts([new]), p.table, p.lens, most, True,
                            None, p.ks, p.vs)
        _check(o, ref, mag, rows_type, smax, cache_type in seq_ref.TOP, n)


@pytest.mark.parametrize("rows_type,cache_type", [(BF16, BF16), (F16, I8), (F32, E4M3)])
@pytest.mark.parametrize("new", [1, 200])
def test_bad_pages_and_lengths(cuda, rows_type, cache_type, new):
    """Page numbers out of range read as zeros and are not written, lengths are clamped to the
    table, and the status tells; the other sequences are untouched by it."""
    keys = [300, 400, 250]
    p = Pool(keys, 2, 64, 32, rows_type, cache_type, 3)
    p.append()
    capi.stream_status()
    ks, vs = p.held(0), p.held(1)
    p.table[1, 2], p.table[1, 5] = 10 ** 6, -7
    for x in (ks, vs):
        x[1][64:96] = 0
        x[1][160:192] = 0
    count = [new] * 3
    q = _randn(_gen(2), 3 * new, 4, 64, dtype=rows_type)
    smax = float(q.double().norm(dim=-1).max() * torch.cat(ks).norm(dim=-1).max()) * 64 ** -0.5
    o = torch.empty_like(q)
    capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts(count), p.table, p.lens, new, True, None,
                        p.ks, p.vs)
    ref, mag = seq_ref.attention(q, ks, vs, count)
    _check(o, ref, mag, rows_type, smax, cache_type in seq_ref.TOP, 400)
    with pytest.raises(capi.AttnbError, match="out of range") as e:
        capi.stream_status()
    assert e.value.code == capi.ERR_INDEX
    capi.stream_status()  # cleared
    # a length past the table, a negative one: no fault, and the status tells
    before = p.kp.clone()
    lens = torch.tensor([300, 10 ** 9, -5], dtype=torch.int32, device="cuda")
    capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts(count), p.table, lens, new, True, None,
                        p.ks, p.vs)
    _check(o[:new], ref[:new], mag[:new], rows_type, smax, cache_type in seq_ref.TOP, 400)
    assert (o[2 * new:] == 0).all()
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()
    capi.kv_pages_append_dev(p.x[0][:3], p.x[1][:3], p.kp, p.vp, seq_ref.starts([0, 2, 1]), p.table,
                             lens, p.ks, p.vs)
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()
    assert torch.equal(before.view(torch.uint8), p.kp.view(torch.uint8))
    # offsets that are not sorted or leave the rows: clamped
    cu = torch.tensor([-3, 10 ** 8, 5, 2 * new], dtype=torch.int32, device="cuda")
    capi.attn_paged_dev(q, p.kp, p.vp, o, cu, p.table, p.lens, new, True, None, p.ks, p.vs)
    k = _randn(_gen(3), 3 * new, 2, 64, dtype=rows_type)
    capi.attn_packed_dev(q, k, k, o, cu, cu, causal=True)
    torch.cuda.synchronize()


def test_long_pool_offsets_pass_32_bits(cuda):
    """The pages that are read and written lie more than 2^31 elements into the pool."""
    H, page, D = 8, 128, 128
    num = 2 ** 31 // (H * page * D) + 40
    kp = torch.empty(num, H, page, D, dtype=BF16, device="cuda")
    g = _gen(11)
    n = 1000
    k, v, q = (_randn(g, n, h, D, dtype=BF16) for h in (8, 8, 16))
    vp = torch.empty_like(kp)
    table = torch.arange(num - 1, num - 11, -1, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = seq_ref.starts([n])
    capi.kv_pages_append_dev(k, v, kp, vp, cu, table, lens)
    back = [torch.empty_like(k), torch.empty_like(v)]
    capi.kv_pages_read_dev(kp, vp, *back, cu, table, lens)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    o, o1 = torch.empty_like(q), torch.empty_like(q[:1])
    capi.attn_paged_dev(q, kp, vp, o, cu, table, lens, n)
    ref, mag = seq_ref.attention(q, [k], [v], [n])
    _check(o, ref, mag, BF16, _smax(q, k), L=n)
    capi.attn_paged_dev(q[-1:], kp, vp, o1, seq_ref.starts([1]), table, lens, 1)
    _check(o1, ref[-1:], mag[-1:], BF16, _smax(q, k), L=n)
    capi.stream_status()


def test_streams_and_graphs(cuda):
    """Two calls at once on two streams, and a captured step replayed with other lengths, offsets
    and pages while an eager call runs: each equals the same call alone."""
    H, D, page = 2, 128, 32
    p = Pool([500, 900, 77, 30], H, D, page, BF16, E4M3, 12)
    p.append()
    new = [1, 1, 1, 1]
    g = _gen(12)
    q = _randn(g, 4, 8, D, dtype=BF16)
    big = _randn(g, 900, 8, D, dtype=BF16)
    cu, cub = seq_ref.starts(new), seq_ref.starts([0, 900, 0, 0])

    def step(q, cu, lens, most, o):
        capi.attn_paged_dev(q, p.kp, p.vp, o, cu, p.table, lens, most, True, None, p.ks, p.vs)

    alone, alone_big = torch.empty_like(q), torch.empty_like(big)
    step(q, cu, p.lens, 1, alone)
    step(big, cub, p.lens, 900, alone_big)
    other_lens = torch.tensor([123, 800, 5, 1], dtype=torch.int32, device="cuda")
    alone_other = torch.empty_like(q)
    step(q, cu, other_lens, 1, alone_other)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        o1, o2 = torch.zeros_like(q), torch.zeros_like(big)
        s1.wait_stream(torch.cuda.current_stream())
        s2.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s1):
            step(q, cu, p.lens, 1, o1)
        capi.attn_paged_dev(big, p.kp, p.vp, o2, cub, p.table, p.lens, 900, True, None, p.ks, p.vs,
                            stream=s2)
        outs.append((o1, o2))
    torch.cuda.synchronize()
    for o1, o2 in outs:
        assert torch.equal(o1, alone) and torch.equal(o2, alone_big)
    lens, o = p.lens.clone(), torch.zeros_like(q)
    ob = torch.zeros_like(big)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, cu, lens, 1, o)
    with torch.cuda.graph(graph2):
        step(big, cub, p.lens, 900, ob)
    for want, ln in ((alone, p.lens), (alone_other, other_lens), (alone, p.lens)):
        lens.copy_(ln)
        o.zero_()
        ob.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graph.replay()
        with torch.cuda.stream(s2):
            graph2.replay()
        eager = torch.zeros_like(big)
        step(big, cub, p.lens, 900, eager)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(ob, alone_big) and torch.equal(eager, alone_big)


@pytest.mark.parametrize("dtype", [BF16, E4M3, I8])
def test_serving_run(cuda, dtype):
    """Prompts, then steps and chunks, through the cache object: every output equals attention over
    the tokens so far, as the cache holds them; sequences end and others take their pages."""
    rng = np.random.default_rng(8)
    B, H, heads, D = 5, 2, 8, 64
    cache = capi.PagedKVCacheDev(B, H, D, num_pages=60, page_size=16, dtype=dtype)
    g = _gen(20)
    hist = [[torch.zeros(0, H, D, dtype=BF16, device="cuda") for _ in range(B)] for _ in range(2)]
    plan = [[40, 0, 130, 7, 1], [1, 20, 1, 1, 1], [1, 1, 1, 0, 33], "end 2", [1, 1, 90, 1, 1],
            [0, 0, 0, 0, 0], [4, 1, 1, 5, 2]]
    for new in plan:
        if new == "end 2":
            cache.truncate(2, 0)
            cache.truncate(0, 30)
            for x in hist:
                x[2], x[0] = x[2][:0], x[0][:30]
            continue
        n = sum(new)
        q, k, v = (_randn(g, n, h, D, dtype=BF16) for h in (heads, H, H))
        cache.append(k, v, new)
        for x, y in zip(hist, (k, v)):
            for b, part in enumerate(_split(y, new)):
                x[b] = torch.cat([x[b], part])
        assert cache.lengths == [len(x) for x in hist[0]]
        o = torch.full_like(q, float("nan"))
        cache.attend(q, o)
        held = []
        for x in hist:
            if dtype in seq_ref.TOP:
                coded = [seq_ref.quantise(t, dtype) for t in x]
                held.append([codes * scale.double()[..., None] for codes, scale in coded])
            else:
                held.append(x)
        ref, mag = seq_ref.attention(q, *held, new)
        smax = _smax(q.cpu(), torch.cat([h.double().cpu() for h in held[0]]))
        _check(o, ref, mag, BF16, smax, dtype in seq_ref.TOP, 200)
    b = 4
    k, v = (torch.empty(cache.lengths[b], H, D, dtype=BF16, device="cuda") for _ in range(2))
    cache.read(b, k, v)
    want = held[0][b].double().cpu() if dtype == BF16 else held[0][b]
    assert (k.double().cpu() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    with pytest.raises(ValueError, match="too few free pages"):
        cache.append(*(torch.zeros(900, H, D, dtype=BF16, device="cuda") for _ in range(2)),
                     [900, 0, 0, 0, 0])
    with pytest.raises(ValueError, match="sum"):
        cache.append(k, v, [0, 0, 0, 0, 0])
    capi.stream_status()


def test_python_layer_refusals(cuda):
    q, k = torch.zeros(4, 4, 64, device="cuda"), torch.zeros(4, 2, 64, device="cuda")
    cu = seq_ref.starts([4])
    with pytest.raises(ValueError, match="int32"):
        capi.attn_packed_dev(q, k, k, q.clone(), cu.long())
    with pytest.raises(ValueError, match="not on|must be on"):
        capi.attn_packed_dev(q, k.cpu(), k, q.clone(), cu)
    with pytest.raises(ValueError, match="unit stride"):
        capi.attn_packed_dev(q.transpose(1, 2), k, k, q.clone(), cu)
    with pytest.raises(ValueError, match="multiple"):
        capi.attn_packed_dev(q[:, :3], k, k, q[:, :3].clone(), cu)
    with pytest.raises(ValueError, match="not supported"):
        capi.attn_packed_dev(q.double(), k.double(), k.double(), q.double(), cu)
    with pytest.raises(ValueError, match="scale must be positive"):
        capi.attn_packed_dev(q, k, k, q.clone(), cu, scale=0)
    pages = torch.zeros(3, 2, 16, 64, device="cuda")
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), seq_ref.starts([])[:1]
    with pytest.raises(ValueError, match="contiguous"):
        capi.attn_paged_dev(q, pages.transpose(0, 1), pages.transpose(0, 1), q.clone(), cu, table,
                            lens)
    with pytest.raises(ValueError, match="one type"):
        capi.attn_paged_dev(q, pages, pages.half(), q.clone(), cu, table, lens)
    with pytest.raises(ValueError, match="entries"):
        capi.attn_paged_dev(q, pages, pages, q.clone(), seq_ref.starts([2, 2]), table, lens)
    with pytest.raises(ValueError, match="float32"):
        capi.kv_pages_append_dev(k, k, pages.to(E4M3), pages.to(E4M3), cu, table, lens,
                                 torch.zeros(3, 2, 16, device="cuda").half(),
                                 torch.zeros(3, 2, 16, device="cuda"))
    with pytest.raises(capi.AttnbError, match="workspace too small"):
        o = q.clone()
        capi.check(capi.lib().attnb_attn_packed_dev(
            *(capi._rows(t, "x", q.device) for t in (q, k, k, o)), cu.data_ptr(), cu.data_ptr(), 1,
            1, 0.0, o.data_ptr(), 64, capi._stream()))


def test_cache_object_refused_append_and_truncated_read(cuda):
    """A rejected append leaves the cache as it was; a truncated sequence reads back its prefix."""
    H, D = 2, 64
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=12, page_size=16, dtype=BF16)
    g = _gen(30)
    k, v = (_randn(g, 70, H, D, dtype=BF16) for _ in range(2))
    cache.append(k, v, [50, 20])
    with pytest.raises(capi.AttnbError, match="matching the pages"):
        cache.append(*(torch.zeros(60, H + 1, D, dtype=BF16, device="cuda") for _ in range(2)),
                     [60, 0])
    assert cache.lengths == [50, 20]
    k2, v2 = (_randn(g, 3, H, D, dtype=BF16) for _ in range(2))
    cache.append(k2, v2, [3, 0])
    cache.truncate(0, 33)
    back = [torch.empty(33, H, D, dtype=BF16, device="cuda") for _ in range(2)]
    cache.read(0, *back)
    assert torch.equal(back[0], k[:33]) and torch.equal(back[1], v[:33])
    back = [torch.empty(20, H, D, dtype=BF16, device="cuda") for _ in range(2)]
    cache.read(1, *back)
    assert torch.equal(back[0], k[50:]) and torch.equal(back[1], v[50:])
    with pytest.raises(ValueError, match="append first"):
        cache.attend(k[:1].expand(1, H, D), torch.empty(1, H, D, dtype=BF16, device="cuda"))


@pytest.mark.parametrize("cache_type", [E4M3, I8])
@pytest.mark.parametrize("new", [1, 60])
def test_queries_and_keys_of_any_magnitude(cuda, cache_type, new):
    """Rows of queries next to overflow, tiny ones and zeros, and keys and values whose scales are
    far apart: codes and rows are brought to f16 by powers of two."""
    p = Pool([200], 1, 64, 16, BF16, cache_type, 31)
    p.x[0][:] *= 2.0 ** -100
    p.x[1][::3] *= 2.0 ** -20
    p.x[1][1::3] *= 2.0 ** 30
    p.append()
    q = _randn(_gen(31), new, 4, 64, dtype=BF16)
    q *= 2.0 ** 100
    q[:, 2] = 0
    q[:, 3] = (q[:, 3].sign() * 1.5) * 2.0 ** 127  # scores of 2^28: one key takes all
    o = torch.empty_like(q)
    capi.attn_paged_dev(q, p.kp, p.vp, o, seq_ref.starts([new]), p.table, p.lens, new, True, None,
                        p.ks, p.vs)
    ks, vs = p.held(0), p.held(1)
    ref, mag = seq_ref.attention(q, ks, vs, [new])
    assert torch.isfinite(o.float()).all() and (o[:, 3] != 0).any()
    # Weights and values are f16 over codes.  Below 2^-14 f16 has steps of 2^-24, so a weight is off
    # by up to 2^-25 of the row's largest one (which is at least 1 before it is rounded, and at most
    # the sum it is divided by): 2^-25 sum |v_j| in all.  A value is off by up to 2^-25 of a unit that
    # is at most the largest |v| of its 64 keys, twice (two roundings), and the weights sum to 1.
    v = vs[0][:, 0].abs()
    floor = 2.0 ** -25 * v.sum(0) + 2.0 ** -24 * v.max()
    _check(o[:, :3], ref[:, :3], mag[:, :3], BF16, _smax(q[:, :3].cpu(), ks[0]), True, 200, floor)


def test_no_keys_at_all(cuda):
    for dtype in (F32, BF16):
        q = _randn(_gen(32), 20, 4, 64, dtype=dtype)
        k = q[:0, :2]
        o = torch.full_like(q, float("nan"))
        none = torch.zeros(3, dtype=torch.int32, device="cuda")
        capi.attn_packed_dev(q, k, k, o, seq_ref.starts([5, 15]), none)
        assert (o == 0).all()


def test_masked_infinities_in_many_short_sequences(cuda):
    """Sequences of a tile or less, every second one with values that only its last row may see:
    the notes about masked values of one item do not reach its neighbours."""
    new = [3, 70, 1, 40, 129, 5] * 120
    D, g = 64, _gen(33)
    q = _randn(g, sum(new), 4, D, dtype=BF16)
    k, v = (_randn(g, sum(new), 2, D, dtype=BF16) for _ in range(2))
    ref, mag = seq_ref.attention(q, _split(k, new), _split(v, new), new)
    smax = _smax(q, k)
    first, last = [], 0
    for i, n in enumerate(new):
        last += n
        if i % 2 and n > 1:
            v[last - 1] = float("inf") if i % 4 == 1 else float("nan")
            first.append(last - 1)
    o = torch.full_like(q, 3.0)
    capi.attn_packed_dev(q, k, v, o, seq_ref.starts(new), causal=True)
    poisoned = torch.zeros(len(q), dtype=torch.bool)
    poisoned[first] = True
    assert not torch.isfinite(o[poisoned.cuda()].float()).any()
    _check(o[~poisoned.cuda()], ref[~poisoned], mag[~poisoned], BF16, smax, L=130)
    capi.stream_status()
