"""The cache in 4 bits: codes, factors and scales to the last bit, reading back, and attention over it in
every kernel against 64-bit forms."""
from __future__ import annotations

import pytest
import torch

import seq_ref
import seq_ref_more as more
from attn_cpu import capi
from test_gpu_rope_append import I4, Pages
from test_gpu_seq_ops import BF16, F16, F32, _check, _gen, _randn, _split

pytestmark = pytest.mark.gpu


def _held(p, name, b, n):
    """The first n tokens of sequence b as the pages hold them, [n, H, D] in 64 bits."""
    at = p.table[b, : -(-n // p.page)].long()
    x = more.values4(getattr(p, name)[at], p.kw[name + "_scale"][at], p.kw[name + "_group"][at])
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:n]


def _rows(g, n, H, D, dtype):
    """Vectors of all kinds: strong channels, quiet groups, zeros, ties, extremes of the type."""
    x = _randn(g, n, H, D, dtype=F32)
    x *= torch.exp(2 * _randn(g, 1, H, D))
    top = {F32: 3e38, BF16: 3e38, F16: 65504.0}[dtype]
    low = {F32: 2.0 ** -140, BF16: 2.0 ** -130, F16: 2.0 ** -22}[dtype]
    if n > 12:
        x[1] = 0
        x[2, :, 32:] = 0
        x[3, :, :32] *= 1e-6
        x[4] = torch.randint(-14, 15, (H, D), device="cuda", generator=g) / 2.0  # ties
        x[4, :, 0] = 7
        x[5] = torch.randint(-14, 15, (H, D), device="cuda", generator=g) / 2.0 * 17  # of other factors
        x[6] = x[6] / x[6].abs().amax() * top
        x[7] = x[7] / x[7].abs().amax() * low
        x[8, :, 5] = float("inf")
        x[9, :, 6] = float("nan")
        x[10] = -x[4]
        x[11] = 1
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 256])
def test_codes(cuda, dtype, D):
    new, keys, H = [60, 0, 1, 300], [60, 9, 33, 411], 3
    p = Pages(keys, H, D, 16, I4)
    for t in (p.k, p.v, *p.kw.values()):  # whatever was there before
        t.view(torch.uint8).fill_(0xA5)
    n = sum(new)
    g = _gen(D)
    k, v = (_rows(g, n, H, D, dtype) for _ in range(2))
    capi.kv_pages_append_dev(k, v, p.k, p.v, *p.where(new), **p.kw)
    at, slot = _places(p, new, keys)
    for x, name in ((k, "k"), (v, "v")):
        codes, factor, scale = more.quantise4(x.nan_to_num(0, 0, 0) * torch.isfinite(x).all(-1, keepdim=True))
        pages = getattr(p, name)[at, :, slot].cpu()
        got = torch.stack([pages & 15, pages >> 4], -1).flatten(-2).double() - 8
        bad = ~torch.isfinite(x).all(-1).cpu()
        got_scale = p.kw[name + "_scale"][at, :, slot].cpu()
        assert torch.isnan(got_scale[bad]).all() and torch.equal(got_scale[~bad], scale[~bad])
        got_factor = p.kw[name + "_group"][at, :, slot].cpu().double()
        assert torch.equal(got_factor[..., : D // 32], factor) and (got_factor[..., D // 32:] == 0).all()
        assert torch.equal(got, codes)
    # and back: one product in fp32, one rounding to the type
    back = [torch.full_like(k, 7), torch.full_like(v, 7)]
    capi.kv_pages_read_dev(p.k, p.v, *back, *p.where(new), **p.kw)
    for x, name in zip(back, ("k", "v")):
        t = torch.stack([(y := getattr(p, name)[at, :, slot]) & 15, y >> 4], -1).flatten(-2).float() - 8
        f = p.kw[name + "_group"][at, :, slot][..., : D // 32].float().repeat_interleave(32, -1)
        want = (t * f * p.kw[name + "_scale"][at, :, slot][..., None]).to(dtype)
        assert torch.equal(x.nan_to_num(5), want.nan_to_num(5)) and torch.equal(torch.isnan(x), torch.isnan(want))
    capi.stream_status()


def _places(p, new, keys):
    at, slot = [], []
    for b, (n, k) in enumerate(zip(new, keys)):
        pos = torch.arange(k - n, k, device="cuda")
        at.append(p.table[b, pos // p.page].long())
        slot.append(pos % p.page)
    return torch.cat(at), torch.cat(slot)


def _filled(keys, H, D, page, dtype, seed=1, spread=1.0):
    """Pages that hold all tokens of the sequences."""
    p = Pages(keys, H, D, page, I4, seed)
    g = _gen(seed)
    k, v = (_randn(g, sum(keys), H, D, dtype=F32) * torch.exp(spread * _randn(g, 1, H, D)) for _ in range(2))
    capi.kv_pages_append_dev(k.to(dtype), v.to(dtype), p.k, p.v, *p.where(keys), **p.kw)
    return p


def _attend(p, q, new, most=0, causal=True, scale=None):
    o = torch.full_like(q, float("nan"))
    capi.attn_paged_dev(q, p.k, p.v, o, *p.where(new), most, causal, scale, **p.kw)
    return o


def _against(p, q, new, keys, dtype, most=0, causal=True, scale=None):
    ks, vs = ([_held(p, x, b, n) for b, n in enumerate(keys)] for x in ("k", "v"))
    ref, mag = seq_ref.attention(q, ks, vs, new, causal, scale)
    D = q.shape[-1]
    smax = float(q.double().norm(dim=-1).max().cpu() * max(k.norm(dim=-1).max() for k in ks if len(k)))
    smax *= D ** -0.5 if scale is None else scale
    floor = 0.0 if dtype == F32 else more.weight_floor(q, ks, vs, new, causal, scale)
    _check(_attend(p, q, new, most, causal, scale), ref, mag, dtype, smax, True, max(keys), floor)
    capi.stream_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 64, 16), (8, 2, 128, 64), (6, 1, 96, 32), (3, 3, 32, 16), (4, 1, 256, 128),
                                                   (40, 2, 128, 32), (8, 4, 160, 16), (64, 4, 64, 128)])
@pytest.mark.parametrize("new,keys", [([1, 1, 1], [1, 77, 400]), ([1, 0, 3, 20], [1, 5, 3, 250]), ([130, 64, 1], [130, 500, 63])])
def test_attention(cuda, dtype, heads, kv_heads, D, page, new, keys):
    p = _filled(keys, kv_heads, D, page, dtype)
    q = _randn(_gen(2), sum(new), heads, D, dtype=dtype)
    _against(p, q, new, keys, dtype, max(new))
    if max(new) > 1:
        _against(p, q, new, keys, dtype, 0, False, 0.07)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3, 77, 600])
def test_one_long_context(cuda, dtype, new):
    keys = [20011]
    p = _filled(keys, 2, 128, 64, dtype, spread=0.3)
    q = _randn(_gen(3), new, 8, 128, dtype=dtype)
    for most in (0, new, 1):
        _against(p, q, [new], keys, dtype, most)


@pytest.mark.parametrize("new", [1, 200])
def test_values_of_any_size(cuda, new):
    """V from 2^-100 to 2^60, zeros among it, and sizes that change from block to block; groups that
    are far smaller than the others of their vector come out as exactly as their codes are."""
    keys, H, D = [700], 1, 128
    g = _gen(8)
    for kind in range(4):
        p = Pages(keys, H, D, 16, I4)
        k, v = (_randn(g, 700, H, D) for _ in range(2))
        if kind == 0:
            v *= 2.0 ** -100
        elif kind == 1:
            v *= 2.0 ** 60
        elif kind == 2:
            v *= 2.0 ** (torch.arange(700, device="cuda") // 64 * 9 % 100 - 50)[:, None, None]
            v[100:300] = 0
        else:
            v[..., 32:64] *= 2.0 ** -7
        k, v = k.to(BF16), v.to(BF16)
        capi.kv_pages_append_dev(k, v, p.k, p.v, *p.where(keys), **p.kw)
        q = _randn(g, new, 4, D, dtype=BF16)
        _against(p, q, [new], keys, BF16)


@pytest.mark.parametrize("new", [1, 5, 200])
@pytest.mark.parametrize("by", [(115, -115), (100, -100), (-100, 100), (-110, 118), (60, -50)])
def test_queries_and_keys_of_any_size(cuda, new, by):
    """Large queries over small keys and the other way round, scores of ordinary size or one far above
    the others."""
    keys, H, D = [500], 1, 128
    g = _gen(9)
    p = Pages(keys, H, D, 64, I4)
    k, v = (_randn(g, 500, H, D) for _ in range(2))
    k = (k * 2.0 ** by[1]).to(BF16)
    capi.kv_pages_append_dev(k, v.to(BF16), p.k, p.v, *p.where(keys), **p.kw)
    q = (_randn(g, new, 4, D) * 2.0 ** by[0]).to(BF16)
    if by[0] + by[1] <= 0:
        _against(p, q, [new], keys, BF16, new)
        return
    # Rows whose best key is 30 above the next have no other: 500 e^-30 is below 2^-34.  They get that
    # key's value.
    ks, vs = _held(p, "k", 0, 500), _held(p, "v", 0, 500)
    s = torch.einsum("ihd,jd->ihj", q.double().cpu(), ks[:, 0])
    s = s.masked_fill(~torch.ones(new, 500, dtype=torch.bool).tril(500 - new)[:, None], -torch.inf)
    o = _attend(p, q, [new], new).double().cpu()
    top = s.topk(2, -1)
    sure = (top.values[..., 0] - top.values[..., 1]) * D ** -0.5 > 30
    assert sure.any() and torch.isfinite(o).all()
    want = vs[:, 0][top.indices[..., 0]]
    assert ((o - want).abs()[sure] <= 2.0 ** -7 * want.abs()[sure] + 1e-6).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 100])
def test_stale_pages_stay_out(cuda, dtype, new):
    """What lies in the pages behind a sequence's last token, NaN scales among it, does not count."""
    keys = [100, 333]
    p = _filled(keys, 2, 64, 32, dtype)
    ks, vs = ([_held(p, x, b, n) for b, n in enumerate(keys)] for x in ("k", "v"))
    for b, n in enumerate(keys):
        last = p.table[b, (n - 1) // 32]
        for t in (p.k, p.v, p.kw["k_group"], p.kw["v_group"]):
            t[last, :, n % 32 or 32:] = 255
        for name in ("k_scale", "v_scale"):
            p.kw[name][last, :, n % 32 or 32:] = float("nan")
    count = [new, new]
    q = _randn(_gen(4), 2 * new, 4, 64, dtype=dtype)
    ref, mag = seq_ref.attention(q, ks, vs, count)
    smax = float(q.double().norm(dim=-1).max().cpu() * max(k.norm(dim=-1).max() for k in ks)) / 8
    floor = 0.0 if dtype == F32 else more.weight_floor(q, ks, vs, count)
    _check(_attend(p, q, count, new), ref, mag, dtype, smax, True, 333, floor)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 60])
def test_vectors_that_are_not_finite(cuda, dtype, new):
    """A key that is not finite makes the rows that see it NaN, and no other."""
    keys = [300]
    p = Pages(keys, 1, 64, 16, I4)
    k, v = (_randn(_gen(6), 300, 1, 64, dtype=dtype) for _ in range(2))
    k[270, 0, 3] = float("inf")
    capi.kv_pages_append_dev(k, v, p.k, p.v, *p.where(keys), **p.kw)
    q = _randn(_gen(7), new, 4, 64, dtype=dtype)
    o = _attend(p, q, [new], new)
    sees = torch.arange(300 - new, 300) >= 270
    assert torch.isnan(o.float()[sees.cuda()]).all()
    assert torch.isfinite(o.float()[~sees.cuda()]).all()


def test_bad_pages(cuda):
    keys = [300, 200]
    p = _filled(keys, 2, 64, 32, BF16)
    ks, vs = ([_held(p, x, b, n) for b, n in enumerate(keys)] for x in ("k", "v"))
    p.table[0, 2] = -9
    for x in (ks, vs):
        x[0][64:96] = 0
    for new in (1, 100):
        q = _randn(_gen(4), 2 * new, 4, 64, dtype=BF16)
        ref, mag = seq_ref.attention(q, ks, vs, [new, new])
        smax = float(q.double().norm(dim=-1).max().cpu() * max(k.norm(dim=-1).max() for k in ks)) / 8
        _check(_attend(p, q, [new, new], new), ref, mag, BF16, smax, True, 300,
               more.weight_floor(q, ks, vs, [new, new]))
        with pytest.raises(capi.AttnbError, match="out of range"):
            capi.stream_status()


def test_cache_object(cuda):
    """The paged cache object in 4 bits, with the rotation on the way."""
    H, heads, D = 2, 8, 128
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=30, page_size=32, dtype=torch.uint8)
    f = (10000.0 ** (-torch.arange(64) / 64)).cuda()
    held = [torch.zeros(0, H, D, dtype=BF16, device="cuda") for _ in range(4)]  # K, K, V, V
    for step, new in enumerate(([100, 7], [1, 1], [0, 60], [1, 1])):
        n = sum(new)
        q, k, v = (_randn(_gen(step), n, h, D, dtype=BF16) for h in (heads, H, H))
        at = torch.cat([torch.arange(m, m + c) for m, c in zip(cache.lengths, new)])
        turned = torch.empty_like(q)
        cache.append(k, v, new, inv_freq=f, q=q, q_out=turned)
        ref, bound = more.rotate(q, at, f, False)
        assert ((turned.double().cpu() - ref).abs() <= bound).all()
        o = torch.full_like(q, float("nan"))
        cache.attend(turned, o)
        ks, vs = [], []
        for b in range(2):
            pair = [torch.empty(cache.lengths[b], H, D, device="cuda") for _ in range(2)]
            cache.read(b, *pair)
            ks.append(pair[0])
            vs.append(pair[1])
        ref, mag = seq_ref.attention(turned, ks, vs, new)
        smax = float(turned.double().norm(dim=-1).max() * max(k.double().norm(dim=-1).max() for k in ks)) * D ** -0.5
        _check(o, ref, mag, BF16, smax, True, 200, more.weight_floor(turned, ks, vs, new))
        # what was appended is there, a code's step off at most
        for b, x in enumerate(_split(v, new)):
            held[2 + b] = torch.cat([held[2 + b], x])
            step_size = held[2 + b].float().abs().amax(-1, keepdim=True) / 7
            assert ((vs[b] - held[2 + b].float()).abs() <= step_size * 0.51).all()


def test_captured_attend_is_replayed_after_later_appends(cuda):
    """A generation step of the cache object through one graph, as the context grows over pages."""
    H, heads, D = 2, 4, 64
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=20, page_size=16, dtype=torch.uint8)
    k, v = (_randn(_gen(i), 90, H, D, dtype=BF16) for i in (1, 2))
    cache.append(k, v, [60, 30])
    q, graph = torch.empty(2, heads, D, dtype=BF16, device="cuda"), None
    o = torch.empty_like(q)
    for step in range(40):
        kn, vn = (_randn(_gen(100 * step + i), 2, H, D, dtype=BF16) for i in (3, 4))
        cache.append(kn, vn, [1, 1])
        q.copy_(_randn(_gen(step), 2, heads, D, dtype=BF16))
        if graph is None:
            cache.attend(q, o)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                cache.attend(q, o)
        o.fill_(float("nan"))
        graph.replay()
        want = torch.full_like(o, float("nan"))
        cache.attend(q, want)
        assert torch.equal(o, want)
    ks, vs = [], []
    for b in range(2):
        pair = [torch.empty(cache.lengths[b], H, D, device="cuda") for _ in range(2)]
        cache.read(b, *pair)
        ks.append(pair[0])
        vs.append(pair[1])
    ref, mag = seq_ref.attention(q, ks, vs, [1, 1])
    smax = float(q.double().norm(dim=-1).max() * max(x.double().norm(dim=-1).max() for x in ks)) * D ** -0.5
    _check(o, ref, mag, BF16, smax, True, 100, more.weight_floor(q, ks, vs, [1, 1]))


def test_long_pool_offsets_pass_32_bits(cuda):
    """The pages that are used lie more than 2^31 bytes of codes into the pool."""
    H, page, D, n = 8, 128, 128, 300
    num = 2 ** 31 // (H * page * D // 2) + 20
    pools = [torch.empty(num, H, page, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    kw = {x + "_scale": torch.zeros(num, H, page, device="cuda") for x in "kv"}
    kw |= {x + "_group": torch.zeros(num, H, page, 4, dtype=torch.uint8, device="cuda") for x in "kv"}
    table = torch.arange(num - 1, num - 4, -1, dtype=torch.int32, device="cuda")[None]
    where = seq_ref.starts([n]), table, torch.tensor([n], dtype=torch.int32, device="cuda")
    k, v = (_randn(_gen(i), n, H, D, dtype=BF16) for i in (1, 2))
    capi.kv_pages_append_dev(k, v, *pools, *where, **kw)
    back = [torch.empty_like(k, dtype=F32), torch.empty_like(v, dtype=F32)]
    capi.kv_pages_read_dev(*pools, *back, *where, **kw)
    for x, y in zip((k, v), back):
        assert ((x.float() - y).abs() <= x.float().abs().amax(-1, keepdim=True) / 7 * 0.51).all()
    for new in (1, 100):
        q = _randn(_gen(3), new, 16, D, dtype=BF16)
        o = torch.empty_like(q)
        w = seq_ref.starts([new]), *where[1:]
        capi.attn_paged_dev(q, *pools, o, *w, new, **kw)
        ref, mag = seq_ref.attention(q, [back[0]], [back[1]], [new])
        smax = float(q.double().norm(dim=-1).max() * back[0].double().norm(dim=-1).max()) * D ** -0.5
        _check(o, ref, mag, BF16, smax, True, n, more.weight_floor(q, [back[0]], [back[1]], [new]))
    bounds = torch.zeros(num, H, 2, D, dtype=BF16, device="cuda")
    capi.kv_blocks_bounds_dev(pools[0], bounds, *where, kw["k_scale"], kw["k_group"])
    want = torch.stack([back[0][:128].amin(0), back[0][:128].amax(0)], 1).to(BF16)
    assert torch.equal(bounds[num - 1], want)


def test_two_streams_at_once(cuda):
    """Two calls over one cache in flight together have workspaces of their own."""
    keys = [5000]
    p = _filled(keys, 2, 128, 64, BF16)
    qs = [_randn(_gen(i), 1, 8, 128, dtype=BF16) for i in range(6)]
    want = [_attend(p, q, [1], 1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [torch.empty_like(q) for q in qs]
    for _ in range(20):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                capi.attn_paged_dev(q, p.k, p.v, got[i], *p.where([1]), 1, **p.kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_off_their_alignment(cuda, dtype):
    """Rows one element off and with gaps give the same codes, and are read back the same."""
    keys, H, D = [70, 3], 2, 96
    n = sum(keys)
    x = _randn(_gen(1), n, 2 * H, D, dtype=dtype)
    got = []
    for shift in (0, 1):
        wide = torch.empty(n * (2 * H + 1) * D + 1, dtype=dtype, device="cuda")[shift: shift + n * (2 * H + 1) * D]
        rows = wide.view(n, 2 * H + 1, D)
        rows[:, : 2 * H] = x
        p = Pages(keys, H, D, 16, I4)
        capi.kv_pages_append_dev(rows[:, :H], rows[:, H:2 * H], p.k, p.v, *p.where(keys), **p.kw)
        back = torch.full_like(wide, 7).view(n, 2 * H + 1, D)
        capi.kv_pages_read_dev(p.k, p.v, back[:, :H], back[:, H:2 * H], *p.where(keys), **p.kw)
        assert (back[:, 2 * H] == 7).all()
        got.append(p.bits() + [back[:, : 2 * H].clone()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("new", [1, 40, 200])
def test_pages_off_16_bytes(cuda, new):
    """Pages and factors on 4-byte boundaries only: another kernel, the same attention."""
    keys = [400]
    p = _filled(keys, 2, 64, 16, BF16)
    q = _randn(_gen(3), new, 8, 64, dtype=BF16)

    def moved(t):
        return torch.empty(t.numel() + 4, dtype=t.dtype, device="cuda")[4:].view_as(t).copy_(t)

    p.k, p.v = moved(p.k), moved(p.v)
    p.kw = {name: moved(t) if t.dtype == torch.uint8 else t for name, t in p.kw.items()}
    _against(p, q, [new], keys, BF16, new)
    p.k = torch.empty(p.k.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(p.k)
    with pytest.raises(capi.AttnbError, match="4-byte boundaries"):
        _attend(p, q, [new], new)
