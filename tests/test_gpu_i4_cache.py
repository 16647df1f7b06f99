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
