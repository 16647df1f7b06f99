"""4-bit pages at the small end: queries down to the type's least values, groups that are tiny beside
the rest of their vector."""
from __future__ import annotations

import pytest
import torch

import seq_ref_more as more
from attn_cpu import capi
from test_gpu_i4_cache import I4, _against, _filled, _places
from test_gpu_rope_append import Pages
from test_gpu_seq_ops import BF16, F16, F32, _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 5, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("by,keys_by", [(-112, 0), (-115, 0), (-120, 0), (-126, 0), (-130, 0), (-115, 112), (-126, 119), (-128, 119)])
def test_queries_down_to_the_least(cuda, new, D, by, keys_by):
    """Scores next to zero, and ordinary ones where the keys are as large as the queries are small."""
    keys, H = [500], 1
    g = _gen(9)
    p = Pages(keys, H, D, 64, I4)
    k, v = (_randn(g, 500, H, D) for _ in range(2))
    capi.kv_pages_append_dev((k * 2.0 ** keys_by).to(BF16), v.to(BF16), p.k, p.v, *p.where(keys), **p.kw)
    q = (_randn(g, new, 4, D) * 2.0 ** by).to(BF16)
    q[0, 0] = 0
    q[0, 1, 1:] = 0  # zeros next to one value
    _against(p, q, [new], keys, BF16, new)


def test_rows_of_all_sizes_at_once(cuda):
    """Each row is brought to its own size: tiny ones, ordinary ones and zeros in one item."""
    keys, D = [300, 70], 128
    p = _filled(keys, 2, D, 32, BF16)
    for new in (1, 40):
        q = _randn(_gen(3), 2 * new, 8, D)
        q *= 2.0 ** torch.tensor([0, -126, -113, -114, -119, -50, -130, 3], device="cuda", dtype=F32)[:, None]
        q[:, 5] = 0
        _against(p, q.to(BF16), [new, new], keys, BF16, new)


@pytest.mark.parametrize("dtype,top,least", [(BF16, 120, -130), (BF16, 61, -90), (F32, 127, -140), (F32, 100, -87), (F32, 60, -140),
                                             (BF16, -70, -133), (F16, 15, -24)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_codes_of_tiny_groups(cuda, dtype, top, least, D):
    """A group next to zero beside one next to the type's largest value: factor 1 and codes 8, as the exact
    quotients give."""
    n, H = 200, 2
    p = Pages([n], H, D, 32, I4)
    for t in (p.k, p.v, *p.kw.values()):  # whatever was there before
        t.view(torch.uint8).fill_(0xA5)
    k, v = (_randn(_gen(D + i), n, H, D) for i in range(2))
    for x in (k, v):
        small = 2.0 ** torch.linspace(least, top, n, device="cuda", dtype=torch.float64)
        x /= x.abs().amax(-1, keepdim=True)
        x[..., :32] = (x[..., :32].double() * small[:, None, None]).to(F32)
        x[..., 32:] = (x[..., 32:].double() * 2.0 ** top).to(F32)
    k[:7, 0, 5] = 2.0 ** least
    k, v = k.to(dtype), v.to(dtype)
    capi.kv_pages_append_dev(k, v, p.k, p.v, *p.where([n]), **p.kw)
    at, slot = _places(p, [n], [n])
    for x, name in ((k, "k"), (v, "v")):
        assert torch.isfinite(x).all()
        codes, factor, scale = more.quantise4(x)
        pages = getattr(p, name)[at, :, slot].cpu()
        got = torch.stack([pages & 15, pages >> 4], -1).flatten(-2).double() - 8
        assert torch.equal(p.kw[name + "_scale"][at, :, slot].cpu(), scale)
        assert torch.equal(p.kw[name + "_group"][at, :, slot].cpu().double()[..., : D // 32], factor)
        assert torch.equal(got, codes)
