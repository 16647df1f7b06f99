"""Scores of blocks whose bounds or queries are not finite, against their definition: the sum over query heads
and dimensions of max(q least, q greatest)."""
from __future__ import annotations

import pytest
import torch

import seq_ref_more as more
from attn_cpu import capi
from test_gpu_blocks import _bound, _filled, _select
from test_gpu_rope_append import Pages
from test_gpu_seq_ops import BF16, E4M3, F16, F32, _gen, _randn

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _scores(q, low, high):
    """q [G, D], low, high [blocks, D], as defined; a NaN of either product is the maximum."""
    q, low, high = q.double().cpu(), low.double().cpu(), high.double().cpu()
    return torch.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2))


def _check(p, q, new, keys, take, first=1, last=1):
    blocks = _select(p, q, [new], take, first, last).cpu()
    G, kinds = q.shape[1] // p.H, set()
    for t in range(0, new, 47):
        own = (keys - new + t) // p.page
        for h in range(p.H):
            low, high = p.bounds[p.table[0, : own + 1].long(), h].unbind(1)
            s = _scores(q[t, h * G:(h + 1) * G], low, high)
            s[max(0, own + 1 - last):] = 0.0  # these have no bounds yet
            assert blocks[t, h].tolist() == more.select(s, take, first, last), (t, h)
            kinds |= {("nan" if x != x else "finite" if abs(x) < INF else str(x)) for x in s.tolist()}
    return kinds


# A row alone of up to 512 blocks, of more, and rows that fill the machine; head sizes off 16 bytes too.
@pytest.mark.parametrize("n,new", [(60, 1), (700, 1), (560, 330)])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 33), (BF16, 128), (F16, 80), (F16, 33), (F32, 256)])
def test_infinite_keys(cuda, n, new, dtype, D):
    """Keys of +inf and -inf in single dimensions, under queries that are all positive there, all negative, of both
    signs, and zero."""
    keys, page, H, G = 16 * n - 3, 16, 2, 3
    p = _filled([keys], H, D, page, dtype, dtype)
    at = p.table[0].long()
    for j, (d, x) in enumerate([(1, -INF), (1, INF), (2, -INF), (2, INF), (3, -INF), (3, INF), (4, -INF), (4, INF), (5, INF), (6, NAN)]):
        p.k[at[2 * j + 3], :, 5, d] = x
    p.k[at[40], :, :, 1] = -INF  # all keys of a block
    p.k[at[41], :, :, 2] = INF
    p.k[at[42], :, 0, 1], p.k[at[42], :, 1, 1] = INF, -INF
    _bound(p, [keys])
    q = _randn(_gen(4), new, H * G, D, dtype=dtype)
    q[..., 1] = q[..., 1].abs() + 0.5
    q[..., 2] = -q[..., 2].abs() - 0.5
    q[..., 4] = 0
    q[..., 5] = q[..., 5].abs()
    q[:, 1::3, 5] = -0.0
    kinds = set()
    for take in (2, 4, 9, 25, 50):
        kinds |= _check(p, q, new, keys, take)
    assert kinds == {"finite", "inf", "-inf", "nan"}
    capi.stream_status()


@pytest.mark.parametrize("n", [60, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinite_queries(cuda, n, dtype):
    keys, D = 16 * n, 64
    p = _filled([keys], 1, D, 16, dtype, dtype)
    _bound(p, [keys])
    p.bounds[p.table[0, 7].long(), 0, :, 9] = torch.tensor([-1.0, 0.0], device="cuda")
    p.bounds[p.table[0, 8].long(), 0, :, 9] = torch.tensor([-2.0, -1.0], device="cuda")
    for x in (INF, -INF, NAN):
        q = _randn(_gen(4), 1, 4, D, dtype=dtype)
        q[0, 2, 9] = x
        for take in (4, 20):
            _check(p, q, 1, keys, take)


def test_f16_bounds_of_large_codes(cuda):
    """Codes stand for values past f16's largest: infinite bounds, and scores that are still what they are defined as."""
    n, page, D = 80, 16, 64
    p = Pages([page * n], 1, D, page, E4M3)
    k = _randn(_gen(1), page * n, 1, D)
    k[5 * page + 3, 0, 2], k[9 * page + 3, 0, 2], k[11 * page, 0, 2] = 1e6, -1e6, -1e6
    capi.kv_pages_append_dev(k.to(BF16), k.to(BF16), p.k, p.v, *p.where([page * n]), **p.kw)
    p.bounds = torch.zeros(p.k.shape[0], 1, 2, D, dtype=F16, device="cuda")
    _bound(p, [page * n])
    assert torch.isinf(p.bounds).any() and not torch.isnan(p.bounds).any()
    q = _randn(_gen(2), 1, 4, D, dtype=F16)
    for sign in (1, -1):
        q[..., 2] = sign * (q[..., 2].abs() + 0.1)
        for take in (3, 8, 30):
            assert _check(p, q, 1, page * n, take) == {"finite", "inf"}
