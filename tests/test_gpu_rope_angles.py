"""Angles of the rotated append next to half a turn, where sines are small and show what an angle is off by."""
from __future__ import annotations

import pytest
import torch

from attn_cpu import capi
from test_gpu_rope_append import Pages
from test_gpu_seq_ops import E4M3, F32, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,pairs,interleaved,shift", [(128, 64, False, 0), (128, 64, True, 0), (128, 64, False, 1), (96, 20, True, 0),
                                                       (64, 17, False, 0), (64, 8, True, 1)])
@pytest.mark.parametrize("kind", [F32, E4M3])
def test_angles_next_to_half_a_turn(cuda, D, pairs, interleaved, shift, kind):
    """With a pair (1, 0) the results are cosine and sine.  Where a fraction of a turn is within 2^-8 of a half, the
    sine is s = 2 pi 2^-8 at most.  It is off by two units of its last place, 2^-22 s, and by roundings of a product and a sum
    and of the angle's small rest, under 2^-22 s in all.  The angle is a product of 64-bit numbers, three roundings of
    up to 2^-53 of 2^14 turns here, 2^-37 turns or 2^-34; so are the reference's.  (An angle of 32 bits is off by up to 2 pi 2^-26.)"""
    g = torch.Generator().manual_seed(pairs)
    n, H = 300, 2
    where = torch.arange(1, n + 1, dtype=torch.float64)
    # fractions of a turn of 1/2 + m / 2^k at some positions: odd multiples of about half a turn
    freq = (torch.pi * (2 * torch.randint(0, 50, (pairs,), generator=g) + 1 + (torch.rand(pairs, generator=g) - 0.5) / 2 ** 14)).float()
    p = Pages([n + 1], H, D, 16, kind)
    flat = torch.zeros(n * H * D + shift, device="cuda")
    k = flat[shift:].view(n, H, D)
    first = torch.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    k[..., first] = 1
    q = torch.zeros(n * H * D + shift, device="cuda")[shift:].view(n, H, D).copy_(k)
    out = torch.empty_like(q)
    capi.kv_pages_append_rope_dev(k, k, p.k, p.v, *p.where([n]), freq.cuda(), interleaved, q, out, **p.kw)
    angle = where[:, None] * freq.double()
    near = ((angle / (2 * torch.pi)) % 1 - 0.5).abs() < 2.0 ** -8
    assert near.sum() > 100
    sine = angle.sin()[:, None]
    got = [out] if kind == E4M3 else [out, p.k[p.table[0, where.long().cuda() // 16].long(), :, where.long().cuda() % 16]]
    for x in got:
        off = (x[..., second].double().cpu() - sine).abs()
        assert (off <= sine.abs() * 2.0 ** -21 + 2.0 ** -33)[near[:, None].expand_as(off)].all()
        assert (off <= 8 * 2.0 ** -24).all()
        assert ((x[..., first].double().cpu() - angle.cos()[:, None]).abs() <= 8 * 2.0 ** -24).all()
