"""64-bit forms of the rotation, the 4-bit cache and the selection of blocks."""
from __future__ import annotations

import torch

from seq_ref import HALF


def rotate(x, position, inv_freq, interleaved):
    """x [tokens, heads, D] at `position` [tokens], in 64 bits, and a bound on the kernels' error
    before their rounding to x's type: the fraction of a turn is rounded to fp32 (at most half a turn, so
    pi 2^-24 of angle), sine and cosine have an error of up to 2 * 2^-23 of their own, the products and
    their sum three roundings: under 16 * 2^-24 of |x| + |y|; then the rounding to the type."""
    dtype = x.dtype
    x = x.double().cpu()
    n = len(inv_freq)
    a = position.double().cpu()[:, None, None] * inv_freq.double().cpu()
    i = torch.arange(n)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    out, size = x.clone(), torch.zeros_like(x)
    out[..., p] = x[..., p] * a.cos() - x[..., q] * a.sin()
    out[..., q] = x[..., q] * a.cos() + x[..., p] * a.sin()
    size[..., p] = size[..., q] = x[..., p].abs() + x[..., q].abs()
    half = HALF[dtype] * out.abs() * 1.001
    half[..., 2 * n:] = 0  # these stay
    if dtype == torch.float16:
        half = half + 2.0 ** -25
    return out, size * 16 * 2.0 ** -24 + half + 1e-40


def quantise4(x):
    """Codes (-7 to 7), factors and scale of x [..., D], D a multiple of 32."""
    x = x.double().cpu()
    top = x.abs().amax(-1, keepdim=True)
    some = torch.where(top > 0, top, 1.0)
    each = x.abs().unflatten(-1, (-1, 32)).amax(-1)
    factor = torch.ceil(255.0 * each / some)  # exact where it is whole: 53 bits hold 255 * each
    spread = torch.where(factor > 0, factor, 1.0).repeat_interleave(32, -1)
    codes = torch.round(x * 1785.0 / (some * spread))
    return codes, factor, top.squeeze(-1).float() / 1785.0


def values4(pages, scale, group):
    """What 4-bit pages hold, in 64 bits."""
    pages, group = pages.cpu(), group.cpu()
    codes = torch.stack([pages & 15, pages >> 4], -1).flatten(-2).double() - 8
    factor = group[..., : codes.shape[-1] // 32].double().repeat_interleave(32, -1)
    return codes * factor * scale.double().cpu()[..., None]


def scores(q, low, high):
    """q [G, D], low and high [blocks, D]: the blocks' scores."""
    q, low, high = q.double().cpu(), low.double().cpu(), high.double().cpu()
    return q.clamp(max=0).sum(0) @ low.T + q.clamp(min=0).sum(0) @ high.T


def select(score, take, first, last):
    """Block numbers that a token in the last block takes; score [blocks]."""
    n = len(score)
    if n <= take:
        return list(range(n))
    inner = torch.sort(score[first:n - last], descending=True, stable=True)[1] + first
    return sorted(list(range(first)) + inner[: take - first - last].tolist() + list(range(n - last, n)))


def weight_floor(q, ks, vs, new, causal=True, scale=None):
    """What subnormal weights add to attention_bound, [tokens, heads, 1].  Over codes the kernels round
    a weight to f16 relative to 2^rho <= max_j p_j scale_j, which is absolute below 2^-14: by at most 2^-25.  The
    codes (times their factors) are at most max |v_j| / scale_j, so that L keys are off by at most
    2^-25 L max_j p_j max |v_j|."""
    heads, D = q.shape[1:]
    out = torch.zeros(q.shape[0], heads, 1, dtype=torch.float64)
    first = 0
    for n, k, v in zip(new, ks, vs):
        L, H = k.shape[:2]
        if n and L:
            qq = q[first:first + n].double().cpu().permute(1, 0, 2)
            kk, vv = (x.double().cpu().permute(1, 2, 0).repeat_interleave(heads // H, 0) for x in (k, v))
            s = (qq @ kk) * (D ** -0.5 if scale is None else scale)
            if causal:
                s = s.masked_fill(~torch.ones(n, L, dtype=torch.bool).tril(L - n), -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[first:first + n, :, 0] = (p * vv.abs().amax(1)[:, None]).amax(-1).T * (2.0 ** -25 * L)
        first += n
    return out
