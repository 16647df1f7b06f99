"""64-bit forms of the operators over ragged sequences and paged KV caches, and the bounds that
the tests hold the kernels to."""
from __future__ import annotations

import numpy as np
import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
# Half a step of the type, relative to the value: one rounding.
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def attention(q, ks, vs, new, causal=True, scale=None):
    """q [tokens, heads, D] packed by `new`; ks, vs: per sequence [L, kv_heads, D].  Also returns,
    per element, sum_j p_j |v_j|: what the relative error of each weight is a share of."""
    heads, D = q.shape[1:]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    first = 0
    for n, k, v in zip(new, ks, vs):
        L, H = k.shape[:2]
        G = heads // H
        if n and L:
            qq = q[first:first + n].double().cpu().permute(1, 0, 2)
            kk = k.double().cpu().permute(1, 2, 0).repeat_interleave(G, 0)
            vv = v.double().cpu().permute(1, 0, 2).repeat_interleave(G, 0)
            s = (qq @ kk) * (D ** -0.5 if scale is None else scale)
            seen = torch.ones(n, L, dtype=torch.bool)
            if causal:
                seen = seen.tril(L - n)
            s = s.masked_fill(~seen, -np.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top > -np.inf, top, 0.0)), 0.0)
            p = p / torch.where(p.sum(-1, keepdim=True) > 0, p.sum(-1, keepdim=True), 1.0)
            vv = torch.where(seen.any(0)[None, :, None], vv, 0.0)
            out[first:first + n] = (p @ vv).permute(1, 0, 2)
            mag[first:first + n] = (p @ vv.abs()).permute(1, 0, 2)
        first += n
    return out, mag


def attention_bound(dtype, mag, out, smax, coded=False, D=128, L=1):
    """|error| per element.  smax bounds scale * sum |q k| (|q| |k| * scale).  The D roundings of a
    score, 2^-24 of smax each, add like sqrt(D), three times that for the largest of many: under
    40 * 2^-24 * smax for D <= 128 (another sqrt(2) at 256 is in the 16), which is the relative error
    of its weight; the sums over L keys and D add sqrt terms of their own.  16-bit kernels round each
    weight to the type (bf16 over 8-bit pages), half a step of sum p |v|, and the result once."""
    p = HALF[torch.float32] * (40 * smax + 4 * np.sqrt(D) + 2 * np.sqrt(L) + 16)
    if dtype != torch.float32:
        p += HALF[torch.bfloat16 if coded else dtype]
    return mag * p + out.abs() * 1.01 * HALF[dtype] + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0)


def quantise(x, dtype):
    """The values that the codes of x stand for, in 64 bits, and the scales."""
    x = x.double().cpu()
    if not x.numel():
        return x, x[..., 0].float()
    top = x.abs().amax(-1, keepdim=True)
    y = x * TOP[dtype] / torch.where(top > 0, top, 1.0)
    if dtype == torch.int8:
        codes = torch.round(y)
    else:
        e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        codes = torch.round(y / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
    scale = (top.float() / TOP[dtype]).squeeze(-1)
    return codes, scale


def random_pages(counts, page, num_pages, width, gen):
    """A table for sequences of `counts` tokens with pages in any order; unused entries are -1."""
    order = torch.randperm(num_pages, generator=gen).tolist()
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        for i in range(-(-n // page)):
            table[b, i] = order.pop()
    return table


def starts(counts, device="cuda"):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=device)
