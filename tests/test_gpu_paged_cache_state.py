"""The paged cache object's state: refused appends, streams other than the constructor's, captured
attention that is replayed after later appends."""
from __future__ import annotations

import pytest
import torch

import seq_ref
from attn_cpu import capi
from test_gpu_seq_ops import BF16, E4M3, _gen, _randn, _smax

pytestmark = pytest.mark.gpu

H, HEADS, D = 2, 4, 64


def _rows(seed, n):
    g = _gen(seed)
    return tuple(_randn(g, n, h, D, dtype=BF16) for h in (HEADS, H, H))


def _attended(cache, q, ks, vs, new):
    o = torch.full_like(q, float("nan"))
    cache.attend(q, o)
    ref, mag = seq_ref.attention(q, ks, vs, new)
    bound = seq_ref.attention_bound(BF16, mag, ref, _smax(q, torch.cat(ks)), False, D, 400)
    assert ((o.double().cpu() - ref).abs() <= bound).all()


def test_refused_append_keeps_the_tokens_appended_last(cuda):
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=12, page_size=16, dtype=BF16)
    q, k, v = _rows(1, 70)
    cache.append(k, v, [50, 20])
    wrong = torch.zeros(90, H + 1, D, dtype=BF16, device="cuda")
    with pytest.raises(capi.AttnbError, match="matching the pages"):
        cache.append(wrong, wrong, [60, 30])
    assert cache.lengths == [50, 20]
    _attended(cache, q, [k[:50], k[50:]], [v[:50], v[50:]], [50, 20])
    q2, k2, v2 = _rows(2, 3)
    cache.append(k2, v2, [1, 2])
    _attended(cache, q2, [torch.cat([k[:50], k2[:1]]), torch.cat([k[50:], k2[1:]])],
              [torch.cat([v[:50], v2[:1]]), torch.cat([v[50:], v2[1:]])], [1, 2])


def test_captured_attend_is_replayed_after_later_appends(cuda):
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=40, page_size=16, dtype=BF16)
    q, k, v = _rows(3, 90)
    cache.append(k, v, [60, 30])
    ks, vs = [k[:60], k[60:]], [v[:60], v[60:]]
    q, o, graph = torch.empty(2, HEADS, D, dtype=BF16, device="cuda"), None, None
    for step in range(40):
        qn, kn, vn = _rows(100 + step, 2)
        cache.append(kn, vn, [1, 1])
        ks = [torch.cat([x, kn[i:i + 1]]) for i, x in enumerate(ks)]
        vs = [torch.cat([x, vn[i:i + 1]]) for i, x in enumerate(vs)]
        q.copy_(qn)
        if graph is None:
            o = torch.full_like(q, float("nan"))
            _attended(cache, q, ks, vs, [1, 1])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                cache.attend(q, o)
        o.fill_(float("nan"))
        graph.replay()
        if step % 10 == 9:
            ref, mag = seq_ref.attention(q, ks, vs, [1, 1])
            bound = seq_ref.attention_bound(BF16, mag, ref, _smax(q, torch.cat(ks)), False, D, 400)
            assert ((o.double().cpu() - ref).abs() <= bound).all()
