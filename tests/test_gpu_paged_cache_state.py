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


def test_first_append_on_another_stream(cuda):
    """The constructor's own work is done before any stream may use the cache, also when the
    constructor's stream is busy."""
    q, k, v = _rows(4, 70)
    stream = torch.cuda.Stream()
    for _ in range(3):
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda._sleep(20_000_000)  # about 10 ms
        cache = capi.PagedKVCacheDev(2, H, D, num_pages=12, page_size=16, dtype=E4M3)
        cache.append(k, v, [50, 20], stream=stream)
        torch.cuda.synchronize()
        assert cache.lens.tolist() == [50, 20] and cache.cu.tolist() == [0, 50, 70]
        assert sorted(cache.table[0, :4].tolist() + cache.table[1, :2].tolist()) == list(range(6))


def test_memory_stays_while_another_stream_works_on_it(cuda):
    """The cache goes while its last attend is still waiting on another stream: its memory is not
    given to others meanwhile."""
    q, k, v = _rows(5, 70)
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=12, page_size=16, dtype=BF16)
    cache.append(k, v, [50, 20])
    want, o = torch.empty_like(q), torch.empty_like(q)
    cache.attend(q, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)
        o.record_stream(stream)
        q.record_stream(stream)
        cache.attend(q, o)
    places = {t.data_ptr() for t in (cache.k_pages, cache.v_pages, cache.table, cache.lens, cache.cu)}
    shape = cache.k_pages.shape
    del cache
    other = [torch.full(shape, float("nan"), dtype=BF16, device="cuda") for _ in range(4)]
    other += [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (2, 3, 24) for _ in range(4)]
    assert not places & {t.data_ptr() for t in other}
    torch.cuda.synchronize()
    assert torch.equal(o, want)


def test_refused_append_on_a_busy_stream(cuda):
    """The lengths that come back are behind those that were sent."""
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=12, page_size=16, dtype=BF16)
    q, k, v = _rows(6, 70)
    cache.append(k, v, [50, 20])
    wrong = torch.zeros(90, H + 1, D, dtype=BF16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
    with pytest.raises(capi.AttnbError, match="matching the pages"):
        cache.append(wrong, wrong, [60, 30], stream=stream)
    torch.cuda.synchronize()
    assert cache.lens.tolist() == [50, 20] and cache.cu.tolist() == [0, 50, 70]
    _attended(cache, q, [k[:50], k[50:]], [v[:50], v[50:]], [50, 20])
