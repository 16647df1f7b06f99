"""Attention to selected blocks: bounds, the choice to the last index, attention over lists against
64-bit forms, lists of the caller's own, ties, NaN, strides, streams and graphs."""
from __future__ import annotations

import pytest
import torch

import seq_ref
import seq_ref_more as more
from attn_cpu import capi
from test_gpu_i4_cache import _held
from test_gpu_rope_append import I4, Pages
from test_gpu_seq_ops import BF16, E4M3, F16, F32, I8, _check, _gen, _randn

pytestmark = pytest.mark.gpu


def _values(p, name, b, n):
    if p.kind == I4:
        return _held(p, name, b, n)
    at = p.table[b, : -(-n // p.page)].long()
    x = getattr(p, name)[at].double()
    if p.kw:
        x = x * p.kw[name + "_scale"][at].double()[..., None]
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:n].cpu()


def _keys(p):
    return {x: p.kw[x] for x in ("k_scale", "k_group") if x in p.kw}


def _filled(keys, H, D, page, dtype, kind, seed=1):
    p = Pages(keys, H, D, page, kind, seed)
    g = _gen(seed)
    n = sum(keys)
    k, v = (_randn(g, n, H, D, dtype=F32) for _ in range(2))
    k += _randn(g, -(-n // page), H, D).repeat_interleave(page, 0)[:n]
    capi.kv_pages_append_dev(k.to(dtype), v.to(dtype), p.k, p.v, *p.where(keys), **p.kw)
    p.bounds = torch.full((p.k.shape[0], H, 2, D), 7.0, dtype=dtype, device="cuda")
    return p


def _bound(p, new):
    capi.kv_blocks_bounds_dev(p.k, p.bounds, *p.where(new), **_keys(p))


CASES = [  # types, H, D, page
    (F32, F32, 2, 80, 16), (BF16, BF16, 3, 128, 64), (F16, F16, 1, 33, 32), (BF16, E4M3, 2, 64, 128), (F16, I8, 2, 256, 16),
    (BF16, I4, 2, 128, 32), (F32, I4, 1, 64, 16), (F32, E4M3, 2, 128, 64), (BF16, I4, 1, 256, 16),
]


@pytest.mark.parametrize("dtype,kind,H,D,page", CASES)
def test_bounds(cuda, dtype, kind, H, D, page):
    keys = [5 * page + 3, page - 1, 3 * page, 0, 7 * page + 1]
    p = _filled(keys, H, D, page, dtype, kind)
    new = [2 * page + 4, page - 1, 1, 0, 1]  # from token 3 page - 1 on: complete blocks 2 to 4; none; block 2; none; none
    _bound(p, new)
    made = {(0, 2), (0, 3), (0, 4), (2, 2)}
    for b, n in enumerate(keys):
        x = _values(p, "k", b, n)
        for j in range(n // page):
            got = p.bounds[p.table[b, j]]
            if (b, j) in made:
                y = x[j * page:(j + 1) * page].float()  # one product in fp32
                want = torch.stack([y.amin(0), y.amax(0)], 1).to(dtype)
                assert torch.equal(got.cpu(), want), (b, j)
            else:
                assert (got == 7).all()
    capi.stream_status()
    _bound(p, keys)
    _bound(p, keys)
    for b, n in enumerate(keys):
        x = _values(p, "k", b, n).float()
        for j in range(n // page):
            y = x[j * page:(j + 1) * page]
            assert torch.equal(p.bounds[p.table[b, j]].cpu(), torch.stack([y.amin(0), y.amax(0)], 1).to(dtype))


def test_bounds_of_many_sequences(cuda):
    """More sequences than a CTA has threads."""
    keys = [16 + (i % 40) for i in range(700)]
    p = _filled(keys, 2, 64, 16, BF16, BF16)
    _bound(p, [1] * 700)
    done = [b for b, n in enumerate(keys) if n % 16 == 0]
    assert len(done) > 50
    for b in range(700):
        last = p.table[b, keys[b] // 16 - 1]
        if keys[b] % 16 == 0:
            x = p.k[last]
            assert torch.equal(p.bounds[last], torch.stack([x.amin(1), x.amax(1)], 1))
        else:
            assert (p.bounds[last] == 7).all()


def test_bounds_keep_nan(cuda):
    p = Pages([32], 1, 64, 16, F32)
    k = _randn(_gen(1), 32, 1, 64)
    k[3, 0, 5], k[20, 0, 6], k[21, 0, 7] = float("nan"), float("inf"), -float("inf")
    capi.kv_pages_append_dev(k, k, p.k, p.v, *p.where([32]))
    p.bounds = torch.zeros(p.k.shape[0], 1, 2, 64, device="cuda")
    _bound(p, [32])
    a, b = (p.bounds[p.table[0, i], 0] for i in range(2))
    assert torch.isnan(a[:, 5]).all() and torch.isnan(a).sum() == 2
    assert b[1, 6] == float("inf") and b[0, 7] == -float("inf") and not torch.isnan(b).any()


def _select(p, q, new, take, first=1, last=1):
    blocks = torch.full((q.shape[0], p.H, take), 99, dtype=torch.int32, device="cuda")
    capi.kv_blocks_select_dev(q, p.bounds, blocks, *p.where(new), p.page, keep_first=first, keep_last=last)
    return blocks


def _wanted(p, q, new, keys, take, first, last):
    G = q.shape[1] // p.H
    want, t = torch.full((q.shape[0], p.H, take), -1, dtype=torch.int32), 0
    for b, (n, L) in enumerate(zip(new, keys)):
        for i in range(n):
            own = (L - n + i) // p.page
            for h in range(p.H):
                low, high = p.bounds[p.table[b, : own + 1].long(), h].unbind(1)
                chosen = more.select(more.scores(q[t, h * G:(h + 1) * G], low, high), take, first, last)
                want[t, h, : len(chosen)] = torch.tensor(chosen)
            t += 1
    return want


def _attended(p, q, blocks, new, keys, dtype, scale=None):
    o = torch.full_like(q, float("nan"))
    capi.attn_blocks_dev(q, p.k, p.v, o, blocks, *p.where(new), scale, **p.kw)
    G, D = q.shape[1] // p.H, q.shape[2]
    ref, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    floor = torch.zeros(*q.shape[:2], 1, dtype=torch.float64)
    ks, vs = ([_values(p, x, b, n) for b, n in enumerate(keys)] for x in ("k", "v"))
    t = 0
    for b, (n, L) in enumerate(zip(new, keys)):
        for i in range(n):
            pos = L - n + i
            for h in range(p.H):
                mine = [j for j in blocks[t, h].tolist() if j >= 0]
                at = [x for j in mine for x in range(j * p.page, (j + 1) * p.page) if x <= pos]
                one = q[t:t + 1, h * G:(h + 1) * G], [ks[b][at][:, h:h + 1]], [vs[b][at][:, h:h + 1]], [1]
                r, m = seq_ref.attention(*one, scale=scale)
                ref[t, h * G:(h + 1) * G], mag[t, h * G:(h + 1) * G] = r[0], m[0]
                if p.kind != dtype and dtype != F32:
                    floor[t, h * G:(h + 1) * G] = more.weight_floor(*one, scale=scale)[0]
            t += 1
    smax = float(q.double().norm(dim=-1).max().cpu() * max(k.norm(dim=-1).max() for k in ks if len(k))) * (D ** -0.5 if scale is None else scale)
    _check(o[:t], ref[:t], mag[:t], dtype, smax, p.kind != dtype, blocks.shape[2] * p.page, floor[:t])
    return o


@pytest.mark.parametrize("dtype,kind,H,D,page", CASES)
@pytest.mark.parametrize("G,take,first,last", [(1, 4, 1, 1), (4, 6, 0, 2), (5, 3, 2, 1), (2, 1, 0, 1)])
def test_select_and_attend(cuda, dtype, kind, H, D, page, G, take, first, last):
    new, keys = [1, 3, 0, 1, 20], [9 * page + 5, 3, 5 * page, 15 * page, 6 * page + 9]
    new[1] = 2
    p = _filled(keys, H, D, page, dtype, kind)
    _bound(p, keys)
    q = _randn(_gen(G), sum(new) + 2, H * G, D, dtype=dtype)
    blocks = _select(p, q, new, take, first, last)
    n = sum(new)
    assert torch.equal(blocks[:n].cpu(), _wanted(p, q[:n], new, keys, take, first, last))
    assert (blocks[n:] == 99).all()
    o = _attended(p, q, blocks, new, keys, dtype)
    assert torch.isnan(o[n:].float()).all()
    capi.stream_status()


@pytest.mark.parametrize("dtype,kind", [(BF16, BF16), (F16, I4), (F32, F32), (BF16, E4M3)])
@pytest.mark.parametrize("new", [1, 5])
def test_one_long_context(cuda, dtype, kind, new):
    """A list that is split over many CTAs."""
    keys, D = [40003], 128
    p = _filled(keys, 2, D, 32, dtype, kind)
    _bound(p, keys)
    q = _randn(_gen(3), new, 8, D, dtype=dtype)
    for take in (200, 37):
        blocks = _select(p, q, [new], take, 1, 2)
        assert torch.equal(blocks.cpu(), _wanted(p, q, [new], keys, take, 1, 2))
        _attended(p, q, blocks, [new], keys, dtype, 0.1)


@pytest.mark.parametrize("n", [300, 512, 513, 700, 5000])
def test_ties_go_to_the_lower_block(cuda, n):
    """Blocks of equal bounds, as many as each form of the selection takes, and all of them zero."""
    keys, page, D = [16 * n], 16, 64
    p = _filled(keys, 1, D, page, BF16, BF16)
    _bound(p, keys)
    q = _randn(_gen(2), 1, 2, D, dtype=BF16)
    at = p.table[0].long()
    p.bounds[at] = p.bounds[at[0]].clone()
    p.bounds[at[200]] += 1  # a better one, and a worse one
    p.bounds[at[3]] -= 1
    s = more.scores(q[0], *p.bounds[at[[0, 200, 3]], 0].unbind(1))
    better, worse = (s[1] > s[0]), (s[2] < s[0])
    blocks = _select(p, q, [1], 150, 1, 1)[0, 0].tolist()
    assert blocks == _wanted(p, q, [1], keys, 150, 1, 1)[0, 0].tolist()
    assert (200 in blocks) == bool(better) and (3 not in blocks) == bool(worse)
    p.bounds.zero_()
    assert _select(p, q, [1], 9, 2, 3)[0, 0].tolist() == [0, 1, 2, 3, 4, 5, n - 3, n - 2, n - 1]
    p.bounds[at[[50, 60]]] = float("nan")  # the greatest
    assert _select(p, q, [1], 9, 2, 3)[0, 0].tolist() == [0, 1, 2, 3, 50, 60, n - 3, n - 2, n - 1]


@pytest.mark.parametrize("n", [64, 700])
def test_scores_next_to_each_other(cuda, n):
    """Scores that differ in the last place of fp32 are told apart, next to one far off the others."""
    keys, page, D = [16 * n], 16, 64
    p = _filled(keys, 1, D, page, F32, F32)
    p.bounds.zero_()
    at = p.table[0].long()
    one = torch.full((n,), 1000.0, device="cuda")
    one[45] = -1e30
    one[20:40] = torch.nextafter(one[20:40], one[20:40] * 2)
    p.bounds[at, 0, :, 0] = one[:, None]
    p.bounds[at, 0, :, 1] = 16777216.0  # the same for all, far greater
    q = torch.zeros(1, 1, D, device="cuda")
    q[0, 0, :2] = 1
    assert _select(p, q, [1], 12, 1, 1)[0, 0].tolist() == [0] + list(range(20, 30)) + [n - 1]
    assert _select(p, q, [1], 50, 1, 1)[0, 0].tolist() == [j for j in range(50) if j != 45] + [n - 1]


def test_lists_of_the_callers_own(cuda):
    """Empty lists, lists that end early, own block or not; wrong entries end a list and are told."""
    keys, page, H, D = [200, 90], 16, 2, 64
    p = _filled(keys, H, D, page, BF16, BF16)
    q = _randn(_gen(5), 4, 4, D, dtype=BF16)
    new = [2, 2]  # own blocks 12, 12, 5, 5
    blocks = torch.tensor([[[0, 3, 12, -1], [-1, -1, -1, -1]], [[12, -1, -1, -1], [1, 2, 3, 4]],
                           [[5, -1, 7, 8], [0, 1, 2, 5]], [[4, 5, -1, -1], [2, -1, -1, -1]]], dtype=torch.int32, device="cuda")
    want = blocks.clone()
    want[2, 0] = torch.tensor([5, -1, -1, -1])  # nothing counts behind a -1
    o = _attended(p, q, want, new, keys, BF16)
    capi.stream_status()
    assert (o[0, 2:] == 0).all()
    got = torch.empty_like(q)
    capi.attn_blocks_dev(q, p.k, p.v, got, blocks, *p.where(new))
    assert torch.equal(got, o)
    capi.stream_status()
    for wrong in ([0, 3, 3, 4], [0, 3, 2, 4], [0, 3, 13, -1], [0, 3, 10 ** 9, -1], [0, 3, -2, 5]):
        blocks[0, 0] = torch.tensor(wrong, dtype=torch.int32)
        want[0, 0] = torch.tensor([0, 3, -1, -1])
        capi.attn_blocks_dev(q, p.k, p.v, got, blocks, *p.where(new))
        with pytest.raises(capi.AttnbError, match="out of range"):
            capi.stream_status()
        capi.attn_blocks_dev(q, p.k, p.v, o, want, *p.where(new))
        assert torch.equal(got, o)
        capi.stream_status()


def test_long_lists(cuda):
    """Lists longer than a warp, with their end next to a multiple of 32."""
    keys, page, D = [16 * 150], 16, 64
    p = _filled(keys, 1, D, page, F16, F16)
    q = _randn(_gen(5), 1, 2, D, dtype=F16)
    for n in (31, 32, 33, 64, 96, 100):
        blocks = torch.full((1, 1, 100), -1, dtype=torch.int32, device="cuda")
        blocks[0, 0, :n] = torch.arange(n, device="cuda") + 50
        _attended(p, q, blocks, [1], keys, F16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_is_not_selected_stays_out(cuda, dtype):
    """NaN and infinities in other blocks, and behind a token's own position."""
    keys, page, H, D = [320], 16, 1, 64
    p = _filled(keys, H, D, page, dtype, dtype)
    q = _randn(_gen(6), 3, 4, D, dtype=dtype)
    blocks = torch.tensor([[[1, 7, 19]]] * 3, dtype=torch.int32, device="cuda")
    want = _attended(p, q, blocks, [3], keys, dtype)
    for j in range(20):
        if j not in (1, 7, 19):
            p.k[p.table[0, j]], p.v[p.table[0, j]] = float("nan"), float("inf")
    p.v[p.table[0, 19], :, 14:] = float("nan")  # seen by the second and the third alone
    got = torch.empty_like(q)
    capi.attn_blocks_dev(q, p.k, p.v, got, blocks, *p.where([3]))
    assert torch.equal(got[0], want[0]) and torch.isnan(got[1:].float()).all()


def test_strides_and_alignment(cuda):
    """Queries as slices off their alignment, an output with gaps, bounds off theirs."""
    new, keys, H, D = [3, 1], [500, 300], 2, 128
    p = _filled(keys, H, D, 16, BF16, BF16)
    _bound(p, keys)
    n = 4
    q = _randn(_gen(7), n, 8, D, dtype=BF16)
    want = _select(p, q, new, 8)
    o = _attended(p, q, want, new, keys, BF16)
    odd = torch.empty(n * 10 * D + 1, dtype=BF16, device="cuda")[1:].view(n, 10, D)
    odd[:, :8] = q
    flat = torch.empty(p.bounds.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(p.bounds).copy_(p.bounds)
    blocks = torch.empty_like(want)
    capi.kv_blocks_select_dev(odd[:, :8], flat, blocks, *p.where(new), 16)
    assert torch.equal(blocks, want)
    out = torch.full((8, n, 2 * D), 7.0, dtype=BF16, device="cuda")
    capi.attn_blocks_dev(odd[:, :8], p.k, p.v, out[:, :, :D].transpose(0, 1), blocks, *p.where(new))
    assert (out[:, :, D:] == 7).all()
    # (another kernel than for aligned rows: weights are not rounded there)
    assert ((out[:, :, :D].transpose(0, 1).float() - o.float()).abs() <= 2.0 ** -6 * o.float().abs() + 2.0 ** -7).all()


def test_bad_pages_and_lengths(cuda):
    keys, page = [320, 200], 16
    p = _filled(keys, 1, 64, page, BF16, BF16)
    _bound(p, keys)
    capi.stream_status()
    q = _randn(_gen(8), 2, 2, 64, dtype=BF16)
    good = _select(p, q, [1, 1], 6)
    p.table[0, 5] = 10 ** 6
    blocks = _select(p, q, [1, 1], 6)
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()
    assert torch.equal(blocks[1], good[1])
    _bound(p, [320, 0])
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()
    lens = torch.tensor([10 ** 9, -4], dtype=torch.int32, device="cuda")
    cu = seq_ref.starts([1, 1])
    capi.kv_blocks_select_dev(q, p.bounds, blocks, cu, p.table, lens, page)
    assert (blocks[1] == -1).all()
    o = torch.full_like(q, float("nan"))
    capi.attn_blocks_dev(q, p.k, p.v, o, blocks, cu, p.table, lens)
    assert (o[1] == 0).all()
    before = p.bounds.clone()
    capi.kv_blocks_bounds_dev(p.k, p.bounds, seq_ref.starts([0, 3]), p.table, lens)
    assert torch.equal(before, p.bounds)
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()


def test_captured_and_replayed(cuda):
    """A step of a growing context through one graph: append, bounds, choice, attention."""
    H, heads, D, page, take = 2, 8, 64, 16, 4
    p = _filled([120], H, D, page, BF16, BF16)
    table = torch.arange(p.table.shape[1] + 3, dtype=torch.int32, device="cuda")[None] % p.k.shape[0]
    p.table[0] = table[0, : p.table.shape[1]]
    p.table = table[:, : p.k.shape[0]]
    p.lens = torch.tensor([120], dtype=torch.int32, device="cuda")
    k = _randn(_gen(11), 120, H, D, dtype=BF16)
    capi.kv_pages_append_dev(k, k, p.k, p.v, *p.where([120]))
    _bound(p, [120])
    q, kn, vn = (_randn(_gen(12), 1, h, D, dtype=BF16) for h in (heads, H, H))
    o, blocks = torch.empty_like(q), torch.empty(1, H, take, dtype=torch.int32, device="cuda")
    where = p.where([1])

    def step():
        capi.kv_pages_append_dev(kn, vn, p.k, p.v, *where)
        capi.kv_blocks_bounds_dev(p.k, p.bounds, *where)
        capi.kv_blocks_select_dev(q, p.bounds, blocks, *where, page)
        capi.attn_blocks_dev(q, p.k, p.v, o, blocks, *where)

    p.lens.fill_(121)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(122, 150):
        p.lens.fill_(n)
        for t in (q, kn, vn):
            t.copy_(_randn(_gen(n + t.shape[1]), *t.shape, dtype=BF16))
        graph.replay()
        assert torch.equal(blocks.cpu(), _wanted(p, q, [1], [n], take, 1, 1))
    got = o.clone()
    assert torch.equal(got, _attended(p, q, blocks, [1], [149], BF16))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    again = torch.empty_like(o)
    capi.attn_blocks_dev(q, p.k, p.v, again, blocks, *where, stream=stream)
    stream.synchronize()
    assert torch.equal(again, got)


def test_cache_object(cuda):
    """The paged cache object over selected blocks, as a user's program runs it."""
    H, heads, D, page = 2, 8, 64, 16
    cache = capi.PagedKVCacheDev(2, H, D, num_pages=80, page_size=page, dtype=BF16, bounds=True)
    f = (10000.0 ** (-torch.arange(32) / 32)).cuda()
    for step, new in enumerate(([300, 70], [1, 1], [0, 25], [1, 1])):
        q, k, v = (_randn(_gen(step), sum(new), h, D, dtype=BF16) for h in (heads, H, H))
        turned, o, full = (torch.empty_like(q) for _ in range(3))
        cache.append(k, v, new, inv_freq=f, q=q, q_out=turned)
        blocks = cache.attend_blocks(turned, o, take=6, keep_last=2)
        p = Pages([1], H, D, page, BF16)
        p.k, p.v, p.table, p.lens, p.bounds = cache.k_pages, cache.v_pages, cache.table, cache.lens, cache.bounds
        assert torch.equal(blocks.cpu(), _wanted(p, turned, new, cache.lengths, 6, 1, 2))
        assert torch.equal(_attended(p, turned, blocks, new, cache.lengths, BF16), o)
        # as many blocks as there are: the same as attending to all
        cache.attend_blocks(turned, o, take=40)
        cache.attend(turned, full)
        assert ((o.float() - full.float()).abs() <= 2.0 ** -6 * full.float().abs() + 2.0 ** -7).all()
    with pytest.raises(ValueError, match="bounds"):
        capi.PagedKVCacheDev(1, H, D, num_pages=2, dtype=BF16).attend_blocks(q, o, take=4)


@pytest.mark.parametrize("dtype,kind,D,page,n,H,new", [
    (BF16, BF16, 64, 16, 700, 2, 160),  # rows enough to fill the machine, more keys than a warp chooses from
    (F32, F32, 256, 16, 1300, 1, 300),
    (F16, I4, 128, 32, 600, 8, 40),
])
def test_many_rows_of_many_blocks(cuda, dtype, kind, D, page, n, H, new):
    keys = [page * n - 3]
    p = _filled(keys, H, D, page, dtype, kind)
    _bound(p, keys)
    q = _randn(_gen(3), new, 2 * H, D, dtype=dtype)
    for take in (30, 590):
        blocks = _select(p, q, [new], take, 2, 1)
        assert torch.equal(blocks.cpu(), _wanted(p, q, [new], keys, take, 2, 1))


@pytest.mark.parametrize("batch", [65, 300, 700])
def test_many_sequences(cuda, batch):
    """More sequences than lanes of a warp and threads of a CTA, some without a token."""
    keys = [20 + 37 * i % 300 for i in range(batch)]
    new = [i % 3 for i in range(batch)]
    p = _filled(keys, 1, 64, 16, BF16, BF16)
    _bound(p, keys)
    q = _randn(_gen(4), sum(new), 2, 64, dtype=BF16)
    blocks = _select(p, q, new, 5)
    assert torch.equal(blocks.cpu(), _wanted(p, q, new, keys, 5, 1, 1))
    _attended(p, q, blocks, new, keys, BF16)
    capi.stream_status()


def test_rows_in_several_launches(cuda):
    """A table so wide that the scores of all rows would not fit the workspace: the call goes in parts.
    Its pages are a few that repeat, so that nearly all scores are equal to many others."""
    page, D, width, new, few, take = 16, 64, 200_000, 70, 50, 100
    p = Pages([page * few], 1, D, page, BF16)
    k = _randn(_gen(5), page * few, 1, D, dtype=BF16)
    capi.kv_pages_append_dev(k, k, p.k, p.v, *p.where([page * few]))
    p.bounds = torch.zeros(p.k.shape[0], 1, 2, D, dtype=BF16, device="cuda")
    _bound(p, [page * few])
    own = p.table[0, :few].clone()
    g = torch.Generator().manual_seed(6)
    slot = torch.randint(0, few, (width,), generator=g)
    p.table = own[slot.cuda()][None].contiguous()
    L = page * width - 5
    p.lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    q = _randn(_gen(7), new, 2, D, dtype=BF16)
    blocks = _select(p, q, [new], take, 1, 2).cpu()
    low, high = p.bounds[own.long(), 0].unbind(1)
    for i in (0, 1, 30, 39, 40, 41, 42, 43, 69):
        n = (L - new + i) // page + 1
        s = more.scores(q[i], low, high)[slot[:n]]
        assert blocks[i, 0].tolist() == more.select(s, take, 1, 2), i
    o = torch.empty_like(q)
    capi.attn_blocks_dev(q, p.k, p.v, o, blocks.cuda(), *p.where([new]))
    ks = k.view(few, page, 1, D)
    for i in (0, 69):
        at, pos = blocks[i, 0].long(), L - new + i
        x = ks[slot[at].cuda()].flatten(0, 1)
        x = x[: len(x) - (page - 1 - pos % page)]
        ref, mag = seq_ref.attention(q[i:i + 1], [x], [x], [1])
        _check(o[i:i + 1], ref, mag, BF16, float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) / 8, L=1600)
    capi.stream_status()


@pytest.mark.parametrize("dtype,kind,D", [(BF16, BF16, 80), (BF16, I4, 128), (F16, I4, 64), (F32, F32, 64), (F16, I8, 96)])
@pytest.mark.parametrize("G", [9, 20])
def test_many_query_heads(cuda, dtype, kind, D, G):
    """More query heads of a KV head than an item has rows."""
    new, keys, page = [2, 1, 3], [700, 40, 333], 16
    p = _filled(keys, 2, D, page, dtype, kind)
    _bound(p, keys)
    q = _randn(_gen(G), 6, 2 * G, D, dtype=dtype)
    blocks = _select(p, q, new, 7, 1, 2)
    assert torch.equal(blocks.cpu(), _wanted(p, q, new, keys, 7, 1, 2))
    _attended(p, q, blocks, new, keys, dtype)
