"""Appending with the position rotation on the way: against 64-bit angles, against rotating first and
appending then, in every type, layout and alignment, at far positions, in place, on other streams and
replayed."""
from __future__ import annotations

import pytest
import torch

import seq_ref
import seq_ref_more as more
from attn_cpu import capi
from test_gpu_seq_ops import BF16, E4M3, F16, F32, I8, _gen, _randn

pytestmark = pytest.mark.gpu
I4 = torch.uint8


class Pages:
    """A pool for sequences that hold `keys` tokens, the pages in any order."""

    def __init__(self, keys, H, D, page, kind, seed=0, spare=5):
        g = torch.Generator().manual_seed(seed)
        num = sum(-(-k // page) for k in keys) + spare
        self.page, self.H, self.D, self.kind = page, H, D, kind
        self.table = seq_ref.random_pages(keys, page, num, max(1, max(-(-k // page) for k in keys)), g).cuda()
        self.lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
        self.kw = {}
        wide = D // 2 if kind == I4 else D
        self.k, self.v = (torch.zeros(num, H, page, wide, dtype=kind, device="cuda") for _ in range(2))
        if kind in (E4M3, I8, I4):
            for name in ("k_scale", "v_scale"):
                self.kw[name] = torch.zeros(num, H, page, device="cuda")
        if kind == I4:
            for name in ("k_group", "v_group"):
                self.kw[name] = torch.zeros(num, H, page, capi.i4_group_bytes(D), dtype=torch.uint8, device="cuda")

    def where(self, new):
        return seq_ref.starts(new), self.table, self.lens

    def bits(self):
        return [t.view(torch.uint8).clone() for t in (self.k, self.v, *self.kw.values())]


def _positions(new, keys):
    return torch.cat([torch.arange(k - n, k) for n, k in zip(new, keys)]) if new else torch.zeros(0)


def _freq(pairs, base=10000.0):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))).float().cuda()


CASES = [  # D, pairs, interleaved
    (64, 32, False), (128, 64, False), (128, 64, True), (128, 32, False), (128, 20, False), (80, 40, False),
    (80, 7, True), (33, 16, False), (33, 5, True), (256, 128, False), (256, 64, True), (2, 1, False), (96, 48, True),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D,pairs,interleaved", CASES)
def test_rotation(cuda, dtype, D, pairs, interleaved):
    new, keys = [3, 0, 1, 70, 40], [3, 5, 200, 1000, 40]
    p = Pages(keys, 2, D, 16, dtype)
    g = _gen(D + pairs)
    q, k, v = (_randn(g, sum(new) + 3, h, D, dtype=dtype) for h in (5, 2, 2))
    out = torch.full_like(q, 7.0)
    f = _freq(pairs)
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, interleaved, q, out)
    n = sum(new)
    position = _positions(new, keys)
    ref, bound = more.rotate(q[:n], position, f, interleaved)
    assert ((out[:n].double().cpu() - ref).abs() <= bound).all()
    assert (out[n:] == 7).all()
    back = [torch.full_like(k, 7.0), torch.full_like(v, 7.0)]
    capi.kv_pages_read_dev(p.k, p.v, *back, *p.where(new))
    ref, bound = more.rotate(k[:n], position, f, interleaved)
    assert ((back[0][:n].double().cpu() - ref).abs() <= bound).all()
    assert torch.equal(back[1][:n], v[:n])
    # rows without queries, and queries in place
    before = p.bits()
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, interleaved)
    again = q.clone()
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, interleaved, again, again)
    assert all(torch.equal(a, b) for a, b in zip(before, p.bits()))
    assert torch.equal(again[:n], out[:n]) and torch.equal(again[n:], q[n:])
    capi.stream_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", [None, E4M3, I8, I4])
@pytest.mark.parametrize("D,pairs,interleaved", [(64, 32, False), (128, 64, True), (128, 12, False), (256, 128, False)])
def test_as_rotating_first(cuda, dtype, kind, D, pairs, interleaved):
    """The pages are those of an append of rotated rows, to the last bit."""
    new, keys = [130, 1, 7], [130, 900, 70]
    kind = kind or dtype
    one, two = (Pages(keys, 4, D, 32, kind) for _ in range(2))
    g = _gen(3)
    k, v = (_randn(g, sum(new), 4, D, dtype=dtype) for _ in range(2))
    f = _freq(pairs, 500000.0)
    capi.kv_pages_append_rope_dev(k, v, one.k, one.v, *one.where(new), f, interleaved, **one.kw)
    turned = torch.empty_like(k)
    capi.kv_pages_append_rope_dev(k, v, two.k, two.v, *two.where(new), f, interleaved, k, turned, **two.kw)
    for t in (two.k, two.v, *two.kw.values()):
        t.view(torch.uint8).zero_()
    capi.kv_pages_append_dev(turned, v, two.k, two.v, *two.where(new), **two.kw)
    assert all(torch.equal(a, b) for a, b in zip(one.bits(), two.bits()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("position", [0, 1, 65535, 131071, 1000003, 8000000])
def test_far_positions(cuda, dtype, position):
    """One token at a far position: the table names the same page for all others."""
    D, page = 128, 128
    width = position // page + 1
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    k, v = (torch.zeros(2, 1, page, D, dtype=dtype, device="cuda") for _ in range(2))
    lens = torch.tensor([position + 1], dtype=torch.int32, device="cuda")
    g = _gen(position)
    x = _randn(g, 1, 1, D, dtype=dtype)
    f = _freq(64)
    out = torch.empty_like(x)
    capi.kv_pages_append_rope_dev(x, x, k, v, seq_ref.starts([1]), table, lens, f, Q=x, Q_out=out)
    ref, bound = more.rotate(x, torch.tensor([position]), f, False)
    assert ((out.double().cpu() - ref).abs() <= bound).all()
    assert torch.equal(k[1, 0, position % page], out[0, 0])
    assert (k[0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(cuda, dtype):
    """Slices of one projection, an output with gaps, rows off their alignment by one element."""
    new, keys, D = [40, 3], [300, 3], 64
    n = sum(new)
    g = _gen(9)
    flat = torch.empty(n * 12 * D + 1, dtype=dtype, device="cuda")
    f = _freq(32)
    want = None
    for shift in (0, 1):
        p = Pages(keys, 2, D, 16, dtype)
        qkv = flat[shift: shift + n * 12 * D].view(n, 12, D)
        qkv.copy_(_randn(_gen(9), n, 12, D, dtype=dtype))
        q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
        out = torch.full((8, n, 2 * D), 7.0, dtype=dtype, device="cuda")
        capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, False, q, out[:, :, :D].transpose(0, 1))
        ref, bound = more.rotate(q, _positions(new, keys), f, False)
        assert ((out[:, :, :D].transpose(0, 1).double().cpu() - ref).abs() <= bound).all()
        assert (out[:, :, D:] == 7).all()
        if want is not None:
            assert all(torch.equal(a, b) for a, b in zip(want, p.bits() + [out]))
        want = p.bits() + [out]


def test_zeros_infinities_and_nan_of_what_stays(cuda):
    """Dimensions that are not rotated keep their bits; a NaN reaches its partner alone."""
    D, pairs = 64, 8
    p = Pages([1], 1, D, 16, F32)
    x = torch.zeros(1, 1, D, device="cuda")
    x[0, 0, 16:] = -0.0
    x[0, 0, 20], x[0, 0, 21], x[0, 0, 3] = float("inf"), float("nan"), float("nan")
    capi.kv_pages_append_rope_dev(x, x, p.k, p.v, *p.where([1]), _freq(pairs))
    got = p.k[p.table[0, 0], 0, 0]
    assert torch.equal(got[16:].view(torch.int32), x[0, 0, 16:].view(torch.int32))
    assert torch.isnan(got[:16]).nonzero().flatten().tolist() == [3, 11]


def test_bad_pages_are_not_written(cuda):
    new, keys = [40, 40], [64, 64]
    p = Pages(keys, 2, 64, 16, BF16)
    p.table[0, 2] = 10 ** 6
    q, k, v = (_randn(_gen(4), 80, h, 64, dtype=BF16) for h in (4, 2, 2))
    out = torch.full_like(q, float("nan"))
    f = _freq(32)
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, False, q, out)
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()
    ref, bound = more.rotate(q, _positions(new, keys), f, False)
    assert ((out.double().cpu() - ref).abs() <= bound).all()  # every token's queries
    back = [torch.empty_like(k), torch.empty_like(v)]
    capi.kv_pages_read_dev(p.k, p.v, *back, *p.where(new))
    gone = torch.zeros(80, dtype=torch.bool)
    gone[8:24] = True  # positions 32 to 47 of the first sequence, whose tokens start at 24
    assert (back[1][gone.cuda()] == 0).all() and torch.equal(back[1][~gone.cuda()], v[~gone.cuda()])
    with pytest.raises(capi.AttnbError, match="out of range"):
        capi.stream_status()


def test_captured_and_replayed(cuda):
    """Later lengths and tokens through one captured call, on a stream of its own."""
    D, f = 64, _freq(32)
    p = Pages([200, 300], 2, D, 16, BF16)
    lens = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    p.lens = lens
    q, k, v = (_randn(_gen(5), 2, h, D, dtype=BF16) for h in (4, 2, 2))
    out, where = torch.empty_like(q), p.where([1, 1])
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *where, f, False, q, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *where, f, False, q, out)
    for at in (11, 100, 199):
        lens.copy_(torch.tensor([at, at + 50], dtype=torch.int32))
        q.copy_(_randn(_gen(at), 2, 4, D, dtype=BF16))
        graph.replay()
        ref, bound = more.rotate(q, torch.tensor([at - 1, at + 49]), f, False)
        assert ((out.double().cpu() - ref).abs() <= bound).all()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    want = out.clone()
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *where, f, False, q, out, stream=stream)
    stream.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", [None, E4M3, I4])
@pytest.mark.parametrize("pairs,interleaved", [(32, False), (32, True), (20, False)])
def test_coded_rows_off_their_alignment(cuda, kind, pairs, interleaved):
    new, keys, D, H = [40, 3], [300, 3], 64, 2
    n = sum(new)
    x = _randn(_gen(9), n, 4 * H, D, dtype=BF16)
    got = []
    for shift in (0, 1):
        rows = torch.empty(n * 4 * H * D + 1, dtype=BF16, device="cuda")[shift: shift + n * 4 * H * D].view(n, 4 * H, D)
        rows.copy_(x)
        p = Pages(keys, H, D, 16, kind or BF16)
        out = torch.empty(n, 2 * H, D, dtype=BF16, device="cuda")
        capi.kv_pages_append_rope_dev(rows[:, :H], rows[:, H:2 * H], p.k, p.v, *p.where(new), _freq(pairs), interleaved,
                                      rows[:, 2 * H:], out, **p.kw)
        got.append(p.bits() + [out])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_more_tokens_than_a_cta_takes(cuda):
    """Thousands of tokens of many sequences, some without any, and few heads."""
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 90, (300,), generator=g).tolist()
    keys = [n + int(k) for n, k in zip(new, torch.randint(0, 40, (300,), generator=g))]
    p = Pages(keys, 1, 64, 16, BF16)
    n = sum(new)
    q, k, v = (_randn(_gen(i), n, 1, 64, dtype=BF16) for i in (1, 2, 3))
    out, f = torch.empty_like(q), _freq(32)
    capi.kv_pages_append_rope_dev(k, v, p.k, p.v, *p.where(new), f, True, q, out)
    ref, bound = more.rotate(q, _positions(new, keys), f, True)
    assert ((out.double().cpu() - ref).abs() <= bound).all()
    back = [torch.empty_like(k), torch.empty_like(v)]
    capi.kv_pages_read_dev(p.k, p.v, *back, *p.where(new))
    ref, bound = more.rotate(k, _positions(new, keys), f, True)
    assert ((back[0].double().cpu() - ref).abs() <= bound).all() and torch.equal(back[1], v)
    capi.stream_status()
