"""Refusals of the rotated append, the 4-bit cache and the selected blocks, at the C ABI and in the
Python layer; everything here is refused before any device work, so it runs without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from attn_cpu import capi
from test_seq_refusals import BF16, E4M3, F16, F32, I8, PTR, pages, refused, rows, seqs

I4 = 6


def pages4(k=PTR, v=PTR, ks=PTR, vs=PTR, kg=PTR, vg=PTR, Dh=64, type=I4):
    return capi.KvPages(k, v, ks, vs, type, 4, 2, 16, Dh, kg, vg)


def rope(f=PTR, pairs=32, interleaved=0):
    return capi.Rope(f, pairs, interleaved)


def append(Q=None, QO=None, K=None, V=None, pg=None, sq=None, rp=None):
    K = K or rows(heads=2)
    return capi.lib().attnb_kv_pages_append_rope_dev(Q, QO, K, V or K, pg or pages(), sq or seqs(), rp or rope(), None)


def bounds(data=PTR, type=BF16):
    return capi.Bounds(data, type)


def bound(pg=None, b=None, sq=None):
    return capi.lib().attnb_kv_blocks_bounds_dev(pg or pages(), b or bounds(), sq or seqs(), None)


def select(Q=None, b=None, num=4, H=2, page=16, sq=None, first=1, last=1, blocks=PTR, take=4, ws=PTR, n=1 << 30):
    return capi.lib().attnb_kv_blocks_select_dev(Q or rows(), b or bounds(), num, H, page, sq or seqs(), first, last, blocks,
                                                 take, ws, n, None)


def attend(Q=None, pg=None, O=None, sq=None, blocks=PTR, take=4, scale=0.0, ws=PTR, n=1 << 30):
    Q = Q or rows()
    return capi.lib().attnb_attn_blocks_dev(Q, pg or pages(), O or Q, sq or seqs(), blocks, take, scale, ws, n, None)


@pytest.mark.parametrize("kw,words", [
    (dict(rp=rope(f=None)), "Null data pointer (inv_freq)"),
    (dict(rp=rope(f=PTR + 2)), "inv_freq is not aligned"),
    (dict(rp=rope(pairs=0)), "pairs must be in"),
    (dict(rp=rope(pairs=33)), "pairs must be in"),
    (dict(Q=rows()), "both be given"),
    (dict(QO=rows()), "both be given"),
    (dict(Q=rows(type=F16), QO=rows(type=F16)), "K's type"),
    (dict(Q=rows(), QO=rows(type=F16)), "K's type"),
    (dict(Q=rows(tokens=7), QO=rows(tokens=7)), "K's tokens"),
    (dict(Q=rows(Dh=32), QO=rows(Dh=32)), "K's tokens"),
    (dict(Q=rows(), QO=rows(heads=2)), "matching Q"),
    (dict(Q=rows(), QO=rows(sT=0)), "rows that overlap"),
    (dict(Q=rows(), QO=rows(sT=512)), "must have Q's strides"),
    (dict(Q=rows(data=None), QO=rows()), "Null data pointer (Q)"),
    (dict(K=rows(heads=3)), "matching the pages"),
    (dict(V=rows(heads=2, type=F32)), "one type"),
    (dict(pg=pages(type=F32)), "pages must have the rows' type"),
    (dict(sq=seqs(lens=None)), "Null cu, lens or table"),
])
def test_rotated_append(kw, words):
    refused(append(**kw), words)


def test_no_rope_descriptor():
    K = rows(heads=2)
    refused(capi.lib().attnb_kv_pages_append_rope_dev(None, None, K, K, pages(), seqs(), None, None), "Null rope")


@pytest.mark.parametrize("kw,words", [
    (dict(kg=None), "need k_group and v_group"),
    (dict(vg=None), "need k_group and v_group"),
    (dict(ks=None), "need scales"),
    (dict(k=PTR + 2), "4-byte boundaries"),
    (dict(v=PTR + 1), "4-byte boundaries"),
    (dict(kg=PTR + 2), "4-byte boundaries"),
    (dict(vg=PTR + 3), "4-byte boundaries"),
    (dict(Dh=48), "multiple of 32"),
])
def test_pages_of_four_bits(kw, words):
    Q = rows(Dh=kw.get("Dh", 64))
    K = rows(heads=2, Dh=kw.get("Dh", 64))
    L = capi.lib()
    refused(L.attnb_attn_paged_dev(Q, pages4(**kw), Q, seqs(), 0, 1, 0.0, PTR, 1 << 30, None), words)
    refused(L.attnb_kv_pages_append_dev(K, K, pages4(**kw), seqs(), None), words)
    refused(L.attnb_kv_pages_read_dev(pages4(**kw), K, K, seqs(), None), words)
    refused(attend(Q=Q, pg=pages4(**kw)), words)
    if "v" not in kw and "vg" not in kw:
        refused(bound(pg=pages4(**kw)), words)


@pytest.mark.parametrize("kw,words", [
    (dict(b=bounds(data=None)), "Null data pointer (bounds)"),
    (dict(b=bounds(data=PTR + 1)), "bounds are not aligned"),
    (dict(b=bounds(type=I8)), "bounds must be F32, BF16 or F16"),
    (dict(pg=pages(type=F16)), "pages must have the rows' type"),
    (dict(pg=pages(k=None)), "Null page pointer"),
    (dict(pg=pages(type=E4M3)), "need scales"),
    (dict(sq=seqs(cu=None)), "Null cu, lens or table"),
    (dict(sq=seqs(most=1 << 26)), "below 2^30"),
    (dict(sq=seqs(batch=1 << 16, most=1 << 15)), "below 2^31"),
])
def test_bounds(kw, words):
    refused(bound(**kw), words)


def test_bounds_look_at_keys_alone():
    assert bound(pg=pages(v=None), sq=seqs(batch=0)) == capi.OK


@pytest.mark.parametrize("kw,words", [
    (dict(b=bounds(type=F16)), "bounds' type"),
    (dict(H=3), "multiple of the KV heads"),
    (dict(H=0), "invalid number or H"),
    (dict(num=-1), "invalid number or H"),
    (dict(page=48), "page_size must be"),
    (dict(first=-1), "keep_first must be"),
    (dict(last=0), "keep_last must be"),
    (dict(first=2, last=3), "no more than take"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "no more than take"),
    (dict(take=0), "take must be positive"),
    (dict(blocks=None), "Null data pointer (blocks)"),
    (dict(blocks=PTR + 2), "blocks are not aligned"),
    (dict(Q=rows(tokens=1 << 29)), "below 2^30"),
    (dict(sq=seqs(most=1 << 26)), "below 2^30"),
    (dict(ws=None), "Null workspace"),
])
def test_select(kw, words):
    refused(select(**kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(O=rows(type=F16)), "O must have Q's type"),
    (dict(O=rows(sT=0)), "rows that overlap"),
    (dict(pg=pages(H=3)), "multiple of the KV heads"),
    (dict(pg=pages(Dh=32)), "Dh mismatch"),
    (dict(take=-1), "take must be positive"),
    (dict(take=1 << 26), "below 2^30"),
    (dict(blocks=None), "Null data pointer (blocks)"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(ws=None), "Null workspace"),
])
def test_attend(kw, words):
    refused(attend(**kw), words)


def test_empty_calls_do_nothing():
    none = rows(heads=2, tokens=0)
    assert append(K=none) == capi.OK
    assert append(sq=seqs(batch=0, cu=None, lens=None, table=None)) == capi.OK
    assert bound(sq=seqs(batch=0, cu=None, lens=None, table=None)) == capi.OK
    assert select(Q=rows(tokens=0), blocks=None) == capi.OK
    assert attend(Q=rows(tokens=0), blocks=None) == capi.OK


def test_workspace_refusals():
    n = ctypes.c_size_t()
    ws = capi.lib().attnb_blocks_workspace
    refused(ws(4, 6, 4, 64, 8, 8, ctypes.byref(n)), "multiple of the KV heads")
    refused(ws(4, 8, 4, 300, 8, 8, ctypes.byref(n)), "Dh must be in")
    refused(ws(-1, 8, 4, 64, 8, 8, ctypes.byref(n)), "non-negative")
    refused(ws(4, 8, 4, 64, 0, 8, ctypes.byref(n)), "take must be positive")


def test_python_layer():
    x = torch.zeros(4, 2, 64)
    one = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        capi.kv_pages_append_rope_dev(x, x, x, x, one, one, one, x)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        capi.kv_blocks_bounds_dev(x, x, one, one, one)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        capi.kv_blocks_select_dev(x, x, x, one, one, one, 16)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        capi.attn_blocks_dev(x, x, x, x, x, one, one, one)
    # a pool on the host, as far as its shapes are checked
    kw = dict(device=torch.device("cpu"))
    codes, scale = torch.zeros(3, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 16)
    group = torch.zeros(3, 2, 16, 4, dtype=torch.uint8)
    assert capi._pages(codes, codes, scale, scale, k_group=group, v_group=group, **kw).Dh == 64
    with pytest.raises(ValueError, match="need k_group and v_group"):
        capi._pages(codes, codes, scale, scale, k_group=group, **kw)
    with pytest.raises(ValueError, match="need k_group and v_group"):
        capi._pages(codes, codes, scale, scale, k_group=group[..., :2], v_group=group, **kw)
    with pytest.raises(ValueError, match="only uint8 pages"):
        capi._pages(codes.char(), codes.char(), scale, scale, k_group=group, v_group=group, **kw)
    with pytest.raises(ValueError, match="bounds must be"):
        capi._bounds(torch.zeros(3, 2, 64), 3, 2, 64, torch.device("cpu"))
    with pytest.raises(ValueError, match="blocks must be"):
        capi._lists(torch.zeros(4, 2, 8), 4, 2, torch.device("cpu"))


def test_cache_object():
    with pytest.raises(ValueError, match="multiple of 32"):
        capi.PagedKVCacheDev(1, 2, 80, 4, dtype=torch.uint8, device="cpu")
    with pytest.raises(ValueError, match="have their type"):
        capi.PagedKVCacheDev(1, 2, 64, 4, dtype=torch.float16, device="cpu", bounds=torch.bfloat16)
    with pytest.raises(ValueError, match="bounds must be float32"):
        capi.PagedKVCacheDev(1, 2, 64, 4, dtype=torch.int8, device="cpu", bounds=torch.int8)
