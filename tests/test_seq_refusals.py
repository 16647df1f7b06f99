"""Refusals of the operators over ragged sequences and paged KV caches, at the C ABI and in the
Python layer; everything here is refused before any device work, so it runs without a GPU."""
from __future__ import annotations

import ctypes

import pytest

from attn_cpu import capi

PTR = 1 << 20  # never dereferenced: the calls are refused first
F32, BF16, F16, E4M3, I8 = range(5)


def rows(data=PTR, type=BF16, tokens=8, heads=4, Dh=64, sT=None, sH=None):
    return capi.Rows(data, type, tokens, heads, Dh, heads * Dh if sT is None else sT,
                     Dh if sH is None else sH)


def pages(k=PTR, v=PTR, ks=None, vs=None, type=BF16, n=4, H=2, page=16, Dh=64):
    return capi.KvPages(k, v, ks, vs, type, n, H, page, Dh)


def seqs(cu=PTR, batch=2, table=PTR, stride=2, most=2, lens=PTR):
    return capi.Seqs(cu, batch, table, stride, most, lens)


def packed(Q=None, K=None, V=None, O=None, cu_q=PTR, cu_k=PTR, batch=2, scale=0.0, ws=PTR, n=1 << 30):
    Q = Q or rows()
    K = K or rows(heads=2)
    return capi.lib().attnb_attn_packed_dev(Q, K, V or K, O or Q, cu_q, cu_k, batch, 1, scale, ws, n,
                                            None)


def paged(Q=None, pg=None, O=None, sq=None, max_new=0, scale=0.0, ws=PTR, n=1 << 30):
    Q = Q or rows()
    return capi.lib().attnb_attn_paged_dev(Q, pg or pages(), O or Q, sq or seqs(), max_new, 1, scale,
                                           ws, n, None)


def append(K=None, V=None, pg=None, sq=None):
    K = K or rows(heads=2)
    return capi.lib().attnb_kv_pages_append_dev(K, V or K, pg or pages(), sq or seqs(), None)


def read(K=None, V=None, pg=None, sq=None):
    K = K or rows(heads=2)
    return capi.lib().attnb_kv_pages_read_dev(pg or pages(), K, V or K, sq or seqs(), None)


def refused(rc, words):
    assert rc == capi.ERR_INVALID_ARGUMENT
    assert words in capi.lib().attnb_last_error().decode()


@pytest.mark.parametrize("kw,words", [
    (dict(Q=rows(data=None)), "Null data pointer (Q)"),
    (dict(Q=rows(data=PTR + 1)), "Q is not aligned"),
    (dict(Q=rows(type=E4M3)), "Q must be F32, BF16 or F16"),
    (dict(Q=rows(Dh=257)), "Dh in [1, 256]"),
    (dict(Q=rows(Dh=0)), "Dh in [1, 256]"),
    (dict(Q=rows(tokens=-1)), "negative number of tokens"),
    (dict(Q=rows(heads=3)), "multiple of the KV heads"),
    (dict(K=rows(heads=2, type=F16)), "one type"),
    (dict(V=rows(heads=2, tokens=7)), "matching K"),
    (dict(O=rows(type=F16)), "O must have Q's type"),
    (dict(O=rows(heads=2)), "matching Q"),
    (dict(O=rows(sT=0)), "rows that overlap"),
    (dict(O=rows(sH=32)), "rows that overlap"),
    (dict(K=rows(heads=2, Dh=32)), "Dh mismatch"),
    (dict(batch=-1), "batch must be non-negative"),
    (dict(cu_q=None), "Null cu_q or cu_k"),
    (dict(cu_k=None), "Null cu_q or cu_k"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(ws=None), "Null workspace"),
    (dict(Q=rows(tokens=1 << 29), O=rows(tokens=1 << 29)), "below 2^30"),
])
def test_packed(kw, words):
    refused(packed(**kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(pg=pages(type=F16)), "pages must have the rows' type"),
    (dict(pg=pages(type=5)), "unknown page type"),
    (dict(pg=pages(page=48)), "page_size must be"),
    (dict(pg=pages(page=256)), "page_size must be"),
    (dict(pg=pages(k=None)), "Null page pointer"),
    (dict(pg=pages(type=E4M3)), "need scales"),
    (dict(pg=pages(type=I8, ks=PTR)), "need scales"),
    (dict(pg=pages(ks=PTR, vs=PTR)), "only E4M3 and I8 pages have scales"),
    (dict(pg=pages(H=3)), "multiple of the KV heads"),
    (dict(pg=pages(Dh=32)), "Dh mismatch"),
    (dict(sq=seqs(cu=None)), "Null cu, lens or table"),
    (dict(sq=seqs(lens=None)), "Null cu, lens or table"),
    (dict(sq=seqs(table=None)), "Null cu, lens or table"),
    (dict(sq=seqs(batch=-1)), "batch must be non-negative"),
    (dict(sq=seqs(most=-1)), "max_pages must be non-negative"),
    (dict(sq=seqs(stride=-2)), "table_stride must be non-negative"),
    (dict(sq=seqs(most=1 << 26)), "below 2^30"),
    (dict(max_new=-1), "max_new must be non-negative"),
])
def test_paged(kw, words):
    refused(paged(**kw), words)


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("kw,words", [
    (dict(K=rows(heads=3)), "matching the pages"),
    (dict(K=rows(heads=2, Dh=32)), "matching the pages"),
    (dict(V=rows(heads=2, type=F16)), "one type"),
    (dict(V=rows(heads=2, tokens=3)), "matching the pages"),
    (dict(K=rows(heads=2, type=F32)), "one type"),
    (dict(pg=pages(type=F32)), "pages must have the rows' type"),
])
def test_append_and_read(call, kw, words):
    if words == "one type" and "K" in kw:
        kw = dict(kw, V=rows(heads=2))
    refused(call(**kw), words)


def test_read_needs_rows_of_its_own():
    refused(read(K=rows(heads=2, sT=0)), "rows that overlap")


def test_empty_calls_do_nothing():
    assert packed(Q=rows(tokens=0)) == capi.OK
    assert packed(batch=0, cu_q=None, cu_k=None) == capi.OK
    assert paged(Q=rows(tokens=0)) == capi.OK
    assert append(K=rows(heads=2, tokens=0)) == capi.OK
    assert read(sq=seqs(batch=0, cu=None, lens=None, table=None)) == capi.OK


def test_workspace_refusals():
    n = ctypes.c_size_t()
    refused(capi.lib().attnb_seq_workspace(6, 4, 64, ctypes.byref(n)), "multiple of the KV heads")
    refused(capi.lib().attnb_seq_workspace(8, 4, 300, ctypes.byref(n)), "Dh must be in")


def test_python_layer_refuses_host_tensors():
    import torch

    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="CUDA tensors expected"):
        capi.attn_packed_dev(x, x, x, x, torch.zeros(2, dtype=torch.int32))
