"""Pointers that kernels could not read: scales, offsets, lengths and tables off their elements'
alignment are refused before any device work, so it runs without a GPU."""
from __future__ import annotations

import pytest

from test_seq_refusals import E4M3, PTR, append, packed, paged, pages, read, refused, rows, seqs


@pytest.mark.parametrize("kw,words", [
    (dict(cu_q=PTR + 2), "cu_q is not aligned"),
    (dict(cu_k=PTR + 1), "cu_k is not aligned"),
])
def test_packed(kw, words):
    refused(packed(**kw), words)


@pytest.mark.parametrize("call", [paged, append, read])
@pytest.mark.parametrize("kw,words", [
    (dict(sq=seqs(cu=PTR + 2)), "cu, lens or table is not aligned"),
    (dict(sq=seqs(lens=PTR + 3)), "cu, lens or table is not aligned"),
    (dict(sq=seqs(table=PTR + 1)), "cu, lens or table is not aligned"),
    (dict(pg=pages(type=E4M3, ks=PTR + 2, vs=PTR)), "scales are not aligned"),
    (dict(pg=pages(type=E4M3, ks=PTR, vs=PTR + 1)), "scales are not aligned"),
    (dict(pg=pages(k=PTR + 1)), "pages are not aligned"),
])
def test_pages_and_sequences(call, kw, words):
    refused(call(**kw), words)


def test_a_single_sequence_of_no_pages_needs_no_table():
    assert read(K=rows(heads=2, tokens=0), sq=seqs(batch=1, table=None, most=0)) == 0
