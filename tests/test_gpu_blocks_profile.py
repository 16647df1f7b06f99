"""Timing of the calls for selected blocks."""
from __future__ import annotations

import pytest
import torch

from attn_cpu import capi
from test_gpu_blocks import _bound, _filled, _select
from test_gpu_seq_ops import BF16, _gen, _randn

pytestmark = pytest.mark.gpu


def test_every_call_is_timed(cuda):
    keys = [500]
    p = _filled(keys, 1, 64, 16, BF16, BF16)
    q = _randn(_gen(1), 3, 2, 64, dtype=BF16)
    o = torch.empty_like(q)
    for name in ("kv_blocks", "seq_attn"):
        capi.profile_read(name)
    capi.profile_enable(True)
    try:
        _bound(p, keys)
        blocks = _select(p, q, [3], 5)
        _select(p, q, [3], 5)
        capi.attn_blocks_dev(q, p.k, p.v, o, blocks, *p.where([3]))
    finally:
        capi.profile_enable(False)
    for name, count in (("kv_blocks", 3), ("seq_attn", 1)):
        ms, launches = capi.profile_read(name)
        assert launches == count and ms > 0
