"""Memory that attention over lists takes besides its arguments."""
from __future__ import annotations

import torch
import pytest

from attn_cpu import capi
from test_gpu_blocks import _filled
from test_gpu_seq_ops import BF16, F32, _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 128), (BF16, 256)])
def test_no_more_than_attention_to_all_keys(cuda, dtype, D):
    """A wide table and many tokens: the choice holds scores for them, attention to its lists does not."""
    new, keys = 300, [4000]
    p = _filled(keys, 2, D, 16, dtype, dtype)
    q = _randn(_gen(1), new, 4, D, dtype=dtype)
    o = torch.empty_like(q)
    blocks = torch.arange(4, dtype=torch.int32, device="cuda").expand(new, 2, 4).contiguous()
    table = torch.zeros(1, 20000, dtype=torch.int32, device="cuda")
    table[:, : p.table.shape[1]] = p.table
    p.table = table
    where = p.where([new])

    def peak(call):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        call()
        return torch.cuda.max_memory_allocated() - before

    all_keys = peak(lambda: capi.attn_paged_dev(q, p.k, p.v, o, *where))
    assert peak(lambda: capi.attn_blocks_dev(q, p.k, p.v, o, blocks, *where)) <= all_keys
