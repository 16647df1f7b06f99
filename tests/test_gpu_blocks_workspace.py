"""Memory that the choice of blocks and attention over lists take besides their arguments."""
from __future__ import annotations

import ctypes

import pytest
import torch

from attn_cpu import capi
from test_gpu_blocks import _bound, _filled, _select, _wanted
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


@pytest.mark.parametrize("width", [100, 512])
def test_choice_from_short_tables_holds_no_scores(cuda, width):
    """Rows of up to 512 blocks have their scores in shared memory: what attention takes is enough for both calls."""
    new, H, take = 200, 4, 6
    keys = [16 * width]
    p = _filled(keys, H, 64, 16, BF16, BF16)
    _bound(p, keys)
    q = _randn(_gen(1), new, H, 64, dtype=BF16)
    both, attention = ctypes.c_size_t(), ctypes.c_size_t()
    capi.check(capi.lib().attnb_blocks_workspace(new * 1000, H, H, 64, take, width, ctypes.byref(both)))
    capi.check(capi.lib().attnb_seq_workspace(H, H, 64, ctypes.byref(attention)))
    assert both.value == attention.value
    blocks = _select(p, q, [new], take, 1, 2)
    assert torch.equal(blocks.cpu(), _wanted(p, q, [new], keys, take, 1, 2))
