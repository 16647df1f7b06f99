"""What the paged cache object refuses before it takes any memory."""
from __future__ import annotations

import pytest
import torch

from attn_cpu import capi


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("pages,page,most", [(2 ** 24, 64, None), (2 ** 23, 128, None), (10, 16, 2 ** 30), (10, 16, 2 ** 30 - 15)])
def test_bounds_of_sequences_too_long_for_them(dtype, pages, page, most):
    """An append would write, and rotate in place, before the call for its bounds refused."""
    with pytest.raises(ValueError, match="bounds need max_tokens below"):
        capi.PagedKVCacheDev(1, 1, 32, num_pages=pages, page_size=page, dtype=dtype, max_tokens=most, device="cuda:0", bounds=True)


def test_bounds_of_tables_too_large_for_them():
    with pytest.raises(ValueError, match="fewer than 2\\^31 pages"):
        capi.PagedKVCacheDev(2 ** 10, 1, 32, num_pages=10, page_size=16, max_tokens=2 ** 25, device="cuda:0", bounds=True)
