"""The choice of blocks where scores lie far apart: many close ones next to a few far off."""
from __future__ import annotations

import pytest
import torch

import seq_ref_more as more
from test_gpu_blocks import _select
from test_gpu_rope_append import Pages
from test_gpu_seq_ops import F32

pytestmark = pytest.mark.gpu


def _scored(n, score):
    """Pages of 16 keys whose block j scores score[j] for a query of 1 in dimension 0 (bounds that are equal there)."""
    p = Pages([16 * n], 1, 64, 16, F32)
    p.bounds = torch.zeros(p.k.shape[0], 1, 2, 64, device="cuda")
    p.bounds[p.table[0].long(), 0, :, 0] = score.cuda()[:, None]
    return p


# A row alone: keys of up to 512 blocks are taken by a warp, of more by a CTA of 512 threads.  320 rows of up to 4096: a CTA of 256
# threads.  What counts is how many of the close ones share a part of the range: next to the threads, and many.
@pytest.mark.parametrize("n,rows", [(500, 1), (513, 1), (515, 1), (518, 1), (700, 1), (5000, 1), (700, 320), (4000, 320)])
@pytest.mark.parametrize("below,above", [(0, 1), (1, 1), (1, 40), (0, 300)])
def test_many_close_scores_next_to_far_ones(cuda, n, rows, below, above):
    g = torch.Generator().manual_seed(n + above)
    score = 1000.0 + torch.randperm(n, generator=g).float() / 8  # distinct, and all exact
    far = torch.randperm(n - 2, generator=g)[: below + above] + 1
    score[far[:above]] = 1e30 * (1 + torch.arange(above) / 1024)
    score[far[above:]] = -1e28  # the close ones then lie in part 20 of 2048, else in part 0
    p = _scored(n, score)
    q = torch.zeros(rows, 1, 64, device="cuda")
    q[:, 0, 0] = 1
    for take in (3, 37, 257, 490):
        blocks = _select(p, q, [rows], take)[:, 0].cpu()
        for i in {0, rows // 2, rows - 1}:
            own = (16 * n - rows + i) // 16
            want = more.select(score[: own + 1].double(), take, 1, 1)
            assert blocks[i].tolist() == want, (take, i)


@pytest.mark.parametrize("n", [259, 300, 515, 516, 517, 700])
def test_as_many_close_scores_as_threads(cuda, n):
    """All but one of the n - 2 scored blocks in the lowest part, around the number of threads that rank a part."""
    score = 1000.0 + torch.arange(n).flip(0).float() / 8
    score[7] = 1e30
    for rows in (1, 320):
        p = _scored(n, score)
        q = torch.zeros(rows, 1, 64, device="cuda")
        q[:, 0, 0] = 1
        for take in (4, 200):
            blocks = _select(p, q, [rows], take)[:, 0].cpu()
            for i in range(rows):
                own = (16 * n - rows + i) // 16
                assert blocks[i].tolist() == more.select(score[: own + 1].double(), take, 1, 1), (take, i)
