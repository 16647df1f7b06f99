"""Softmax scales that fp32 does not hold are refused (without a GPU): in units of log2 the largest
ones overflow, and the smallest ones would be 0, which stands for the default."""
from __future__ import annotations

import pytest

from attn_cpu import capi
from test_seq_refusals import packed, paged, refused


@pytest.mark.parametrize("call", [packed, paged])
@pytest.mark.parametrize("scale", [3e38, float("inf"), float("-inf"), float("nan")])
def test_scales_out_of_range(call, scale):
    refused(call(scale=scale), "scale must be finite")


@pytest.mark.parametrize("scale", [0, -1.0, 1e-46, float("nan")])
def test_python_layer(scale):
    with pytest.raises(ValueError, match="scale must be positive"):
        capi._scale(scale)


def test_python_layer_passes_scales_on():
    assert capi._scale(None) == 0.0 and capi._scale(0.25) == 0.25 and capi._scale(1e-44) > 0
