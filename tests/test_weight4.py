"""Weight4 at the ends of its domain, without a GPU."""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import Weight4, linear4, linear4_silu_mul, quantize_weight4


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_no_rows(dtype, group):
    """A weight of no rows, packed, quantised and read back."""
    packed = Weight4.pack(torch.zeros((0, 192), dtype=torch.uint8), torch.zeros((0, 384 // group), dtype=dtype))
    for w in (packed, quantize_weight4(torch.zeros((0, 384), dtype=dtype), group)):
        assert w.shape == (0, 384) and w.group == group and w.dtype == dtype
        assert w.codes.shape == (0, 3, 256) and w.scales.shape == (0, 3 * 128 // group, 16)
        assert w.dequantize().shape == (0, 384) and w.to("cpu").shape == w.shape


@pytest.mark.gpu
def test_products_with_no_rows(hip_device):
    w = quantize_weight4(torch.zeros((0, 384), dtype=torch.bfloat16, device=hip_device))
    x = torch.ones((5, 384), dtype=torch.bfloat16, device=hip_device)
    assert linear4(x, w).shape == (5, 0) and linear4_silu_mul(x, w).shape == (5, 0)
    assert linear4(x[:0], w).shape == (0, 0)
