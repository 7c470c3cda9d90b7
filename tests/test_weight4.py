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


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_quantised_weights_are_finite(dtype, value):
    w = torch.ones((1500, 64), dtype=dtype)
    quantize_weight4(w, 32)
    w[1400, 63] = value
    with pytest.raises(ValueError, match="finite"):
        quantize_weight4(w, 32)


@pytest.mark.parametrize("dtype,top", [(torch.float16, 65504.0), (torch.bfloat16, 7.5e37)], ids=str)
def test_largest_weights(dtype, top):
    """Groups over the type's range, or up to the largest scale: within a step of 2 top / 15, and the scale's rounding."""
    w = (torch.linspace(-1, 1, 64, dtype=torch.float64) * top).to(dtype).repeat(3, 1)
    back = quantize_weight4(w, 64).dequantize(torch.float64)
    step = 2 * top / 15
    assert ((back - w.double()).abs() <= step * (1 + 15 * torch.finfo(dtype).eps / 2)).all()


def test_ranges_past_the_scales():
    top = torch.finfo(torch.bfloat16).max
    for lo, hi in ((-top, top), (0.0, top), (-8e37, 8.1e37)):
        with pytest.raises(ValueError, match="ranges"):
            quantize_weight4(torch.tensor([[lo, hi] * 16], dtype=torch.bfloat16), 32)


@pytest.mark.gpu
def test_products_with_no_rows(hip_device):
    w = quantize_weight4(torch.zeros((0, 384), dtype=torch.bfloat16, device=hip_device))
    x = torch.ones((5, 384), dtype=torch.bfloat16, device=hip_device)
    assert linear4(x, w).shape == (5, 0) and linear4_silu_mul(x, w).shape == (5, 0)
    assert linear4(x[:0], w).shape == (0, 0)
