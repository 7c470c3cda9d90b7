"""Products with 4-bit weights of rows of x near the ends of the types' ranges, against the definition in 64 bits: finite rows
give finite sums wherever the result is one, and infinity with its sign behind the type's range.

The bounds are test_hip_linear4's. A result whose bound reaches past the largest finite value may be either."""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import linear4, linear4_silu_mul
from tests.test_hip_linear4 import U, _bounds, _weight, _x

pytestmark = pytest.mark.gpu


def _check(got, want, err, dtype):
    top = torch.finfo(dtype).max
    bound = U[dtype] * want.abs() + err * (1 + U[dtype]) + torch.finfo(dtype).smallest_normal
    got = got.double()
    assert not got.isnan().any()
    beyond = (want.abs() - bound > top * (1 + U[dtype])) & (got == want.sign() * float("inf"))
    edge = (want.abs() + bound >= top) & (got.sign() == want.sign())  # rounded either way
    assert (((got - want).abs() <= bound) | beyond | edge).all()
    assert (want.abs() + bound < top).any()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n", [(1, 176), (16, 5000), (20, 1040), (64, 176), (70, 16400)])
@pytest.mark.parametrize("size", [1e30, 1e35, 3e36, 3e37, 3.3e38])
def test_large_rows(hip_device, group, m, n, size):
    """Up to the largest values of bf16. Rows where the scales keep the result small, and rows where it overflows."""
    k = 512
    w, W, mag = _weight(n, k, group, torch.bfloat16, hip_device, seed=m)
    x = _x(m, k, torch.bfloat16, hip_device, m).float()
    x = (x / x.abs().amax(1, keepdim=True) * size).clamp(-3.38e38, 3.38e38).bfloat16()
    x[0, 1:] = 0  # one element alone
    want, err = _bounds(x, W, mag)
    _check(linear4(x, w), want, err, torch.bfloat16)


def test_large_rows_of_a_split_product(hip_device):
    w, W, mag = _weight(2048, 8192, 64, torch.bfloat16, hip_device)
    x = (_x(33, 8192, torch.bfloat16, hip_device).float().clamp(-30, 30) * 1e36).bfloat16()
    want, err = _bounds(x, W, mag)
    _check(linear4(x, w), want, err, torch.bfloat16)


def test_largest_rows_of_fp16(hip_device):
    w, W, mag = _weight(176, 512, 32, torch.float16, hip_device)
    x = torch.full((5, 512), 65504.0, dtype=torch.float16, device=hip_device)
    x[1] = -x[1]
    x[2, ::2] = -x[2, ::2]
    x[3:, 1:] = 0
    want, err = _bounds(x, W, mag)
    _check(linear4(x, w), want, err, torch.float16)


def test_large_gates(hip_device):
    """SiLU(g) u of gates and up rows around 1e15."""
    w, W, _ = _weight(64, 256, 128, torch.bfloat16, hip_device)
    x = torch.zeros((2, 256), device=hip_device)
    x[0, 0], x[1, 0] = 1e17, -1e17
    got = linear4_silu_mul(x.bfloat16(), w).double()
    y = x.bfloat16().double() @ W.t().contiguous()
    g, u = y[:, :32], y[:, 32:]
    want = g * torch.sigmoid(g) * u
    assert torch.isfinite(got).all() and ((got - want).abs() <= 2.0**-7 * want.abs() + 1e-30).all()
    assert (want.abs() > 1e30).any()
