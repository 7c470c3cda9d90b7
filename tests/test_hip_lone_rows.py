"""One row alone: its stride is used by nothing and may be anything, in the calls on tensors and in the methods' own path."""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import HipAttention, _lib, linear4, linear4_silu_mul
from tests.test_hip_linear4 import _weight, _x
from tests.test_hip_norm_rope import _caches

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["calls", "method"])
def path(request, monkeypatch):
    _lib.load()
    if request.param == "method":
        monkeypatch.setattr(_lib, "_calls", None)


def _lone(t: torch.Tensor, stride: int) -> torch.Tensor:
    return t.as_strided(t.shape, (stride, *t.stride()[1:]))


@pytest.mark.parametrize("stride", [0, 1, 7, 2**40])
@pytest.mark.parametrize("n", [160, 70, 16])
def test_linear4(hip_device, path, stride, n):
    w, _, _ = _weight(n, 256, 64, torch.bfloat16, hip_device)
    x = _x(1, 256, torch.bfloat16, hip_device)
    want = linear4(x, w)
    assert torch.equal(linear4(_lone(x, stride), w), want)
    out = torch.full((3, n), 5.0, dtype=x.dtype, device=hip_device)
    linear4(x, w, out=_lone(out[1:2], stride))
    assert torch.equal(out[1:2], want) and (out[[0, 2]] == 5).all()
    if n % 32 == 0:
        assert torch.equal(linear4_silu_mul(_lone(x, stride), w), linear4_silu_mul(x, w))


def test_a_column_turned_round(hip_device, path):
    w, _, _ = _weight(48, 128, 32, torch.float16, hip_device)
    x = _x(1, 128, torch.float16, hip_device)
    assert torch.equal(linear4(x.reshape(128, 1).t(), w), linear4(x, w))


@pytest.mark.parametrize("stride", [0, 1, 7, 2**40])
@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
def test_norm_rope_and_cache(hip_device, path, stride, kv):
    dev = hip_device
    qkv = torch.randn((1, 8 * 64), device=dev).bfloat16()
    cos, sin = torch.rand((9, 32), device=dev), torch.rand((9, 32), device=dev)
    got = []
    for lone in (False, True):
        k, v, scales = _caches(kv, 2, 16, 2, 64, torch.bfloat16, dev)
        buf = torch.full((3, 4, 64), 5.0, dtype=qkv.dtype, device=dev)
        x, out = (_lone(qkv, stride), _lone(buf[1:2], stride)) if lone else (qkv, buf[1:2])
        one = torch.tensor([3], device=dev)
        HipAttention.norm_rope_and_cache(x, one, cos, sin, k, v, one, 4, out=out, **scales)
        got.append([buf, *(t.view(torch.uint8) for t in (k, v))])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert not (got[0][0][1] == 5).all() and (got[0][0][[0, 2]] == 5).all()
