"""Norms of the heads, rotation and cache write in one kernel, against the definition in 64 bits.

In fp32 the sum of up to 256 squares is off by at most (8 + 5 + 1) 2^-24 of itself (8 in a lane, 5 steps over the lanes, the
division), rsqrt by an ulp 2^-23 and half of its argument's error, the two products of the norm by 2^-24 each, the
rotation's product and sum by 2^-24 each: below 2^-19 of |a cos| + |b sin|, called A here. What is stored is rounded
once: u |y| (u = 2^-8 bf16, 2^-11 fp16, 2^-4 E4M3, none in fp32; fixed steps below the normal numbers), MXFP4 by half a
step of its block. Values are copied or quantised as write_kv does it, bit for bit.
"""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import HipAttention, fp4_caches
from oracle import fp4

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}
E4M3 = torch.float8_e4m3fn


def _caches(kv, nb, bs, hkv, D, dtype, dev):
    """(k, v, scale arguments) with every byte 0x11."""
    if kv == "fp4":
        k, v, ks, vs = fp4_caches(nb, bs, hkv, D, dev)
        scales = {"k_scale": ks, "v_scale": vs}
    else:
        t = E4M3 if kv == "e4m3" else dtype
        k, v = (torch.zeros((nb, bs, hkv, D * t.itemsize), dtype=torch.uint8, device=dev).view(t) for _ in range(2))
        scales, ks, vs = ({"k_scale": 0.25, "v_scale": 0.5}, None, None) if kv == "e4m3" else ({}, None, None)
    for t in (k, v, ks, vs):
        if t is not None:
            t.view(torch.uint8).fill_(0x11)
    return k, v, scales


def _turn(x, weight, eps, cos, sin, interleaved):
    """(y, A) in 64 bits of heads x [T, h, D]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[:, None], sin.double()[:, None]
    y, a = x.clone(), x.abs()
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    a[..., lo] = (x[..., lo] * c).abs() + (x[..., hi] * s).abs()
    a[..., hi] = (x[..., hi] * c).abs() + (x[..., lo] * s).abs()
    return y, a


def _check_fp4(code, s, y, a):
    """Codes and scales of rows within the format's rounding of y, whose fp32 form is within 2^-19 a of it."""
    b = y.unflatten(-1, (-1, 32))
    top, off = b.abs().amax(-1), 2.0**-19 * a.unflatten(-1, (-1, 32)).amax(-1)
    lo, hi = (fp4.quantize(t.clamp(min=0).cpu().repeat_interleave(32, -1), torch.float32)[1].int() for t in (top - off, top + off))
    got = s.cpu().int()
    assert ((got == lo) | (got == hi)).all()
    unit = fp4.power_of_two(s.int() - 127).repeat_interleave(32, -1)
    z = (y / unit).abs()
    half = torch.where(z < 2, 0.25, torch.where(z < 4, 0.5, 1.0))
    err = (fp4.dequantize(code, s) - y).abs()
    assert (err <= half * unit * (1 + 2.0**-15) + 2.0**-18 * a).all()


def _run(dev, T, H, Hkv, D, rotary, interleaved, dtype, kv, norms="qk", seed=0, bs=16, wide=0, eps=1e-6, scale=1.0, slots=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    width = (H + 2 * Hkv) * D
    qkv = (torch.randn((T, width + wide), generator=g, device=dev) * scale).to(dtype)[:, :width]
    nb, P = -(-T // bs) + 2, 50
    angle = torch.rand((P, rotary // 2), generator=g, device=dev, dtype=torch.float64) * 6.3
    cos, sin = (torch.cos(angle) * 1.3).float(), (torch.sin(angle) * 1.3).float()
    positions = torch.randint(0, P, (T,), generator=g, device=dev)
    if slots is None:
        slots = torch.randperm(nb * bs, generator=g, device=dev)[:T]
    w = {n: (torch.randn(D, generator=g, device=dev) * 0.4 + 1).to(dtype) if n in norms else None for n in "qk"}
    k, v, scales = _caches(kv, nb, bs, Hkv, D, dtype, dev)
    out = HipAttention.norm_rope_and_cache(qkv, positions, cos, sin, k, v, slots, H, w["q"], w["k"], eps, interleaved, **scales)
    x = qkv.unflatten(1, (-1, D))
    c, s = cos[positions], sin[positions]
    y, a = _turn(x[:, :H], w["q"], eps, c, s, interleaved)
    assert out.shape == (T, H, D) and out.dtype == dtype
    assert ((out.double() - y).abs() <= U[dtype] * y.abs() + 2.0**-19 * a + TINY[dtype]).all()
    y, a = _turn(x[:, H : H + Hkv], w["k"], eps, c, s, interleaved)
    vals = x[:, H + Hkv :]
    keep = (slots >= 0) & (slots < nb * bs)
    at, y, a, vals = slots[keep], y[keep], a[keep], vals[keep]
    untouched = torch.ones(nb * bs, dtype=torch.bool, device=dev)
    untouched[at] = False
    for t in (k, v, *(scales.values() if kv == "fp4" else ())):
        assert (t.view(torch.uint8).flatten(0, 1)[untouched] == 0x11).all()
    if kv == "fp4":
        code, e = (t.view(torch.uint8).flatten(0, 1)[at] for t in (k, scales["k_scale"]))
        _check_fp4(code, e, y, a)
        wc, we = fp4.quantize(vals)
        assert torch.equal(v.view(torch.uint8).flatten(0, 1)[at].cpu(), wc)
        assert torch.equal(scales["v_scale"].view(torch.uint8).flatten(0, 1)[at].cpu(), we)
        return
    kr = k.flatten(0, 1).view(torch.uint8)[at].view(k.dtype)
    vr = v.flatten(0, 1).view(torch.uint8)[at].view(v.dtype)
    if kv == "e4m3":
        got, z = kr.float().double(), y / 0.25
        assert ((got - z.clamp(-448, 448)).abs() <= 2.0**-4 * z.abs().clamp(max=448) + 2.0**-10 + 2.0**-18 * a / 0.25).all()
        assert torch.equal(vr.view(torch.uint8), (vals.float() / 0.5).clamp(-448, 448).to(E4M3).view(torch.uint8))
    else:
        assert ((kr.double() - y).abs() <= U[dtype] * y.abs() + 2.0**-19 * a + TINY[dtype]).all()
        assert torch.equal(vr, vals)


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,rotary", [(1, 1, 1, 32, 32), (3, 32, 8, 64, 64), (37, 32, 8, 128, 64), (9, 5, 1, 96, 96),
                                              (2, 7, 7, 160, 16), (5, 3, 1, 256, 256), (4, 6, 2, 192, 96), (6, 4, 2, 64, 0)])  # fmt: skip
def test_layouts(hip_device, dtype, kv, interleaved, T, H, Hkv, D, rotary):
    _run(hip_device, T, H, Hkv, D, rotary, interleaved, dtype, kv, seed=T, wide=32)


@pytest.mark.parametrize("kv", ["own", "e4m3"])
@pytest.mark.parametrize("D,rotary", [(8, 0), (24, 16), (40, 32), (72, 48), (136, 112), (248, 240)])
def test_odd_heads(hip_device, kv, D, rotary):
    for interleaved in (False, True):
        _run(hip_device, 11, 3, 2, D, rotary, interleaved, torch.bfloat16, kv, seed=D)


@pytest.mark.parametrize("norms", ["", "q", "k"])
@pytest.mark.parametrize("kv", ["own", "fp4"])
def test_one_norm_or_none(hip_device, norms, kv):
    _run(hip_device, 21, 8, 2, 128, 128, False, torch.bfloat16, kv, norms=norms)


@pytest.mark.parametrize("T", [511, 512, 2049])
def test_many_tokens(hip_device, T):
    """Both forms of the grid: a workgroup a pass over the heads, and one a token."""
    _run(hip_device, T, 32, 8, 128, 128, False, torch.bfloat16, "own", seed=T)
    _run(hip_device, T, 9, 3, 64, 32, True, torch.float16, "fp4", seed=T)


@pytest.mark.parametrize("scale,eps", [(1e-4, 1e-6), (1e4, 1e-5), (0.0, 1e-6)])
def test_small_large_and_zero_rows(hip_device, scale, eps):
    """Rows far below the norm's epsilon, far above it (their E4M3 keys past 448 without a norm), and of zeros."""
    for kv in ("own", "e4m3"):
        _run(hip_device, 17, 4, 2, 128, 64, False, torch.bfloat16, kv, scale=scale, eps=eps)
    _run(hip_device, 17, 4, 2, 128, 64, False, torch.bfloat16, "e4m3", norms="", scale=scale, eps=eps)


def test_slots_outside_the_pool_and_positions_past_the_tables(hip_device):
    dev = hip_device
    slots = torch.tensor([-1, 3, 48, 10**15, 0, -(2**62), 47, 20], device=dev)  # a pool of 3 pages of 16
    _run(dev, 8, 4, 2, 64, 64, False, torch.bfloat16, "own", slots=slots)
    _run(dev, 8, 4, 2, 64, 64, False, torch.bfloat16, "fp4", slots=slots)
    qkv = torch.randn((3, 4 * 64), device=dev).bfloat16()
    cos, sin = torch.rand((5, 32), device=dev), torch.rand((5, 32), device=dev)
    k, v, _ = _caches("own", 2, 16, 1, 64, torch.bfloat16, dev)
    args = (cos, sin, k, v, torch.arange(3, device=dev), 2)
    far = HipAttention.norm_rope_and_cache(qkv, torch.tensor([-7, 5, 2**40], device=dev), *args)
    near = HipAttention.norm_rope_and_cache(qkv, torch.tensor([0, 4, 4], device=dev), *args)
    assert torch.equal(far, near)


def test_agrees_with_rope_and_cache(hip_device):
    """Without norms and over whole heads in fp32: rope_and_cache's rotation up to the order of its roundings."""
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn((9, 8 * 64), generator=g, device=dev)
    angle = torch.rand((20, 32), generator=g, device=dev) * 6
    cos, sin = torch.cos(angle), torch.sin(angle)
    positions, slots = torch.arange(9, device=dev), torch.arange(9, device=dev) + 4
    a, b = _caches("own", 2, 16, 2, 64, torch.float32, dev), _caches("own", 2, 16, 2, 64, torch.float32, dev)
    q1 = HipAttention.norm_rope_and_cache(qkv, positions, cos, sin, a[0], a[1], slots, 4)
    q2 = HipAttention.rope_and_cache(qkv, positions, cos.repeat(1, 2), sin.repeat(1, 2), b[0], b[1], slots, 4)
    assert torch.allclose(q1, q2, rtol=0, atol=2.0**-20) and torch.allclose(a[0], b[0], rtol=0, atol=2.0**-20)
    assert torch.equal(a[1], b[1])


def test_out_streams_and_graphs(hip_device):
    """A slice of a wider output, another stream, and a captured call on new inputs."""
    dev = hip_device
    qkv = torch.randn((5, 8 * 128), device=dev).bfloat16()
    cos, sin = torch.rand((9, 32), device=dev), torch.rand((9, 32), device=dev)
    k, v, _ = _caches("own", 2, 16, 2, 128, torch.bfloat16, dev)
    positions, slots = torch.arange(5, device=dev), torch.arange(5, device=dev) * 3
    w = torch.rand(128, device=dev).bfloat16()
    call = lambda **kw: HipAttention.norm_rope_and_cache(qkv, positions, cos, sin, k, v, slots, 4, w, w, **kw)  # noqa: E731
    want = call()
    wide = torch.zeros((7, 6, 128), dtype=torch.bfloat16, device=dev)
    assert torch.equal(call(out=wide[:5, 1:5]), want)
    assert not wide[5:].any() and not wide[:, 0].any() and not wide[:, 5].any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(3):
        qkv.copy_(torch.randn((5, 8 * 128), device=dev))
        positions.add_(1)
        k.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, keys = held.clone(), k.clone()
        k.zero_()
        assert torch.equal(got, call()) and torch.equal(keys, k)


def test_refusals(hip_device):
    dev = hip_device
    qkv = torch.randn((3, 8 * 64), device=dev).bfloat16()
    cos, sin = torch.rand((9, 32), device=dev), torch.rand((9, 32), device=dev)
    k, v, _ = _caches("own", 2, 16, 2, 64, torch.bfloat16, dev)
    i = torch.arange(3, device=dev)
    w = torch.rand(64, device=dev).bfloat16()
    good = [qkv, i, cos, sin, k, v, i, 4, w, w]
    assert HipAttention.norm_rope_and_cache(qkv[:0], i[:0], cos, sin, k, v, i[:0], 4).shape == (0, 4, 64)
    for at, bad in [(0, qkv[:, :-8]), (0, qkv.cpu()), (0, qkv.float()), (1, i.int()), (1, i[:2]), (2, cos.double()),
                    (2, cos[:, :24].contiguous()), (3, sin[:5]), (5, v.float()), (6, i[:2]), (7, 5), (7, 0), (8, w[:32]),
                    (9, w.float()), (9, w.cpu())]:  # fmt: skip
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            HipAttention.norm_rope_and_cache(*args)
    for r in (20, 40):  # pairs that are no multiple of 8, a rotation wider than the head
        t = torch.rand((9, r), device=dev)
        with pytest.raises(ValueError):
            HipAttention.norm_rope_and_cache(qkv, i, t, t, k, v, i, 4)
    for eps in (-1.0, float("nan")):
        with pytest.raises(RuntimeError):
            HipAttention.norm_rope_and_cache(*good, eps)
