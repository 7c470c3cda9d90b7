"""Products with 4-bit weights on the GPU, against the definition in 64 bits.

The operands 16 + q and x are exact, so the sums alone round: with W' = s (q - z) and N the sum of |x| s (16 + q + 16 + z)
(at most 47 s |x| an element), k products summed in fp32 in any order are off by at most k 2^-24 of N's terms. The test
takes 2^-24 (k / 4 + 64) N: a row's k is summed in four or more slices, those in steps of 32 inside an instruction. The
output is rounded once, u |y| with u = 2^-8 (bf16) or 2^-11 (fp16; 2^-25 where it is subnormal). The gated form: with eg, eu the
bounds of g and u before rounding, SiLU's slope is below 1.1 and exp and the division are off by less than 2^-20 of its
value.
"""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import Weight4, linear4, linear4_silu_mul, quantize_weight4

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _weight(n, k, group, dtype, dev, seed=0, symmetric=False):
    """(Weight4, W, s (32 + q + z)) of random codes, scales over a wide range and zero points from end to end."""
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=g, device=dev)
    scales = (0.02 * torch.exp(torch.randn((n, k // group), generator=g, device=dev))).to(dtype)
    scales[:: max(1, n // 3), 0] = 0.0
    z = torch.randint(0, 16, (n, k // group), generator=g, device=dev, dtype=torch.uint8)
    if symmetric:
        z.fill_(8)
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)
    s, zz = (t.double().repeat_interleave(group, 1) for t in (scales, z))
    return Weight4.pack(codes, scales, None if symmetric else z), s * (q - zz), s * (32 + q + zz)


def _bounds(x, w, mag):
    """The product in 64 bits and how far fp32 sums may be from it."""
    x, k = x.double(), x.shape[1]
    return x @ w.t().contiguous(), 2.0**-24 * (k / 4 + 64) * (x.abs() @ mag.t().contiguous())


def _check(got, want, err, dtype):
    bound = U[dtype] * want.abs() + err * (1 + U[dtype]) + 2.0**-25
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"{float((off - bound).max()):.3e} past the bound"


def _x(m, k, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    return (torch.randn((m, k), generator=g, device=dev) * torch.exp(torch.randn(k, generator=g, device=dev))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 48, 49, 64, 65, 130, 257])
def test_rows(hip_device, dtype, group, m):
    w, W, mag = _weight(176, 1024, group, dtype, hip_device, seed=m)
    x = _x(m, 1024, dtype, hip_device, m)
    _check(linear4(x, w), *_bounds(x, W, mag), dtype)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 7, 16, 30, 513])
@pytest.mark.parametrize("groups", [1, 2, 3, 7, 21, 40])
@pytest.mark.parametrize("m", [3, 50])
def test_odd_weights(hip_device, group, n, groups, m):
    """Rows that fill no tile, k that fills no block, fewer blocks than waves."""
    k = group * groups
    w, W, mag = _weight(n, k, group, torch.bfloat16, hip_device, seed=n + groups)
    x = _x(m, k, torch.bfloat16, hip_device, n)
    _check(linear4(x, w), *_bounds(x, W, mag), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,n,k,group", [(1, 4096, 4096, 128), (16, 6144, 4096, 128), (20, 2048, 8192, 64), (64, 16400, 512, 32),
                                         (5, 40000, 256, 128), (300, 2048, 2048, 128), (1, 128, 20480, 128)])  # fmt: skip
def test_sizes(hip_device, dtype, m, n, k, group):
    w, W, mag = _weight(n, k, group, dtype, hip_device, seed=m)
    x = _x(m, k, dtype, hip_device, m)
    _check(linear4(x, w), *_bounds(x, W, mag), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,inter,k", [(1, 16, 256), (3, 48, 640), (8, 8192, 1024), (17, 304, 384), (40, 1008, 896), (64, 2064, 512), (150, 80, 1024)])
def test_silu_mul(hip_device, dtype, group, m, inter, k):
    w, W, mag = _weight(2 * inter, k, group, dtype, hip_device, seed=m)
    x = 0.3 * _x(m, k, dtype, hip_device, m)
    y, err = _bounds(x, W, mag)
    g, u, eg, eu = y[:, :inter], y[:, inter:], err[:, :inter], err[:, inter:]
    act = g * torch.sigmoid(g)
    want = act * u
    off = (1.1 * eg + 2.0**-20 * act.abs()) * (u.abs() + eu) + act.abs() * eu
    _check(linear4_silu_mul(x, w), want, off, dtype)


def test_gates_far_from_zero(hip_device):
    """SiLU of -1e4 and 1e4: zero and the gate itself, with no NaN of an exponential's infinity."""
    w, W, _ = _weight(64, 128, 128, torch.bfloat16, hip_device, symmetric=True)
    x = torch.zeros((4, 128), device=hip_device)
    x[:, 0] = torch.tensor([1e6, -1e6, 1e4, 0.0], device=hip_device)
    got = linear4_silu_mul(x.bfloat16(), w).double()
    y = x.bfloat16().double() @ W.t().contiguous()
    g, u = y[:, :32], y[:, 32:]
    want = g * torch.sigmoid(g) * u
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= 2.0**-7 * want.abs() + 1e-30).all()


def test_packing_round_trips(hip_device):
    for n, k, group in ((40, 384, 64), (16, 96, 32), (1, 128, 128)):
        w, W, _ = _weight(n, k, group, torch.float16, hip_device, seed=n)
        assert torch.equal(w.dequantize().double(), W)
        assert torch.equal(w.to("cpu").dequantize().double(), W.cpu())


def test_quantised_weights(hip_device):
    """Every element within half a step of its group (and the scale's rounding), zero exactly, and the product with them."""
    g = torch.Generator(device=hip_device).manual_seed(1)
    W = (torch.randn((100, 512), generator=g, device=hip_device) * 0.05).bfloat16()
    W[3] = 0
    W[4, :128] = W[4, :128].abs() + 0.25  # a group on one side of zero
    w = quantize_weight4(W, 64)
    back = w.dequantize().double()
    grp = W.double().unflatten(1, (-1, 64))
    step = (grp.amax(-1).clamp(min=0) - grp.amin(-1).clamp(max=0)) / 15
    # half a step for the code, half a step where the zero point was rounded (the ends), 15 steps of the scale's rounding
    assert ((back - W.double()).abs().unflatten(1, (-1, 64)) <= (1.0 + 15 * 2.0**-8) * step[..., None] + 1e-12).all()
    assert not back[3].any()
    x = _x(5, 512, torch.bfloat16, hip_device)
    y, err = x.double() @ back.t().contiguous(), 2.0**-24 * 200 * (x.double().abs() @ (48 * step.repeat_interleave(64, 1)).t().contiguous())
    _check(linear4(x, w), y, err, torch.bfloat16)


def test_strides_out_and_neighbours(hip_device):
    """Rows of x and y inside wider ones, y at odd places; what lies beside y stays as it was."""
    for dtype in (torch.bfloat16, torch.float16):
        w, W, mag = _weight(70, 256, 64, dtype, hip_device)
        wide = _x(9, 512, dtype, hip_device)
        x = wide[:, 128:384]
        want, err = _bounds(x, W, mag)
        for off in (0, 1, 3):
            y = torch.full((10, 90), 5.0, dtype=dtype, device=hip_device)
            got = linear4(x, w, out=y[:9, off : off + 70])
            _check(got, want, err, dtype)
            assert (y[9] == 5).all() and (y[:, off + 70 :] == 5).all() and (y[:, :off] == 5).all()


def test_rows_do_not_meet(hip_device):
    """A row of NaN, and one of infinities, spoil themselves alone."""
    w, W, mag = _weight(64, 256, 128, torch.bfloat16, hip_device)
    x = _x(20, 256, torch.bfloat16, hip_device)
    clean = linear4(x, w)
    x[7] = float("nan")
    x[12, 3] = float("inf")
    got = linear4(x, w)
    rows = torch.ones(20, dtype=torch.bool, device=hip_device)
    rows[[7, 12]] = False
    assert torch.equal(got[rows], clean[rows])
    assert got[7].isnan().all() and got[12].isnan().all()


def test_graphs_and_streams(hip_device):
    w, _, _ = _weight(512, 1024, 128, torch.bfloat16, hip_device)
    x = _x(12, 1024, torch.bfloat16, hip_device)
    want = linear4(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear4(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, gated = linear4(x, w), linear4_silu_mul(x, w)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        a, b = held.clone(), gated.clone()
        assert torch.equal(a, linear4(x, w)) and torch.equal(b, linear4_silu_mul(x, w))


def test_refusals(hip_device):
    dev = hip_device
    w, _, _ = _weight(48, 256, 64, torch.bfloat16, dev)
    x = _x(3, 256, torch.bfloat16, dev)
    assert linear4(x[:0], w).shape == (0, 48)
    for bad in (x[:, :128], x.half(), x.cpu(), x[0], x.t().contiguous().t()):
        with pytest.raises(ValueError):
            linear4(bad, w)
    with pytest.raises(ValueError):
        linear4_silu_mul(x, w)  # 24 gate rows fill no tile
    with pytest.raises(ValueError):
        linear4(x, w.to("cpu"))
    for out in (torch.empty((3, 47), dtype=x.dtype, device=dev), torch.empty((3, 48), device=dev), torch.empty((3, 48), dtype=x.dtype)):
        with pytest.raises(ValueError):
            linear4(x, w, out=out)
    with pytest.raises(RuntimeError):
        linear4(torch.empty((3, 260), dtype=x.dtype, device=dev)[:, 2:258], w)  # rows that are not 16-byte aligned


@pytest.mark.parametrize("dtype,group", [(torch.bfloat16, 128), (torch.float16, 32), (torch.bfloat16, 64)], ids=str)
@pytest.mark.parametrize("m,n", [(40, 1040), (64, 1040), (200, 2064), (24, 12320), (40, 12320), (64, 12320), (500, 2080), (20, 20000),
                                 (40, 20000), (64, 20000), (24, 40032), (33, 40032), (200, 16448), (100, 33024)])  # fmt: skip
def test_wide_products(hip_device, dtype, group, m, n):
    """Workgroups of 32 to 256 weight rows, plain and gated, k of an odd number of blocks."""
    k = 1056 if group == 32 else 1088 if group == 64 else 1152
    w, W, mag = _weight(n, k, group, dtype, hip_device, seed=m)
    x = _x(m, k, dtype, hip_device, n)
    y, err = _bounds(x, W, mag)
    _check(linear4(x, w), y, err, dtype)
    if n % 32 == 0:
        x = x / float(y.std())  # gates of a spread of 1
        y, err = _bounds(x, W, mag)
        (g, u), (eg, eu) = y.chunk(2, -1), err.chunk(2, -1)
        silu = g * torch.sigmoid(g)
        es = 1.1 * eg + 2.0**-20 * silu.abs()
        _check(linear4_silu_mul(x, w), silu * u, es * u.abs() + (silu.abs() + es) * eu, dtype)


@pytest.mark.parametrize("m,n,k", [(24, 1024, 12288), (40, 512, 8320), (64, 4096, 14336), (100, 1000, 4224), (300, 1024, 8192)])
def test_split_products(hip_device, m, n, k):
    """k over several workgroups."""
    w, W, mag = _weight(n, k, 64, torch.bfloat16, hip_device, seed=m)
    x = _x(m, k, torch.bfloat16, hip_device, n)
    _check(linear4(x, w), *_bounds(x, W, mag), torch.bfloat16)
