"""The MXFP4 cache without a GPU: the oracle's format against the bits' meaning, the allocation helper, and every
refusal of the C entry points and of HipAttention's methods (they return before any HIP call)."""

from __future__ import annotations

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kvserve_amd import HipAttention, _lib, fp4_caches
from kvserve_amd.attention import AttentionMetadata
from oracle import fp4

ROOT = Path(__file__).resolve().parents[1]


# -- the oracle ------------------------------------------------------------------------------------
def test_magnitudes_are_the_formats():
    assert fp4.MAGNITUDES.tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert [fp4.e2m1_value(c) for c in (8, 9, 15)] == [0, -0.5, -6] and math.copysign(1, fp4.e2m1_value(8)) == -1


def _block(*values: float, dtype=torch.float32) -> torch.Tensor:
    x = torch.zeros(32, dtype=dtype)
    x[: len(values)] = torch.tensor(values, dtype=dtype)
    return x


@pytest.mark.parametrize(
    "values,scale,stored",
    [
        # a mantissa under 1.75 keeps the exponent, 1.75 takes the next
        ((6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), 127, (6, 0, 1, 1, 2, 2, 4, 4)),  # ties to the even code
        ((6.9375, 0.26, 0.74, 1.26, 1.74, 2.51, 3.49, 5.01), 127, (6, 0.5, 0.5, 1.5, 1.5, 3, 3, 6)),
        ((7.0, 1.0, -3.0), 128, (8, 1, -3)),  # 7 / 2 = 3.5, a tie; -3 / 2 = -1.5
        ((4.0, -0.0), 127, (4, -0.0)),
        ((8.0, 0.5, 0.49), 128, (8, 0, 0)),
        ((0.0,), 2, (0,)),
        ((2.0**-126,), 2, (2.0**-126,)),  # scale 2 is 2^-125: half of it
    ],
)
def test_quantize_known_answers(values, scale, stored):
    code, s = fp4.quantize(_block(*values))
    assert s.tolist() == [scale]
    got = fp4.dequantize(code, s)
    assert got[: len(stored)].tolist() == list(stored)
    assert torch.signbit(got[1]) == (math.copysign(1, (*stored, 0)[1]) < 0)


def test_quantize_ends_of_the_types():
    for dtype, top in ((torch.float16, 49152.0), (torch.bfloat16, 1.5 * 2.0**127), (torch.float32, 1.5 * 2.0**127)):
        x = _block(float("inf"), -float("inf"), torch.finfo(dtype).max, 1.0, dtype=dtype)
        got = fp4.dequantize(*fp4.quantize(x))
        assert got[:3].tolist() == [top, -top, top]
        assert torch.isfinite(got.to(dtype)).all()
        x[7] = float("nan")
        assert fp4.dequantize(*fp4.quantize(x)).isnan().all()


def test_quantize_is_off_by_half_a_step_at_most():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4000, 32, generator=g).double() * torch.exp2(torch.randn(4000, 1, generator=g) * 8)
    code, s = fp4.quantize(x, torch.float32)
    y = (x / torch.exp2(s.double() - 127)).abs()
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    off = (fp4.dequantize(code, s) - x).abs() / torch.exp2(s.double() - 127)
    assert (off <= step / 2).all() and y.max() < 7


# -- allocation ------------------------------------------------------------------------------------
def test_fp4_caches_hold_a_heads_tokens_together():
    k, v, ks, vs = fp4_caches(5, 16, 8, 128, "cpu")
    assert k.shape == v.shape == (5, 16, 8, 64) and ks.shape == vs.shape == (5, 16, 8, 4)
    assert k.dtype == fp4.FP4 and ks.dtype == fp4.E8M0
    assert k.stride() == (8 * 16 * 64, 64, 16 * 64, 1) and ks.stride() == (8 * 16 * 4, 4, 16 * 4, 1)
    for bad in (0, 48, 33):
        with pytest.raises(ValueError, match="head sizes"):
            fp4_caches(5, 16, 8, bad, "cpu")


# -- refusals of the C entry points ----------------------------------------------------------------
P = 0x10000  # an aligned address that no call here may reach
ST = {"c": (8192, 64, 1024), "x": (512, 4, 64)}


def _caches(**over):
    a = {"k_cache": P, "kst": ST["c"], "k_scale": P, "kxst": ST["x"], "v_cache": P, "vst": ST["c"], "v_scale": P,
         "vxst": ST["x"]}  # fmt: skip
    a.update({n: over.pop(n) for n in list(over) if n in a})
    return [x if n in ("k_cache", "k_scale", "v_cache", "v_scale") else (_lib.i64x3(x) if x else None)
            for n, x in a.items()], over  # fmt: skip


def _write(**over):
    c, over = _caches(**over)
    a = {"k": P, "kt": 1024, "kh": 128, "v": P, "vt": 1024, "vh": 128, "slots": P, "T": 4, "nb": 10, "hkv": 8, "D": 128,
         "bs": 16, "dtype": 2}  # fmt: skip
    a.update(over)
    return _lib.load().kvh_reshape_and_cache_fp4(*list(a.values())[:6], *c, *list(a.values())[6:], None)


def _rope(**over):
    c, over = _caches(**over)
    a = {"qkv": P, "qt": 6144, "pos": P, "cos": P, "sin": P, "mp": 100, "q": P, "qot": 4096, "qoh": 128, "slots": P,
         "T": 4, "nb": 10, "H": 32, "hkv": 8, "D": 128, "bs": 16, "dtype": 2}  # fmt: skip
    a.update(over)
    return _lib.load().kvh_rope_and_cache_fp4(*list(a.values())[:9], *c, *list(a.values())[9:], None)


def _read(**over):
    c, over = _caches(**over)
    a = {"slots": P, "k": P, "kt": 1024, "kh": 128, "v": P, "vt": 1024, "vh": 128, "T": 4, "nb": 10, "hkv": 8, "D": 128,
         "bs": 16, "dtype": 2}  # fmt: skip
    a.update(over)
    return _lib.load().kvh_read_cache_fp4(*c, *a.values(), None)


def _attend(**over):
    c, over = _caches(**over)
    a = {"q": P, "qt": 4096, "qh": 128, "nb": 10, "out": P, "ot": 4096, "oh": 128, "bt": P, "bts": 200, "W": 200,
         "sl": P, "qsl": P, "T": 4, "B": 4, "H": 32, "hkv": 8, "D": 128, "bs": 16, "mq": 1, "scale": 0.1, "dtype": 2,
         "ws": None, "wsb": 0}  # fmt: skip
    a.update(over)
    v = list(a.values())
    return _lib.load().kvh_paged_attention_fp4(*v[:3], *c, *v[3:], None)


NULL, SHAPE, DTYPE, ALIGN, UNSUP, WS = -1, -2, -3, -4, -5, -6
COMMON = [
    ({"dtype": 3}, DTYPE), ({"dtype": -1}, DTYPE), ({"hkv": 0}, SHAPE), ({"bs": 0}, SHAPE), ({"T": -1}, SHAPE),
    ({"k_cache": None}, NULL), ({"v_scale": None}, NULL), ({"kxst": None}, NULL), ({"kst": (8192, -64, 1024)}, SHAPE),
    ({"kst": (8192, 66, 1024)}, ALIGN), ({"v_cache": P + 2}, ALIGN), ({"vxst": (512, -4, 64)}, SHAPE),
    ({"kst": (8192, 1 << 28, 1024)}, UNSUP), ({"vxst": (512, 1 << 28, 64)}, UNSUP),
]  # fmt: skip


@pytest.mark.parametrize("over,want", COMMON + [
    ({"D": 48}, UNSUP), ({"D": 1056}, UNSUP), ({"k": None}, NULL), ({"slots": None}, NULL), ({"kt": 1028}, ALIGN),
    ({"v": P + 8}, ALIGN), ({"vh": -8}, SHAPE), ({"T": 0}, 0), ({"T": 0, "k": None, "k_cache": None}, 0),
])  # fmt: skip
def test_write_and_read_refusals(over, want):
    assert _write(**dict(over)) == want
    assert _read(**dict(over)) == want


@pytest.mark.parametrize("over,want", COMMON + [
    ({"D": 96}, UNSUP), ({"D": 32}, UNSUP), ({"H": 0}, SHAPE), ({"mp": 0}, SHAPE), ({"qkv": None}, NULL),
    ({"pos": None}, NULL), ({"cos": P + 4}, ALIGN), ({"qt": 6136}, SHAPE), ({"q": P + 4}, ALIGN), ({"qoh": 132}, ALIGN),
    ({"T": 0}, 0),
])  # fmt: skip
def test_rope_refusals(over, want):
    assert _rope(**dict(over)) == want


@pytest.mark.parametrize("over,want", COMMON + [
    ({"dtype": 0}, UNSUP), ({"D": 96}, UNSUP), ({"D": 256}, UNSUP), ({"bs": 8}, UNSUP), ({"bs": 24}, UNSUP),
    ({"H": 33}, SHAPE), ({"q": None}, NULL), ({"out": P + 8}, ALIGN), ({"qt": 4100}, ALIGN), ({"nb": 0}, SHAPE),
    ({"bts": 199}, SHAPE), ({"kst": (8192, 72, 1024)}, ALIGN), ({"k_cache": P + 8}, ALIGN), ({"ws": None}, WS),
    ({"ws": P, "wsb": 100}, WS), ({"T": 0}, 0), ({"B": 0}, 0),
])  # fmt: skip
def test_attention_refusals(over, want):
    assert _attend(**dict(over)) == want


def test_more_tokens_than_a_launch_has_threads_for():
    """A launch holds fewer than 2^32 threads: a workgroup of 256 takes 4 tokens of a write or read, 1 of a rotation."""
    most = (2**32 - 1) // 256
    assert _write(T=4 * most + 1) == SHAPE and _read(T=4 * most + 1) == SHAPE and _rope(T=most + 1) == SHAPE
    assert _write(T=4 * most, k=None) == NULL and _rope(T=most, pos=None) == NULL


# -- refusals of the methods (CPU tensors never reach a kernel) -------------------------------------
def test_methods_refuse_what_is_no_4bit_cache():
    k, v, ks, vs = fp4_caches(4, 16, 2, 64, "cpu")
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.arange(3)
    for bad in ({"k_scale": 1.0}, {"v_scale": ks.view(torch.uint8)}, {}):
        with pytest.raises(ValueError, match="float8_e8m0fnu"):
            HipAttention.write_kv(k, v, rows, rows, slots, **bad)
    with pytest.raises(ValueError, match="dtypes differ"):
        HipAttention.write_kv(k, rows, rows, rows, slots, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="HIP device"):
        HipAttention.write_kv(k, v, rows, rows, slots, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="read_kv reads"):
        HipAttention.read_kv(rows[None], rows[None], slots, torch.float32, ks, vs)
    with pytest.raises(ValueError, match="gemv_rope_and_cache"):
        HipAttention.gemv_rope_and_cache(rows[:, 0], rows[0], slots, rows, rows, k, v, slots, 2, k_scale=ks, v_scale=vs)
    meta = AttentionMetadata(slots, slots[None], slots[:1], slots[:1], slots[:2], 3, 1)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        HipAttention.forward(rows, k, v, meta, 1.0)


def test_abi_takes_the_strides_as_they_are():
    a = _lib.i64x3(fp4_caches(4, 16, 2, 64, "cpu")[0].stride()[:3])
    assert isinstance(a, ctypes.Array) and list(a) == [1024, 32, 512]


def test_a_pytorch_without_the_dtypes_still_imports():
    code = ("import torch; del torch.float4_e2m1fn_x2, torch.float8_e8m0fnu\n"
            "import kvserve_amd, kvserve_amd.engine\n"
            "try: kvserve_amd.fp4_caches(1, 16, 1, 64, 'cpu')\n"
            "except ValueError as e: print(e)")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and "no float4_e2m1fn_x2" in r.stdout, r.stderr
