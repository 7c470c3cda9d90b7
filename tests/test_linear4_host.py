"""4-bit weights without a GPU: the packing's round trip, the rounding of quantize_weight4, and refusals."""

from __future__ import annotations

import ctypes
import random
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from kvserve_amd import Weight4, _lib, linear4, quantize_weight4


def _parts(n=20, k=192, group=64, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(n)
    q = torch.randint(0, 16, (n, k), generator=g)
    s = torch.rand((n, k // group), generator=g).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    return q, (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8), s, z


@pytest.mark.parametrize("n,k,group", [(20, 192, 64), (16, 128, 128), (1, 32, 32), (33, 1184, 32), (1100, 256, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_packed_layout(n, k, group, dtype):
    """Every element at the place that kvh_linear4 documents, and back."""
    q, codes, s, z = _parts(n, k, group, dtype)
    w = Weight4.pack(codes, s, z)
    assert w.shape == (n, k) and w.group == group and w.dtype == dtype
    rep = lambda t: t.double().repeat_interleave(group, 1)  # noqa: E731
    assert torch.equal(w.dequantize(torch.float64), rep(s) * (q - rep(z)))
    flat, pairs = w.codes.view(w.codes.shape[0], -1, 4, 16, 4), w.scales
    for r, c in [(0, 0), (n - 1, k - 1), (n // 2, k // 2), (0, min(k - 1, 37)), (n - 1, 9)]:
        b, u, j, i = c // 128, c % 128 // 32, c % 32 // 8, c % 8
        dword = int(flat[r // 16, b, j, r % 16, u]) & 0xFFFFFFFF
        assert (dword >> (4 * (i // 2) + 16 * (i % 2))) & 15 == int(q[r, c])
        pair = pairs[r // 16, c // group, r % 16 : r % 16 + 1].view(dtype)
        assert pair[0] == s[r, c // group] and int(pair[1]) == 16 + int(z[r, c // group])
    assert not pairs[:, k // group :].any()


def test_no_zero_points_means_eight():
    _, codes, s, _ = _parts()
    a, b = Weight4.pack(codes, s), Weight4.pack(codes, s, torch.full(s.shape, 8, dtype=torch.uint8))
    assert torch.equal(a.scales, b.scales) and torch.equal(a.codes, b.codes)


def test_quantize_weight4():
    g = torch.Generator().manual_seed(2)
    W = torch.randn((40, 256), generator=g).half()
    W[0] = 0
    W[1] = 3.0
    back = quantize_weight4(W, 32).dequantize(torch.float64)
    grp = W.double().unflatten(1, (-1, 32))
    step = (grp.amax(-1).clamp(min=0) - grp.amin(-1).clamp(max=0)) / 15
    assert ((back - W.double()).abs().unflatten(1, (-1, 32)) <= (1.0 + 15 * 2.0**-11) * step[..., None] + 1e-12).all()
    assert not back[0].any() and (back[1] - 3.0).abs().max() < 0.01


def test_refusals():
    _, codes, s, z = _parts()
    for bad in ((codes.int(), s, z), (codes, s.float(), z), (codes[:-1], s, z), (codes, s[:, :2], z), (codes, s, z[:, :2]),
                (codes, s, z.int()), (codes, s, z + 16), (codes[:, :50], s, z), (codes, s[:, :1], z[:, :1])):  # fmt: skip
        with pytest.raises(ValueError):
            Weight4.pack(*bad)
    for W, group in ((torch.zeros(4, 96), 32), (torch.zeros(4, 96).half(), 64), (torch.zeros(4, 96).half(), 48), (torch.zeros(96).half(), 32)):
        with pytest.raises(ValueError):
            quantize_weight4(W, group)
    w = Weight4.pack(codes, s, z)
    for bad in ((w.codes[:1], w.scales, w.shape, 64), (w.codes, w.scales, w.shape, 32), (w.codes.long(), w.scales, w.shape, 64),
                (w.codes, w.scales.transpose(0, 1), w.shape, 64), (w.codes, w.scales, (20, 190), 64)):  # fmt: skip
        with pytest.raises(ValueError):
            Weight4(*bad, torch.bfloat16)
    with pytest.raises(ValueError):  # no CPU form
        linear4(torch.zeros(2, 192).bfloat16(), Weight4.pack(codes, s, z))


def _call(m=1, n=16, k=128, group=128, silu=0, dtype=2, xs=128, ys=16, x=None, y=None):
    return _lib.load().kvh_linear4(x, xs, x, x, y, ys, m, n, k, group, silu, dtype, None, 0, None)


def test_refusals_of_the_c_abi():
    null, shape, dtype, align, unsupported, workspace = -1, -2, -3, -4, -5, -6
    assert _call() == null
    assert _call(m=0) == 0 and _call(n=0) == 0
    assert _call(dtype=0) == dtype and _call(dtype=3) == dtype
    assert _call(m=-1) == shape and _call(n=-1) == shape and _call(k=0) == shape
    assert _call(group=48) == unsupported and _call(k=192) == unsupported and _call(m=16 * 65535 + 1) == unsupported
    assert _call(silu=1) == unsupported and _call(n=0x7FFFFFFF) == unsupported and _call(n=2**28 + 1) == unsupported
    # refused before anything is launched: addresses that are never read
    assert _call(x=16, y=16, xs=127) == shape and _call(x=16, y=16, ys=15) == shape
    assert _call(x=16, y=16, m=64, n=1024, k=8192, xs=8192, ys=1024) == workspace
    assert _call(x=16, y=16, xs=132) == align and _call(x=24, y=16) == align and _call(x=16, y=17) == align


CSRC = Path(__file__).resolve().parent.parent / "kvserve_amd/csrc"

SOURCE = """
#include "linear4.h"
using namespace kvh;
extern "C" int lds(int rows, int rt, int wr, int wk, int s) { return linear4_lds(Linear4Form{rows, rt, wr, wk, s, 1}); }
extern "C" void form(int64_t tiles, int64_t blocks, int64_t m, int glu, int* o) {
  const Linear4Form f = linear4_form(tiles, blocks, m, glu);
  o[0] = f.rows, o[1] = f.rt, o[2] = f.wr, o[3] = f.wk, o[4] = f.s, o[5] = f.splits;
}
"""


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("forms")
    (d / "forms.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "forms.cpp"), "-o", str(d / "forms.so")],
                   check=True)  # fmt: skip
    lib = ctypes.CDLL(str(d / "forms.so"))
    lib.form.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    lib.form.restype = None

    def form(tiles, blocks, m, glu=0):
        o = (ctypes.c_int * 6)()
        lib.form(tiles, blocks, m, glu, o)
        return tuple(o)

    form.lds = lib.lds
    return form


def test_every_form_is_built_and_reached(forms):
    """The forms that the rule gives are those that the launcher has kernels of, within a workgroup's limits; a split has
    four chunks at least, and the workspace covers them."""
    src = (CSRC / "linear4.hip").read_text()
    plain, both = re.search(r"if constexpr \(!GLU\) \{(.*?)\}(.*?)#undef", src, re.S).groups()
    find = lambda t: {tuple(map(int, m)) for m in re.findall(r"KVH_FORM\((\d+), (\d+), (\d+), (\d+), (\d+)\)", t)}  # noqa: E731
    built = {0: find(plain) | find(both), 1: find(both)}
    assert built[1] and all(f[1] % 2 == 0 for f in built[1])
    rng = random.Random(3)
    span = lambda top: min(top, int(2 ** rng.uniform(0, top.bit_length())))  # noqa: E731
    seen = {0: set(), 1: set()}
    for _ in range(40000):
        tiles, blocks, m, glu = span(10000), span(300), span(4000), rng.randint(0, 1)
        if glu:
            tiles += tiles % 2
        *f, z = forms(tiles, blocks, m, glu)
        f = tuple(f)
        assert f in built[glu], (tiles, blocks, m, glu, f)
        seen[glu].add(f)
        rows, rt, wr, wk, s = f
        assert rows >= min(m, 64) and 64 * wr * wk <= 1024 and forms.lds(*f) <= 160 * 1024
        chunks = -(-blocks // (wk * s))
        assert z == 1 or 4 * z <= chunks
        assert -(-m // (16 * -(-rows // 16))) <= 65535 and z <= 65535
        n, k = 16 * tiles, 128 * blocks
        assert _lib.load().kvh_linear4_workspace_size(m, n, k, glu) == (z * m * tiles * 64 if z > 1 else 0)
    assert seen == built
