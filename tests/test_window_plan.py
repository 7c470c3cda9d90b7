"""The prefill part's positions under a sliding window (csrc/prefill_plan.h), compiled for the host and compared with
the definition tile by tile, and the C ABI's refusals of window arguments, which need no GPU."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from kvserve_amd import _lib

CSRC = Path(__file__).resolve().parent.parent / "kvserve_amd/csrc"

SOURCE = """
#define KVH_PLAN_FN static inline
#include "prefill_plan.h"
using namespace kvh;
extern "C" {
int skip(int R, int q, int kv, int64_t ctx, int G, int PR, int W, int S, int t) { return pre_tile_skip({R, q, kv, ctx}, G, PR, W, S, t); }
int64_t skips(int R, int q, int kv, int64_t ctx, int G, int PR, int W, int S, int t) { return pre_skips({R, q, kv, ctx}, G, PR, W, S, t); }
int chunks(int R, int q, int kv, int64_t ctx, int G, int PR, int W, int S, int t) {
  return kTileCost + pre_tile_chunks({R, q, kv, ctx}, G, PR, t) - pre_tile_skip({R, q, kv, ctx}, G, PR, W, S, t);
}
int full_tile(int G, int PR, int W, int S) { return pre_full_tile(G, PR, W, S); }
int whole_tiles(int64_t C, int64_t units, int64_t all, int tile) { return pre_whole_tiles(C, units, all, tile); }
int window_nt(int64_t rows, int64_t seqs, int Hkv, int G, int W, int S, int64_t units) {
  return pre_window_nt(rows, seqs, Hkv, G, W, S, units);
}
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    out = d / "plan.so"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(out)],
                   check=True)  # fmt: skip
    lib = ctypes.CDLL(str(out))
    i, l = ctypes.c_int, ctypes.c_int64
    lib.skip.argtypes = lib.skips.argtypes = [i, i, i, l, i, i, i, i, i]
    lib.skips.restype = l
    lib.chunks.argtypes = lib.skip.argtypes
    lib.whole_tiles.argtypes = [l, l, l, i]
    lib.window_nt.argtypes = [l, l, i, i, i, i, l]
    return lib


@pytest.mark.parametrize("PR,G", [(128, 4), (192, 4), (192, 1), (128, 7), (192, 64)])
def test_whole_tiles_are_shared_out_once(plan, PR, G):
    """Units that take the tiles whose middle lies in their range take every tile once, none more than a round above the
    mean; and no tile is longer than the one the rule counts with."""
    rng = random.Random(PR + G)
    for _ in range(40):
        W, S = rng.randint(1, 3000), rng.choice([0, 0, 1, 33, 200])
        full = plan.full_tile(G, PR, W, S)
        sizes = []
        for _ in range(rng.randint(1, 5)):
            q, ctx = rng.randint(1, 3000), rng.choice([0, rng.randint(0, 9000)])
            R = q * G
            sizes += [plan.chunks(R, q, q + ctx, ctx, G, PR, W, S, t) for t in range(-(-R // PR))] * rng.randint(1, 8)
        assert max(sizes) <= full
        C, units = sum(sizes), rng.randint(1, 512)
        units = min(units, -(-C // 2))
        owner, x = [], 0
        for tw in sizes:
            mid = x + tw // 2
            owner.append(((mid + 1) * units - 1) // C)  # the unit u with u C / units <= mid < (u + 1) C / units
            assert owner[-1] * C // units <= mid < (owner[-1] + 1) * C // units
            x += tw
        load = [0] * units
        for u, tw in zip(owner, sizes):
            load[u] += tw
        assert max(load) <= C // units + 1 + full
        left = C // units % full
        assert bool(plan.whole_tiles(C, units, 512, full)) == (left == 0 or (full - left) * 512 <= 26 * units)


def test_tiles_a_wave(plan):
    """Two where that fills the launch better: the measured cases of 32 heads over 8 on 512 units."""
    for q, seqs, W, S, want in ((8191, 1, 1024, 0, 3), (8191, 1, 4096, 0, 3), (4096, 1, 1024, 0, 2), (2000, 1, 512, 0, 2),
                                (3000, 1, 512, 0, 3), (12000, 1, 1024, 0, 3), (1900, 2, 2048, 64, 2), (200, 1, 1024, 0, 2)):  # fmt: skip
        assert plan.window_nt(4 * q, seqs, 8, 4, W, S, 512) == want
    for args in ((0, 0, 1, 1, 1, 0, 8), (1, 1, 1, 64, 2**31 - 1, 0, 512), (2**40, 65535, 128, 64, 2**30, 2**30, 512)):
        assert plan.window_nt(*args) in (2, 3)


@pytest.mark.parametrize("PR", [128, 192])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 7, 8, 16, 48, 63, 64])
def test_skipped_chunks(plan, G, PR):
    rng = random.Random(G * 1000 + PR)
    shapes = [(q, c, q + c) for q in (1, 5, PR // G + 1, 700) for c in (0, 1, 31, 4095)]
    shapes += [(rng.randint(1, 1500), rng.randint(0, 20000), None) for _ in range(10)]
    shapes += [(300, -100, 200), (300, 500, 640), (64, -64, 0), (40000 // G, 2**31 - 50000, None)]
    for q, ctx, kv in shapes:
        kv = q + ctx if kv is None else kv
        R = q * G
        tiles = -(-R // PR)
        for W, S in [(1, 0), (32, 0), (33, 1), (rng.randint(1, 3000), rng.randint(0, 300)), (2**31 - 1, 0), (5, 2**30)]:
            args = (R, q, kv, ctx, G, PR, W, S)
            total = 0
            for t in range(tiles):
                keys = min(max(ctx + PR * t // G + 1, 0), kv)
                # chunks behind the sinks' that end at or before the first row's first key
                n = max(0, max(0, keys - W) // 32 - -(-S // 32))
                assert plan.skip(*args, t) == n, (args, t)
                last = min(PR * t + PR - 1, R - 1)
                chunks = max(1, -(-min(max(ctx + last // G + 1, 0), kv) // 32))
                assert n < chunks  # a tile keeps one
                if t % 7 == 0 or t < 12:
                    assert plan.skips(*args, t) == total, (args, t)
                total += n
            assert plan.skips(*args, tiles) == total


def _call(**kw):
    """kvh_paged_attention_window with no memory behind it: only what is refused before the pointers are looked at."""
    a = {"W": 8, "bs": 16, "window": 8, "sinks": 0, "fmt": 0, "dtype": 2}
    a.update(kw)
    st = _lib.i64x3((1, 1, 1))
    return _lib.load().kvh_paged_attention_window(
        None, 8, 8, None, st, None, None, None, st, None, None, 4, None, 8, 8, None, a["W"], a["W"], None, None, 1, 1, 8, 2,
        64, a["bs"], 1, a["window"], a["sinks"], 1.0, a["fmt"], 1.0, 1.0, a["dtype"], None, 0, None,
    )  # fmt: skip


def test_refusals_of_the_c_abi():
    null, shape, dtype, unsupported = -1, -2, -3, -5
    assert _call() == null
    assert _call(window=0) == shape and _call(window=-7) == shape and _call(sinks=-1) == shape
    assert _call(fmt=3) == dtype and _call(fmt=-1) == dtype and _call(dtype=5) == dtype
    assert _call(W=0) == shape and _call(bs=0) == shape
    assert _call(W=(2**31 - 32) // 16, bs=16) == unsupported  # positions, rounded up to chunks, within 31 bits
    assert _call(window=2**31 - 1, sinks=2**31 - 1) == null  # sums in 64 bits
