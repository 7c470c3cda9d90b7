"""Windowed prompts whose units take whole tiles (csrc/prefill_plan.h, compiled for the host): every unit walked as the
kernels walk it takes each tile once, and the rule takes whole tiles where the longest unit's are no longer than splitting."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from tests.test_hip_window import Batch

CSRC = Path(__file__).resolve().parent.parent / "kvserve_amd/csrc"

SOURCE = """
#define KVH_PLAN_FN static inline
#include "prefill_plan.h"
using namespace kvh;
extern "C" {
int split_cost() { return kSplitCost; }
int chunks(int q, int kv, int64_t ctx, int G, int PR, int W, int S, int t) {
  const PreSeq s{q * G, q, kv, ctx};
  return kTileCost + pre_tile_chunks(s, G, PR, t) - pre_tile_skip(s, G, PR, W, S, t);
}
int full_tile(int G, int PR, int W, int S) { return pre_full_tile(G, PR, W, S); }
int whole_tiles(int64_t C, int64_t tiles, int64_t units, int64_t all, int tile) { return pre_whole_tiles(C, tiles, units, all, tile); }
int turn(int64_t beg, int64_t tw, int64_t x, int64_t x1) { return pre_tile_turn(beg, tw, x, x1); }
}
"""
SKIP, TAKE, END = range(3)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan.so")],
                   check=True)  # fmt: skip
    lib = ctypes.CDLL(str(d / "plan.so"))
    i, l = ctypes.c_int, ctypes.c_int64
    lib.chunks.argtypes = [i, i, l, i, i, i, i, i]
    lib.whole_tiles.argtypes = [l, l, l, l, i]
    lib.turn.argtypes = [l, l, l, l]
    return lib


def _walk(plan, sizes, units) -> list[list[int]]:
    """The tiles that each unit takes. Unit u stands at u C / units, inside a tile or at its start."""
    C, starts, x = sum(sizes), [], 0
    for tw in sizes:
        starts.append(x)
        x += tw
    taken, t0 = [], 0
    for u in range(units):
        x, x1 = u * C // units, (u + 1) * C // units
        while t0 + 1 < len(sizes) and starts[t0 + 1] <= x:
            t0 += 1
        mine, t = [], t0
        while True:
            turn = plan.turn(starts[t], sizes[t], x, x1)
            if turn == END:
                break
            if turn == TAKE:
                mine.append(t)
            x = starts[t] + sizes[t]
            if x >= x1:
                break
            t += 1
        taken.append(mine)
    return taken


def _sizes(plan, seqs, G, kv_heads, PR, W, S):
    sizes = []
    for q, ctx in seqs:
        sizes += [plan.chunks(q, q + ctx, ctx, G, PR, W, S, t) for t in range(-(-q * G // PR))] * kv_heads
    return sizes


@pytest.mark.parametrize("PR,G", [(128, 4), (192, 4), (192, 1), (128, 7), (192, 64)])
def test_units_take_every_tile_once(plan, PR, G):
    rng = random.Random(PR * G)
    for _ in range(25):
        W, S = rng.randint(1, 3000), rng.choice([0, 0, 1, 33, 200])
        seqs = [(rng.randint(1, 3000), rng.choice([0, rng.randint(0, 9000)])) for _ in range(rng.randint(1, 5))]
        sizes = _sizes(plan, seqs, G, rng.randint(1, 8), PR, W, S)
        units = min(rng.randint(1, 768), -(-sum(sizes) // 2))
        taken = _walk(plan, sizes, units)
        assert [t for mine in taken for t in mine] == list(range(len(sizes)))  # in order, none twice, none left


def _longest(plan, q, seqs, W, nt, G=4, kv_heads=8, all_units=512):
    """(whether the units take whole tiles, the longest unit then, positions of a unit that splits, with its pieces' cost)"""
    PR = 64 * nt
    sizes = _sizes(plan, [(q, 0)] * seqs, G, kv_heads, PR, W, 0)
    C, full = sum(sizes), plan.full_tile(G, PR, W, 0)
    units = min(all_units, -(-C // 2))
    longest = max(sum(sizes[t] for t in mine) for mine in _walk(plan, sizes, units))
    whole = bool(plan.whole_tiles(C, len(sizes), units, all_units, full))
    return whole, longest, C / units + plan.split_cost() * units / all_units


@pytest.mark.parametrize("nt", [2, 3])
@pytest.mark.parametrize("W", [512, 1024, 2048, 4096])
def test_longest_unit(plan, W, nt):
    """Prompts of half a window to four: where the units take whole tiles, the longest one's are at most 1.3 times what a unit
    would have by splitting (two units share a CU, which evens out as much)."""
    for part in (50, 62, 75, 90, 100, 112, 122, 135, 150, 170, 195, 230, 268, 300, 400):
        for seqs in (1, 2, 3, 5, 9):
            whole, longest, split = _longest(plan, W * part // 100, seqs, W, nt)
            assert not whole or longest <= 1.3 * split, (part, seqs, longest, split)


def test_measured(plan):
    """(prompt, prompts, window, row tiles a wave): which was faster."""
    for q, seqs, W, nt, want in ((4600, 1, 4096, 3, False), (5000, 1, 4096, 3, False), (8000, 1, 4096, 3, False), (2500, 1, 2048, 3, False),
                                 (2000, 3, 2048, 3, False), (2000, 2, 2048, 2, False), (3500, 1, 2048, 2, False),
                                 (2000, 1, 1024, 3, True), (4000, 3, 4096, 3, False), (3500, 3, 2048, 3, True), (3000, 4, 2048, 3, True), (5000, 4, 4096, 3, True),
                                 (1000, 8, 1024, 3, True), (500, 8, 512, 3, True), (2000, 4, 512, 2, True),
                                 (8191, 1, 1024, 3, True), (12000, 1, 1024, 3, True), (3000, 1, 512, 3, True), (8191, 1, 2048, 3, False)):  # fmt: skip
        assert _longest(plan, q, seqs, W, nt)[0] == want, (q, seqs, W, nt)


def test_ranges_a_little_longer_than_a_round(plan):
    """C / units = 135.6 positions of tiles of 135: some units are left with two."""
    assert plan.whole_tiles(512 * 135, 512, 512, 512, 135)
    assert not plan.whole_tiles(512 * 135 + 300, 514, 512, 512, 135)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,ctx,window", [([1250], [0], 1024), ([2600], [0], 2048), ([700, 700, 700], [0, 0, 0], 640),
                                               ([40] * 300 + [1] * 20, [0, 300, 90] * 100 + [500] * 20, 64)])  # fmt: skip
def test_prompts_of_few_windows(hip_device, q_lens, ctx, window):
    """Shorter first tiles on the GPU, split and whole, and more sequences than the plan has threads."""
    batch = Batch(hip_device, q_lens, ctx, 16, 4, 128, 16, window, 0)
    batch.check(batch.forward())
