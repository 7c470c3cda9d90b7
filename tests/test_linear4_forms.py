"""The rule that cuts a product with a 4-bit weight (csrc/linear4.h), compiled for the host: what its comment says of it."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "kvserve_amd/csrc"

SOURCE = """
#include "linear4.h"
using namespace kvh;
extern "C" void form(int64_t tiles, int64_t blocks, int64_t m, int glu, int* o) {
  const Linear4Form f = linear4_form(tiles, blocks, m, glu);
  o[0] = f.rows, o[1] = f.rt, o[2] = f.wr, o[3] = f.wk, o[4] = f.s, o[5] = linear4_lds(f);
}
"""


@pytest.fixture(scope="module")
def form(tmp_path_factory):
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

    return form


@pytest.mark.parametrize("m", [1, 8, 16])
@pytest.mark.parametrize("glu", [0, 1])
def test_few_rows_take_one_round(form, m, glu):
    """Up to 2048 weight tiles (two groups of two tiles, two workgroups a CU) no workgroup waits for another's CU."""
    for blocks in (4, 32, 112):
        for tiles in (*range(2, 530, 2), *range(530, 2049, 14), 2048):
            rows, rt, wr, _, _, lds = form(tiles, blocks, m, glu)
            assert -(-tiles // (rt * wr)) <= 256 * (160 * 1024 // lds), (tiles, blocks)


def test_four_groups_up_to_a_round(form):
    """Plain and gated, the form that was the faster one, and where the rule passes from one to the other."""
    two, four = (16, 2, 2, 4, 2), (16, 2, 4, 4, 2)
    for tiles, glu, want in ((1024, 0, two), (1026, 0, four), (1280, 0, four), (1536, 0, four), (1538, 0, two), (1792, 0, two), (2048, 0, two),
                             (1024, 1, two), (1026, 1, four), (1792, 1, four), (1796, 1, four), (2048, 1, four), (2050, 1, two)):  # fmt: skip
        assert form(tiles, 32, 8, glu)[:5] == want, (tiles, glu)
