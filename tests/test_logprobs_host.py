"""token_logprobs without a GPU: every refusal of the C entry point and of the method (before any HIP call), and the
workspace's size."""

from __future__ import annotations

from pathlib import Path

import pytest
import torch

from kvserve_amd import _lib, token_logprobs
from kvserve_amd.logprobs import MAX_TOP

P = 0x10000
NULL, SHAPE, DTYPE, ALIGN, UNSUP, WS = -1, -2, -3, -4, -5, -6


def _call(**over):
    a = {"x": P, "rs": 1000, "tok": P, "lp": P, "ent": P, "tl": P, "ti": P, "rows": 4, "V": 1000, "top": 5, "dtype": 2,
         "ws": P, "wsb": 1 << 30}  # fmt: skip
    a.update(over)
    return _lib.load().kvh_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("over,want", [
    ({"dtype": 3}, DTYPE), ({"rows": -1}, SHAPE), ({"V": 0}, SHAPE), ({"top": -1}, SHAPE), ({"top": 1001}, SHAPE),
    ({"top": 65}, UNSUP), ({"rows": 1 << 30}, UNSUP), ({"V": 1 << 30}, UNSUP), ({"rows": 0}, 0), ({"x": None}, NULL),
    ({"rows": 0, "x": None}, 0), ({"tok": None}, NULL), ({"lp": None}, NULL), ({"ent": None}, NULL), ({"tl": None}, NULL),
    ({"ti": None}, NULL), ({"rs": -1}, SHAPE), ({"x": P + 1}, ALIGN), ({"x": P + 2, "dtype": 0}, ALIGN), ({"tok": P + 4}, ALIGN),
    ({"ti": P + 4}, ALIGN), ({"ent": P + 2}, ALIGN), ({"V": 128256, "rs": 128256, "ws": None}, WS),
    ({"V": 128256, "rs": 128256, "wsb": 100}, WS), ({"V": 128256, "rs": 128256, "ws": P + 8}, WS),
])  # fmt: skip
def test_refusals(over, want):
    assert _call(**over) == want


def test_more_rows_than_a_launch_has_threads_for():
    """A launch holds fewer than 2^32 threads, a workgroup of 256 for each row."""
    most = (2**32 - 1) // 256
    assert _call(rows=most + 1) == UNSUP and _call(rows=most, x=None) == NULL


def test_workspace_size():
    f = _lib.load().kvh_token_logprobs_workspace_size
    assert f(4, 1000, 5, 2) == 0 and f(300, 128256, 5, 2) == 0  # one segment a row
    assert f(4096, 128256, 20, 2) == 0
    assert f(8, 128256, 5, 2) == 8 * 32 * (16 + 5 * 8)
    assert f(100, 128256, 20, 2) == 100 * 5 * (16 + 20 * 8)  # 512 workgroups in all
    assert f(8, 20000, 5, 0) == 8 * 20 * (16 + 5 * 8)  # chunks of 1024 fp32 logits
    assert f(8, 128256, 65, 2) == 0 and f(-1, 10, 1, 2) == 0  # refused anyway


def test_method_refusals():
    x = torch.zeros(3, 100)
    with pytest.raises(ValueError, match="HIP device"):
        token_logprobs(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="contiguous last dim"):
        token_logprobs(x.t(), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="contiguous last dim"):
        token_logprobs(x[0], torch.zeros(3, dtype=torch.long))


def test_the_method_and_the_header_agree_on_the_alternatives():
    header = (Path(__file__).resolve().parents[1] / "include" / "kvhip.h").read_text()
    assert f"#define KVH_LOGPROBS_MAX_TOP {MAX_TOP}\n" in header
    assert _call(V=1000, top=MAX_TOP + 1) == UNSUP
