"""token_logprobs on the GPU against log_softmax in 64 bits and a stable sort.

The bound. s = sum e^(x - m) is a thread's sum over at most V / 256 + 16 entries of non-negative terms, each within
2^-21 + 2^-22 |x - m| of itself (difference, product, exponential in fp32), then joined in some 20 steps: relative error
at most r = (V / 256 + 64) 2^-24 + 2^-20 (the mean of |x - m| under the distribution is below 16 here). log p = x - m -
ln s is off by r and a rounding of each of its two parts: r + 2^-22 (|x - m| + |ln s|) <= r + 2^-22 (|log p| + 2 ln V).
The entropy ln s - t / s: by r (1 + |t / s|) and roundings: r (2 + |entropy| + ln V).
"""

from __future__ import annotations

import math

import pytest
import torch

from kvserve_amd import token_logprobs

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(logits, tokens, top, got=None):
    r = token_logprobs(logits, tokens, top) if got is None else got
    T, V = logits.shape
    x = logits.double()
    lp = torch.log_softmax(x, dim=-1)
    rel = (V / 256 + 64) * 2.0**-24 + 2.0**-20
    want = lp.gather(1, tokens[:, None]).squeeze(1)

    def close(a, b, bound):
        assert torch.equal(a.isnan(), b.isnan())
        b32 = b.float()  # what fp32 holds of it (the type's lowest value less its largest is -inf there)
        assert torch.equal(a.isinf(), b32.isinf()) and torch.equal(a[a.isinf()], b32[b32.isinf()])
        fine = b32.isfinite()
        assert ((a.double() - b).abs() <= bound)[fine].all(), ((a.double() - b).abs() - bound)[fine].max()

    close(r.logprobs, want, rel + 2.0**-22 * (want.abs() + 2 * math.log(V)))
    ent = -(lp.exp() * lp).masked_fill(lp == -math.inf, 0.0).sum(-1)
    close(r.entropy, ent, rel * (2 + ent.abs() + math.log(V)))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    ok = ~x.isnan().any(-1)
    assert r.top_ids.shape == r.top_logprobs.shape == (T, top)
    assert torch.equal(r.top_ids[ok], order[ok])
    best = lp.gather(1, order)[ok]
    close(r.top_logprobs[ok], best, rel + 2.0**-22 * (best.abs() + 2 * math.log(V)))
    return r


def _logits(T, V, dtype, dev, seed=0, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(T, V, generator=g, device=dev)).to(dtype), torch.randint(V, (T,), generator=g, device=dev)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (5, 64, 64), (2, 257, 20), (9, 1000, 5), (33, 2048, 64),
                                     (700, 5003, 3), (2500, 999, 20), (1, 128256, 20), (8, 128256, 5), (70, 128256, 64),
                                     (1100, 32001, 1), (3, 151937, 0)])  # fmt: skip
def test_sizes(hip_device, T, V, top, dtype):
    _check(*_logits(T, V, dtype, hip_device, seed=V), top)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [300, 1030, 2007, 2065, 4200, 128256])
def test_many_alternatives_of_short_segments(hip_device, V, dtype):
    """64 alternatives where a segment has hardly as many groups of threads: hundreds to two thousand entries are listed
    and thinned out. Rows at random, descending (ties in 16 bits), ascending and of one value; few and many rows."""
    x, tok = _logits(4, V, dtype, hip_device, seed=V)
    ramp = torch.arange(V, device=hip_device) * (20.0 / V)
    x[1], x[2], x[3] = (-ramp).to(dtype), ramp.to(dtype), 0.5
    _check(x, tok, 64)
    few = token_logprobs(x[:3], tok[:3], 64)
    many = token_logprobs(x.repeat(300, 1), tok.repeat(300), 64)
    assert torch.equal(many.top_ids[:3], few.top_ids) and torch.equal(many.top_ids[1188:1191], few.top_ids)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("skip,stride", [(0, 4099), (1, 4099), (3, 5001), (5, 4112), (8, 4104)])
def test_strides_and_alignments(hip_device, dtype, skip, stride):
    """Rows that begin at any element, more than a row apart: heads and tails of 0 .. 7 elements."""
    V = 4091
    wide, tok = _logits(40, stride + 8, dtype, hip_device, seed=stride)
    _check(wide[:, skip : skip + V], tok % V, 11)


def test_one_row_seen_many_times(hip_device):
    row, _ = _logits(1, 3001, torch.bfloat16, hip_device)
    _check(row.expand(50, -1), torch.arange(50, device=hip_device), 4)


@pytest.mark.parametrize("T", [2, 2100])
@pytest.mark.parametrize("offset", [-30000.0, 30000.0, -3e37, 3e37])
def test_far_from_zero(hip_device, T, offset):
    """Logits far from 0 (their differences are whole numbers, exact there): the reference cancels whatever its size."""
    x = torch.randint(-20, 20, (T, 3000), device=hip_device).float() * max(1.0, abs(offset) / 2**22)
    _check(x + offset, torch.arange(T, device=hip_device), 9)


@pytest.mark.parametrize("T", [2, 2100])
@pytest.mark.parametrize("V", [515, 40000])
def test_ties_go_to_the_lowest_id(hip_device, T, V):
    x, tok = _logits(T, V, torch.bfloat16, hip_device, seed=V)
    x = x.float().round().to(torch.bfloat16)  # a dozen values in all
    x[0] = 0.0  # all alike
    x[1] = -0.0
    x[1, 100::7] = 0.0  # equal to -0
    _check(x, tok, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,V", [(8, 128256), (2049, 600)])
def test_masked_vocabulary_and_special_rows(hip_device, dtype, T, V):
    x, tok = _logits(T, V, dtype, hip_device, seed=5)
    inf, nan = float("inf"), float("nan")
    x[0] = -inf
    x[0, [5, V // 2, V - 1]] = torch.tensor([1.0, 2.0, -1.0], dtype=dtype, device=hip_device)  # three can be
    tok[0] = V // 2
    x[1, ::2] = -inf
    tok[1] = 4  # cannot be: -inf
    x[2] = -inf  # nothing can be: NaN
    x[3, 17] = inf
    x[4, V - 2] = nan
    x[5] = -inf
    x[5, 9] = -60000.0  # certain
    tok[5] = 9
    x[6] = torch.finfo(dtype).min
    x[6, 3] = torch.finfo(dtype).max
    r = _check(x, tok, 20)
    assert r.logprobs[2].isnan() and r.logprobs[3].isnan() and r.logprobs[4].isnan()
    assert r.logprobs[1] == -inf
    # the one term is 2^delta taken back by 2^-delta, an ulp each: ln s within 2^-22 of 0, ln 2 t / s within as much
    assert r.logprobs[5].abs() <= 2.0**-22 and r.entropy[5].abs() <= 2.0**-21
    assert r.top_ids[2].tolist() == list(range(20))
    assert r.top_ids[0, :4].tolist() == [V // 2, 5, V - 1, 0] and (r.top_logprobs[0, 3:] == -inf).all()
    ids = r.top_ids[4]
    assert len(set(ids.tolist())) == 20 and ids.min() >= 0 and ids.max() < V


def test_nan_rows_alone(hip_device):
    x = torch.full((3, 4097), float("nan"), device=hip_device)
    x[1, 7] = 3.0
    r = token_logprobs(x, torch.zeros(3, dtype=torch.long, device=hip_device), 8)
    assert r.logprobs.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()
    assert r.top_ids[0].tolist() == list(range(8)) and r.top_ids[1].tolist() == [7, *range(7)]


@pytest.mark.parametrize("dtype,per", [(torch.bfloat16, 8), (torch.float32, 4)], ids=str)
@pytest.mark.parametrize("top", [2, 64])
def test_largest_in_few_threads(hip_device, dtype, per, top):
    """Thousands of the largest entries in the strides of eight threads, past what the list of candidates holds: a thread
    of a whole row's pass has elements 256 per i + per t .. of it."""
    V, T = 128256, 2048
    at = torch.arange(V, device=hip_device)
    own = at % (256 * per) < 8 * per
    row = torch.where(own, 1.0 + at / 1024, at % 7 / 8).to(dtype)[None]
    x, tok = row.expand(T, -1), at[-T:]  # every row the same memory, a segment each
    r = token_logprobs(x, tok, top)
    assert (r.top_ids == r.top_ids[0]).all() and (r.top_logprobs == r.top_logprobs[0]).all()
    _check(x[-2:], tok[-2:], top, type(r)(*(f[-2:] for f in r)))
    _check(x[:1], tok[:1], top)  # in 32 segments, none of which lists as many


def test_tokens_outside_the_vocabulary(hip_device):
    x, tok = _logits(4, 100, torch.float32, hip_device)
    tok[1], tok[2] = -1, 100
    r = token_logprobs(x, tok, 3)
    assert r.logprobs.isnan().tolist() == [False, True, True, False]
    assert not r.entropy.isnan().any() and not r.top_logprobs.isnan().any()


def test_empty_and_refused(hip_device):
    dev = hip_device
    r = token_logprobs(torch.zeros(0, 50, device=dev), torch.zeros(0, dtype=torch.long, device=dev), 4)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 4)
    x, tok = _logits(4, 100, torch.float32, dev)
    for bad, match in (((x, tok[:3]), "one token"), ((x, tok.int()), "int64"), ((x, tok.cpu()), "device"),
                       ((x, tok, 65), "top"), ((x[:, :10], tok, 11), "top"), ((x, tok, -1), "top"),
                       ((x.double(), tok), "dtype"), ((x, tok[:, None]), "1-d")):  # fmt: skip
        with pytest.raises(ValueError, match=match):
            token_logprobs(*bad)


def test_same_bits_every_time(hip_device):
    x, tok = _logits(300, 128256, torch.bfloat16, hip_device, seed=2)
    a = token_logprobs(x, tok, 20)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, token_logprobs(x, tok, 20)))


@pytest.mark.parametrize("T", [4, 2100])
def test_graph_replays(hip_device, T):
    """Captured (with and without the joining launch) and replayed over new logits, eager work between."""
    x, tok = _logits(T, 20000, torch.bfloat16, hip_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(x, tok, 5)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, tok, 5)
    for seed in range(1, 5):
        a, b = _logits(T, 20000, torch.bfloat16, hip_device, seed=seed)
        x.copy_(a)
        tok.copy_(b)
        graph.replay()
        got = [f.clone() for f in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, token_logprobs(x, tok, 5)))
        _check(x[:4], tok[:4], 5, type(out)(*(f[:4] for f in got)))


def test_step_by_step_path_gives_the_same_bits(hip_device, monkeypatch):
    from kvserve_amd import _lib

    x, tok = _logits(30, 5000, torch.bfloat16, hip_device)
    assert _lib.calls().token_logprobs(x, tok, 5) is not None
    assert _lib.calls().token_logprobs(x, tok.int(), 5) is None and _lib.calls().token_logprobs(x, tok, 65) is None
    got = token_logprobs(x, tok, 5)
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", None)
        want = token_logprobs(x, tok, 5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0x7F81), (torch.bfloat16, -0x7F), (torch.float16, 0x7C01),
                                        (torch.float32, 0x7F800001), (torch.float32, -0x7FFFFF)], ids=str)  # fmt: skip
@pytest.mark.parametrize("T,V,top", [(4, 5003, 9), (8, 128256, 20), (2100, 2061, 64)])
def test_signalling_nans_hide_no_entry(hip_device, T, V, top, dtype, bits):
    """NaN counts as -inf in the order, a signalling one too, wherever it stands beside larger entries: one in every
    second place, one in each eight (the last of a vector), all but three places, and a single one beside the largest."""
    x, tok = _logits(T, V, dtype, hip_device, seed=V)
    raw = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    raw[0::4, 1::2] = bits
    raw[1::4, 7::8] = bits
    three = [3, V // 2, V - 2]
    kept = raw[2::4, three]
    raw[2::4] = bits
    raw[2::4, three] = kept
    single = raw[3::4]
    best = x[3::4].float().argmax(1, keepdim=True)
    single.scatter_(1, torch.where(best + 1 < V, best + 1, best - 1), bits)
    r = token_logprobs(x, tok, top)
    order = torch.sort(torch.where(x.isnan(), -math.inf, x.float()), dim=-1, descending=True, stable=True).indices
    assert torch.equal(r.top_ids, order[:, :top])
    assert r.logprobs.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()


@pytest.mark.parametrize("top", [65, 101, 10**6])
def test_a_refused_number_of_alternatives_allocates_nothing(hip_device, top):
    x, tok = _logits(4, 100, torch.float32, hip_device)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="top"):
        token_logprobs(x, tok, top)
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.parametrize("top", [9, 64])
def test_largest_in_few_threads_of_two_segments(hip_device, top):
    """As above in segments of a row: the 4096 largest entries of each lie in the strides of sixteen threads, past
    the list of candidates, and the rounds' keys go through the join. 200 rows of 128256 make two segments of 8016 vectors."""
    V, T, per = 128256, 200, 8
    at = torch.arange(V, device=hip_device)
    within = at % (8016 * per)
    own = within % (256 * per) < 16 * per
    row = torch.where(own, 1.0 + at / 1024, at % 7 / 8).to(torch.bfloat16)[None]
    x, tok = row.expand(T, -1), at[-T:]
    r = token_logprobs(x, tok, top)
    assert (r.top_ids == r.top_ids[0]).all() and (r.top_logprobs == r.top_logprobs[0]).all()
    _check(x[-2:], tok[-2:], top, type(r)(*(f[-2:] for f in r)))
