"""The calls on tensors (_kvhtorch) of windowed attention, norm_rope_and_cache and linear4: plain valid calls are taken and give
the bits of the step-by-step path; everything else comes back as None, and the method raises or computes what it does without."""

from __future__ import annotations

import pytest
import torch

from kvserve_amd import HipAttention, _lib, fp4_caches, linear4, linear4_silu_mul, quantize_weight4, workloads
from kvserve_amd.attention import FP8

pytestmark = pytest.mark.gpu

H, HKV, D, BLOCK = 8, 2, 64, 16


class _Sub(torch.Tensor):
    pass


def _both(monkeypatch, name, f):
    """(what f gives with the call taken, what it gives without)"""
    taken = []
    _kvhtorch = _lib.calls()
    real = getattr(_kvhtorch, name)

    class Calls:
        def __getattr__(self, other):
            return getattr(_kvhtorch, other)

    def spy(*a):
        r = real(*a)
        taken.append(r is not None)
        return r

    setattr(Calls, name, staticmethod(spy))
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", Calls())
        got = f()
    assert taken == [True]
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", None)
        return got, f()


@pytest.fixture
def batch(hip_device):
    w = workloads.custom("operator_calls", [1, 3, 40], [30, 500, 7], H, HKV, D, BLOCK, seed=1)
    return workloads.materialize(w, torch.bfloat16, hip_device, seed=1)


def _caches(b, kind):
    """(caches and scales) of the batch's pool in a format"""
    if kind == "bf16":
        return b.k_cache.clone(), b.v_cache.clone(), 1.0, 1.0
    if kind == "e4m3":
        return b.k_cache.to(FP8), b.v_cache.to(FP8), 0.5, 2.0
    k, v, ks, vs = fp4_caches(b.k_cache.shape[0], BLOCK, HKV, D, b.q.device)
    slots = torch.arange(b.k_cache.shape[0] * BLOCK, device=b.q.device)
    HipAttention.write_kv(k, v, b.k_cache.flatten(0, 1), b.v_cache.flatten(0, 1), slots, ks, vs)
    return k, v, ks, vs


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "mxfp4"])
def test_window_bits(batch, kind, monkeypatch):
    b = batch
    k, v, ks, vs = _caches(b, kind)
    for window, sinks in ((20, 0), (64, 4), (2**31 - 1, 0)):
        f = lambda: HipAttention.forward(b.q, k, v, b.meta, 0.125, None, ks, vs, window, sinks)  # noqa: E731
        got, want = _both(monkeypatch, "forward_window", f)
        assert torch.equal(got, want) and got.is_contiguous()
    wide = torch.zeros(b.q.shape[0], H + 8, D, dtype=b.q.dtype, device=b.q.device)
    out = wide[:, 4 : 4 + H]
    assert HipAttention.forward(b.q, k, v, b.meta, 0.125, out, ks, vs, 64, 4) is out and out.any()
    assert not wide[:, :4].any() and not wide[:, 4 + H :].any()


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "mxfp4"])
@pytest.mark.parametrize("normed", [False, True])
def test_norm_rope_bits(batch, kind, normed, monkeypatch):
    b, dev = batch, batch.q.device
    T = b.q.shape[0]
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn((T, (H + 2 * HKV) * D), generator=g, device=dev).bfloat16()
    pos = torch.randint(0, 600, (T,), generator=g, device=dev)
    cos, sin = (torch.rand((600, 16), generator=g, device=dev) for _ in range(2))
    norms = [torch.rand((D,), generator=g, device=dev).bfloat16() if normed else None for _ in range(2)]
    pools = []

    def f():
        k, v, ks, vs = _caches(b, kind)
        out = HipAttention.norm_rope_and_cache(qkv, pos, cos, sin, k, v, b.meta.slot_mapping, H, *norms, 1e-5, normed, None, ks, vs)
        pools.append([t.view(torch.uint8) for t in (k, v, ks, vs) if isinstance(t, torch.Tensor)])
        return out

    got, want = _both(monkeypatch, "norm_rope_and_cache", f)
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(*pools, strict=True))


@pytest.mark.parametrize("m", [1, 9, 40, 130])
@pytest.mark.parametrize("product", [linear4, linear4_silu_mul])
def test_linear4_bits(hip_device, m, product, monkeypatch):
    g = torch.Generator(device=hip_device).manual_seed(5)
    w = quantize_weight4(torch.randn((320, 1024), generator=g, device=hip_device).half())
    x = torch.randn((m, 1024), generator=g, device=hip_device).half()
    got, want = _both(monkeypatch, "linear4", lambda: product(x, w))
    assert torch.equal(got, want)
    out = torch.full((m, got.shape[1] + 8), 7.0, dtype=x.dtype, device=hip_device)
    view = out[:, 3:-5]
    assert product(x, w, out=view) is view and torch.equal(view, want) and (out[:, :3] == 7).all() and (out[:, -5:] == 7).all()


def test_refused_calls_are_left_to_the_method(batch):
    b, m, dev = batch, batch.meta, batch.q.device
    f = _lib.calls().forward_window
    base = {"q": b.q, "k": b.k_cache, "v": b.v_cache, "bt": m.block_tables, "sl": m.seq_lens, "qsl": m.query_start_loc,
            "mq": m.max_query_len, "scale": 0.125, "out": None, "ks": 1.0, "vs": 1.0, "window": 20, "sinks": 0}  # fmt: skip
    assert f(*base.values()) is not None
    for kw in ({"q": b.q.float()}, {"q": b.q.cpu()}, {"q": b.q[..., ::2]}, {"k": b.k_cache.half()}, {"k": b.k_cache[:-1]},
               {"bt": m.block_tables.int()}, {"sl": m.seq_lens[:-1]}, {"ks": 0.5}, {"out": b.q.half()}, {"window": 0},
               {"sinks": -1}, {"window": 1.5}):  # fmt: skip
        a = {**base, **kw}
        assert f(*a.values()) is None, kw.keys()
        meta = type(m)(m.slot_mapping, a["bt"], a["sl"], m.query_lens, a["qsl"], m.max_seq_len, a["mq"])
        with pytest.raises(ValueError):
            HipAttention.forward(a["q"], a["k"], a["v"], meta, 0.125, a["out"], a["ks"], a["vs"], a["window"], a["sinks"])
    # left to the method, which takes them
    for kw in ({"q": b.q.as_subclass(_Sub)}, {"window": 2**40}, {"sinks": 2**40}):
        assert f(*{**base, **kw}.values()) is None
    assert torch.equal(HipAttention.forward(b.q, b.k_cache, b.v_cache, m, 0.125, window=2**40),
                       HipAttention.forward(b.q, b.k_cache, b.v_cache, m, 0.125))  # fmt: skip

    f = _lib.calls().norm_rope_and_cache
    T = b.q.shape[0]
    qkv = torch.zeros((T, (H + 2 * HKV) * D), dtype=torch.bfloat16, device=dev)
    cos = torch.zeros((8, 16), device=dev)
    pos, norm = torch.zeros(T, dtype=torch.int64, device=dev), torch.ones(D, dtype=torch.bfloat16, device=dev)
    base = {"qkv": qkv, "positions": pos, "cos": cos, "sin": cos, "k_cache": b.k_cache, "v_cache": b.v_cache,
            "slots": m.slot_mapping, "num_heads": H, "q_norm": norm, "k_norm": None, "eps": 1e-6, "interleaved": False,
            "out": None, "k_scale": 1.0, "v_scale": 1.0}  # fmt: skip
    assert f(*base.values()) is not None
    for kw in ({"qkv": qkv.half()}, {"qkv": qkv[:, :-D]}, {"qkv": qkv.cpu()}, {"positions": pos.int()}, {"slots": m.slot_mapping[:-1]},
               {"cos": cos.double()}, {"cos": cos[:, :8]}, {"sin": cos[:4]}, {"q_norm": norm.float()}, {"k_norm": norm[:-1]},
               {"num_heads": H + 1}, {"out": qkv}, {"k_scale": 2.0}):  # fmt: skip
        a = {**base, **kw}
        assert f(*a.values()) is None, kw.keys()
        with pytest.raises(ValueError):
            HipAttention.norm_rope_and_cache(**a)
    assert f(*{**base, "interleaved": 1}.values()) is None

    f = _lib.calls().linear4
    w = quantize_weight4(torch.ones((48, 256), dtype=torch.bfloat16, device=dev))
    x = torch.zeros((3, 256), dtype=torch.bfloat16, device=dev)
    code = _lib.KVH_DTYPE[torch.bfloat16]
    assert f(x, w.codes, w.scales, 48, 256, 128, code, False, None) is not None
    for bad_x, out in ((x.half(), None), (x[:, :128], None), (x.cpu(), None), (x.t(), None), (x, x.half()), (x, x)):
        assert f(bad_x, w.codes, w.scales, 48, 256, 128, code, False, out) is None
        with pytest.raises(ValueError):
            linear4(bad_x, w, out=out)
    assert f(x, w.codes, w.scales, 64, 256, 128, code, False, None) is None
    assert f(x, w.codes, w.scales, 48, 256, 64, code, False, None) is None
    assert f(x, w.codes, w.scales, 48, 256, 128, code, True, None) is None  # 48 rows: no whole halves
    with pytest.raises(ValueError):
        linear4_silu_mul(x, w)
    with pytest.raises(ValueError):
        linear4(x, w.to("cpu"))
    with pytest.raises(_lib.KvhError):  # rows of an odd alignment
        linear4(torch.zeros((3, 260), dtype=torch.bfloat16, device=dev)[:, :256], w)
