"""The per-step calls on tensors (_kvhtorch): plain valid calls are taken and give the bits of the
step-by-step path; everything else comes back as None and HipAttention raises (or computes) what it
does without them."""

from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from kvserve_amd import HipAttention, _lib, fp4_caches, token_logprobs, workloads
from kvserve_amd.attention import FP8

pytestmark = pytest.mark.gpu


class _Sub(torch.Tensor):
    pass


@pytest.fixture
def batch(hip_device):
    w = workloads.custom("calls", [1, 3, 40], [30, 500, 7], 32, 8, 64, 16, seed=1)
    return workloads.materialize(w, torch.bfloat16, hip_device, seed=1)


def _args(b, **kw):
    a = {"q": b.q, "k": b.k_cache, "v": b.v_cache, "bt": b.meta.block_tables, "sl": b.meta.seq_lens,
         "qsl": b.meta.query_start_loc, "mq": b.meta.max_query_len, "scale": 0.125, "out": None, "ks": 1.0, "vs": 1.0}  # fmt: skip
    a.update(kw)
    return list(a.values())


def _without(monkeypatch, f):
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", None)
        return f()


def test_taken_calls_give_the_same_bits(batch, monkeypatch):
    b, slots = batch, batch.meta.slot_mapping
    caches = [b.k_cache.clone(), b.v_cache.clone()]
    assert _lib.calls().write_kv(*caches, b.k_new, b.v_new, slots, 1.0, 1.0) is True
    _without(monkeypatch, lambda: HipAttention.write_kv(b.k_cache, b.v_cache, b.k_new, b.v_new, slots))
    assert torch.equal(caches[0], b.k_cache) and torch.equal(caches[1], b.v_cache)
    want = _without(monkeypatch, lambda: HipAttention.forward(b.q, b.k_cache, b.v_cache, b.meta, 0.125))
    got = _lib.calls().forward(*_args(b))
    assert torch.equal(got, want) and got.is_contiguous()
    wide = torch.zeros(b.q.shape[0], 40, 64, dtype=b.q.dtype, device=b.q.device)
    out = wide[:, 4:36]  # a strided output
    assert _lib.calls().forward(*_args(b, out=out)) is out and torch.equal(out, want)
    assert not wide[:, :4].any() and not wide[:, 36:].any()
    strided = torch.cat([b.q, b.q], dim=1)[:, :32]
    assert torch.equal(HipAttention.forward(strided, b.k_cache, b.v_cache, b.meta, 0.125), want)
    assert torch.equal(HipAttention.forward(b.q, b.k_cache, b.v_cache, b.meta, 0.125), want)


def test_refused_calls_are_left_to_the_method(batch):
    b = batch
    f = _lib.calls().forward
    assert f(*_args(b)) is not None
    fp8 = torch.zeros(b.k_cache.shape, dtype=torch.uint8, device=b.q.device).view(FP8)
    for kw in (
        {"q": b.q.float()}, {"q": b.q.cpu()}, {"q": b.q[..., ::2]}, {"q": b.q[0]}, {"q": b.q[:, :31]},
        {"k": b.k_cache.half()}, {"k": b.k_cache[:-1]}, {"k": fp8}, {"bt": b.meta.block_tables.int()},
        {"bt": b.meta.block_tables[:, ::2]}, {"sl": b.meta.seq_lens[:-1]}, {"qsl": b.meta.seq_lens},
        {"sl": b.meta.seq_lens.cpu()}, {"ks": 0.5}, {"out": b.q[:-1].clone()}, {"out": b.q.half()}, {"out": b.q.cpu()},
    ):  # fmt: skip
        assert f(*_args(b, **kw)) is None, kw.keys()
        a = dict(zip(("q", "k", "v", "bt", "sl", "qsl", "mq", "scale", "out", "ks", "vs"), _args(b, **kw)))
        meta = type(b.meta)(b.meta.slot_mapping, a["bt"], a["sl"], b.meta.query_lens, a["qsl"], b.meta.max_seq_len, a["mq"])
        with pytest.raises(ValueError):
            HipAttention.forward(a["q"], a["k"], a["v"], meta, a["scale"], a["out"], a["ks"], a["vs"])
    for s in (0.0, -1.0, float("inf"), float("nan")):
        assert f(*_args(b, k=fp8, v=fp8, ks=s)) is None
    assert f(*_args(b, k=fp8, v=fp8, ks=2.0, vs=0.5)) is not None
    # no plain tensor or number: left to the method, which takes them
    assert f(*_args(b, q=b.q.as_subclass(_Sub))) is None
    assert f(*_args(b, scale=torch.tensor(0.125))) is None
    assert f(*_args(b, mq=True)) is None
    w = _lib.calls().write_kv
    slots = b.meta.slot_mapping
    assert w(b.k_cache, b.v_cache, b.k_new, b.v_new, slots, 1.0, 1.0) is True
    for bad in (
        (b.k_cache, b.v_cache, b.k_new[:-1], b.v_new, slots), (b.k_cache, b.v_cache, b.k_new, b.v_new, slots[:-1]),
        (b.k_cache, b.v_cache, b.k_new.half(), b.v_new.half(), slots), (b.k_cache, b.v_cache, b.k_new, b.v_new, slots.int()),
        (b.k_cache.cpu(), b.v_cache.cpu(), b.k_new, b.v_new, slots),
    ):  # fmt: skip
        assert w(*bad, 1.0, 1.0) is None
        with pytest.raises(ValueError):
            HipAttention.write_kv(*bad)


def test_status_errors_still_raise(batch):
    b = batch
    q = torch.cat([b.q.flatten(), b.q.flatten()])[1 : 1 + b.q.numel()].view(b.q.shape)  # 2 bytes off: KVH_E_ALIGN
    with pytest.raises(_lib.KvhError, match="kvh_paged_attention.*aligned"):
        HipAttention.forward(q, b.k_cache, b.v_cache, b.meta, 0.125)


def _makers(b):
    """Calls that make their outputs: attention, RoPE + write and read-back over 16-bit and MXFP4 caches, log probabilities."""
    w, dev = b.workload, b.q.device
    T, slots = b.q.shape[0], b.meta.slot_mapping
    packed = fp4_caches(*b.k_cache.shape, dev)
    qkv = torch.randn(T, 48 * 64, device=dev).to(b.q.dtype)
    cos, sin = (torch.randn(600, 64, device=dev) for _ in range(2))
    pos = torch.arange(T, device=dev)
    kv = {"": (b.k_cache, b.v_cache, 1.0, 1.0), "_fp4": packed}
    for name, (k, v, ks, vs) in kv.items():
        yield "forward" + name, lambda k=k, v=v, ks=ks, vs=vs: HipAttention.forward(b.q, k, v, b.meta, w.scale, None, ks, vs)
        yield "rope_and_cache" + name, lambda k=k, v=v, ks=ks, vs=vs: HipAttention.rope_and_cache(
            qkv, pos, cos, sin, k, v, slots, 32, k_scale=ks, v_scale=vs)  # fmt: skip
    k, v, ks, vs = packed
    yield "read_kv", lambda: HipAttention.read_kv(k, v, slots, torch.bfloat16, ks, vs)
    yield "token_logprobs", lambda: token_logprobs(qkv, pos, 3)


def test_allocations_are_seen_by_a_dispatch_mode(batch):
    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            got = func(*args, **(kwargs or {}))
            if func is torch.ops.aten.empty.memory_format:
                self.made.append(got.data_ptr())
            return got

    for name, call in _makers(batch):
        with Seen() as seen:
            seen.made = []
            out = call()
        for t in [out] if isinstance(out, torch.Tensor) else out:
            assert t.data_ptr() in seen.made, name


def test_new_outputs_are_filled_under_deterministic_algorithms(batch):
    """As torch.empty's: rows behind the last sequence, which no call writes, are NaN then and not what memory held."""
    b, dev = batch, batch.q.device
    T = b.q.shape[0]
    wide = torch.cat([b.q, torch.ones_like(b.q[:9])])
    packed = fp4_caches(*b.k_cache.shape, dev)
    for caches in ((b.k_cache, b.v_cache, 1.0, 1.0), packed):
        k, v, ks, vs = caches
        want = HipAttention.forward(wide, k, v, b.meta, 0.125, None, ks, vs)[:T].clone()
        torch.full_like(wide, 7.0)  # freed: what the next allocation of this size finds
        torch.use_deterministic_algorithms(True)
        try:
            out = HipAttention.forward(wide, k, v, b.meta, 0.125, None, ks, vs)
        finally:
            torch.use_deterministic_algorithms(False)
        assert torch.equal(out[:T], want) and out[T:].isnan().all()
