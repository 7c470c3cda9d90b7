"""MXFP4 KV caches on the GPU, against the format's oracle in 64 bits (oracle/fp4.py):

  * write_kv and rope_and_cache store the oracle's bytes, bit for bit, at the slots given and nowhere else;
  * read_kv gives every code under every scale, converted to the asked type;
  * forward matches attention in 64 bits over the decoded values within a bound derived from its roundings.

The bound. Keys and values reach the MFMAs exactly (a 4-bit value times a power of two), scores are fp32 sums of exact
products. With u the half step of the 16-bit type (2^-8 bf16, 2^-11 fp16), P is rounded to it before P V: at most u of
sum_j p_j |v_j| =: A. The output is rounded once (u |out|); where the row sum is taken of the rounded P, once more. The
rest is fp32: a score's D = 128 products give an error of at most 128 2^-24 sum |q k| scale < 2^-10 for the values here
(sum |q k| scale < 100), which moves numerator and denominator by as much: 2^-9 A; the sums over up to 12000 keys and
the exponentials' 2^-22 stay far below that. So |got - want| <= (u + 2^-9) A + 2 u |want|.
Below its normal numbers fp16 has a fixed step of 2^-24, so there a rounding is off by up to 2^-25 whatever the value:
2^-25 for the output (normal from 6.1e-5 on), and 2^-25 |v_j| <= 6 2^-25 for each P, whose row has a sum of 1 or more.
"""

from __future__ import annotations

import random

import pytest
import torch

from kvserve_amd import HipAttention, fp4_caches, last_launch_kernels, token_logprobs, workloads
from kvserve_amd.attention import AttentionMetadata
from oracle import fp4

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = [torch.bfloat16, torch.float16]
ALL_TYPES = [*DTYPES, torch.float32]


def _pool(nb, bs, hkv, D, dev, layout, fill=0):
    """(k, v, k_scale, v_scale) under their dtypes: "head" pages (fp4_caches), "token" pages (the 16-bit caches' order) or
    rows "apart" (with room between them), every byte `fill`."""
    if layout == "head":
        caches = fp4_caches(nb, bs, hkv, D, dev)
    else:
        def make(width, dtype):
            gap = width if layout == "apart" else 0
            return torch.zeros((nb, bs, hkv, width + gap), dtype=torch.uint8, device=dev)[..., :width].view(dtype)

        caches = (make(D // 2, fp4.FP4), make(D // 2, fp4.FP4), make(D // 32, fp4.E8M0), make(D // 32, fp4.E8M0))
    if fill:
        for c in caches:
            c.view(torch.uint8).fill_(fill)
    return caches


def _bytes(t):
    return t.view(torch.uint8)


def _random_pool(nb, bs, hkv, D, dev, layout, seed):
    """A pool of random codes under scales 2^-4 .. 2^0, values up to 6."""
    g = torch.Generator(device=dev).manual_seed(seed)
    k, v, ks, vs = _pool(nb, bs, hkv, D, dev, layout)
    for c in (k, v):
        _bytes(c).copy_(torch.randint(0, 256, c.shape, generator=g, device=dev, dtype=torch.uint8))
    for c in (ks, vs):
        _bytes(c).copy_(torch.randint(123, 128, c.shape, generator=g, device=dev, dtype=torch.uint8))
    return k, v, ks, vs


def _values(c, s):
    return fp4.dequantize(_bytes(c), _bytes(s))


def _wild(shape, dtype, gen, dev):
    """N(0, 1) x 10^U(-4, 4) rows with ties, zeros, the ends of the type, infinities and NaNs among them."""
    x = torch.randn(shape, generator=gen, device=dev) * 10 ** (torch.rand(shape, generator=gen, device=dev) * 8 - 4)
    flat = x.view(-1, 32)
    ties = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, -0.0], device=dev)
    flat[0] = 0
    flat[1, :12] = ties
    flat[1, 12:] = 0
    flat[2, :12] = ties / 8
    flat[2, 12:] = 0
    flat[3] = 0.0
    flat[3, 5] = 6.99
    x = x.to(dtype)
    f = x.view(-1, 32)
    f[4, 3] = torch.finfo(dtype).max
    f[5, 9] = float("inf")
    f[6, 0] = -float("inf")
    f[7, 31] = float("nan")
    f[8] = torch.finfo(dtype).smallest_normal
    f[9] = torch.finfo(dtype).smallest_normal / 2 ** torch.arange(32, device=dev).clamp(max=6).to(dtype)
    return x


def _check_rows(caches, before, slots, want_k, want_v):
    """The caches' bytes equal `before` with the rows at `slots` replaced (the codes of NaN blocks are open)."""
    for i, rows in ((0, want_k), (1, want_v)):
        code, s = rows
        c, x = _bytes(caches[i]).cpu().flatten(0, 1), _bytes(caches[i + 2]).cpu().flatten(0, 1)
        wc, wx = before[i].flatten(0, 1).clone(), before[i + 2].flatten(0, 1).clone()
        wc[slots], wx[slots] = code, s
        assert torch.equal(x, wx)
        nan = (wx == 255).repeat_interleave(16, dim=-1)
        assert torch.equal(c.masked_fill(nan, 0), wc.masked_fill(nan, 0))


# -- writing ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["head", "token", "apart"])
@pytest.mark.parametrize("dtype", ALL_TYPES, ids=str)
@pytest.mark.parametrize("T,hkv,D", [(1, 1, 32), (37, 8, 128), (3, 5, 64), (9, 3, 96)])
def test_write_kv_bit_exact(hip_device, layout, dtype, T, hkv, D):
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(T)
    nb, bs = 12, 16
    n = max(T, -(-10 // (hkv * D // 32)))
    k = _wild((n, hkv, D), dtype, g, dev)[:T]
    wide = _wild((n, hkv * D + 64), dtype, g, dev)[:T]
    v = wide[:, 64:].view(T, hkv, D)  # a strided view, like the fused projection's output
    caches = _pool(nb, bs, hkv, D, dev, layout, fill=0x5A)
    before = [_bytes(c).cpu() for c in caches]
    slots = torch.randperm(nb * bs, generator=g, device=dev)[:T]
    if T > 5:
        slots[5], slots[2] = nb * bs, -1  # outside the pool: skipped
    ok = ((slots >= 0) & (slots < nb * bs)).cpu()
    HipAttention.write_kv(*caches[:2], k, v, slots, *caches[2:])
    torch.cuda.synchronize()
    _check_rows(caches, before, slots.cpu()[ok], fp4.quantize(k.cpu()[ok]), fp4.quantize(v.cpu()[ok]))


@pytest.mark.parametrize("T", [0, 1024, 2500])
def test_write_kv_many_tokens(hip_device, T):
    """1, 2 and 4 tokens per workgroup, the last one short."""
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(T)
    hkv, D, bs = 2, 64, 32
    nb = T // bs + 3
    k, v = (torch.randn(T, hkv, D, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    caches = _pool(nb, bs, hkv, D, dev, "head")
    before = [_bytes(c).cpu() for c in caches]
    slots = torch.randperm(nb * bs, generator=g, device=dev)[:T]
    HipAttention.write_kv(*caches[:2], k, v, slots, k_scale=caches[2], v_scale=caches[3])
    torch.cuda.synchronize()
    _check_rows(caches, before, slots.cpu(), fp4.quantize(k), fp4.quantize(v))


def test_a_slot_named_twice(hip_device):
    """Rows that share a slot (a graph's padding) touch that slot alone; where they are equal it holds them."""
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = (torch.randn(40, 2, 64, generator=g, device=dev).bfloat16() for _ in range(2))
    k[20:], v[20:] = k[19], v[19]
    slots = torch.tensor([*range(32, 52), *[51] * 20], device=dev)
    caches = _pool(5, 16, 2, 64, dev, "head", fill=0x5A)
    before = [_bytes(c).cpu().clone() for c in caches]
    HipAttention.write_kv(*caches[:2], k, v, slots, *caches[2:])
    at = slots[:20].cpu()
    _check_rows(caches, before, at, fp4.quantize(k[:20]), fp4.quantize(v[:20]))
    k[30], v[30] = 1.0, -2.0  # not equal: that row is one of theirs or a mixture, the others stay
    HipAttention.write_kv(*caches[:2], k, v, slots, *caches[2:])
    for i, x in ((0, k), (1, v)):
        code, s = fp4.quantize(x[:19])
        assert torch.equal(_bytes(caches[i]).cpu().flatten(0, 1)[at[:19]], code)
        assert torch.equal(_bytes(caches[i + 2]).cpu().flatten(0, 1)[at[:19]], s)


def test_write_then_read_gives_what_the_format_keeps(hip_device):
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(8)
    k, v = (torch.randn(40, 4, 128, generator=g, device=dev).to(torch.float16) for _ in range(2))
    caches = _pool(5, 16, 4, 128, dev, "head")
    slots = torch.randperm(80, generator=g, device=dev)[:40]
    HipAttention.write_kv(*caches[:2], k, v, slots, *caches[2:])
    rk, rv = HipAttention.read_kv(*caches[:2], slots, torch.float16, *caches[2:])
    for x, r in ((k, rk), (v, rv)):
        assert torch.equal(r.cpu().double(), fp4.dequantize(*fp4.quantize(x)))
    # duplicate slots and slots outside the pool
    rk, _ = HipAttention.read_kv(*caches[:2], torch.tensor([-1, 3, 80, 3], device=dev), torch.float32, *caches[2:])
    assert not rk[0].any() and not rk[2].any() and torch.equal(rk[1], rk[3])


# -- RoPE ------------------------------------------------------------------------------------------
def _tables(n, D, dev):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** -(torch.arange(0, D, 2).double() / D)
    return a.cos().float().repeat(1, 2).to(dev), a.sin().float().repeat(1, 2).to(dev)


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("dtype", ALL_TYPES, ids=str)
@pytest.mark.parametrize("T,H,hkv,D", [(1, 4, 1, 64), (45, 32, 8, 128), (7, 6, 3, 192)])
def test_rope_and_cache_bit_exact(hip_device, layout, dtype, T, H, hkv, D):
    """q and the cache's bytes are those of the fp32 operations done one by one, each rounded once at the end."""
    dev = hip_device
    g = torch.Generator(device=dev).manual_seed(T)
    nb, bs = 8, 16
    wide = torch.randn(T, (H + 2 * hkv) * D + 64, generator=g, device=dev).to(dtype) * 4
    qkv = wide[:, : (H + 2 * hkv) * D]
    cos, sin = _tables(200, D, dev)
    pos = torch.randint(0, 200, (T,), generator=g, device=dev)
    at = pos.clone()
    if T > 4:
        pos[1], at[1] = 10**6, 199  # clamped to the tables
        pos[2], at[2] = -5, 0
    slots = torch.randperm(nb * bs, generator=g, device=dev)[:T]
    if T > 4:
        slots[3] = nb * bs + 7
    ok = (slots < nb * bs).cpu()
    caches = _pool(nb, bs, hkv, D, dev, layout, fill=0x33)
    before = [_bytes(c).cpu() for c in caches]
    got = HipAttention.rope_and_cache(qkv, pos, cos, sin, *caches[:2], slots, H, k_scale=caches[2], v_scale=caches[3])
    torch.cuda.synchronize()
    x = qkv.cpu().float().unflatten(1, (-1, D))
    c, s = cos.cpu()[at.cpu()][:, None], sin.cpu()[at.cpu()][:, None]
    rot = x[:, : H + hkv]
    rot = rot * c + torch.cat((-rot[..., D // 2 :], rot[..., : D // 2]), dim=-1) * s
    assert torch.equal(got.cpu(), rot[:, :H].to(dtype))
    _check_rows(caches, before, slots.cpu()[ok], fp4.quantize(rot[ok, H:], dtype), fp4.quantize(x[ok, H + hkv :], dtype))


# -- reading ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL_TYPES, ids=str)
def test_read_kv_every_code_and_scale(hip_device, dtype):
    """Block b of head h of slot s: 32 codes 0 .. 15 twice, under scale byte s; all 256 bytes s, K and V in turn."""
    dev = hip_device
    k, v, ks, vs = _pool(16, 16, 2, 64, dev, "head")
    code = torch.arange(32, device=dev) % 16
    packed = (code[0::2] | (code[1::2] << 4)).to(torch.uint8)
    _bytes(k)[:] = packed.repeat(2)
    _bytes(v)[:] = packed.flip(0).repeat(2)
    scale = torch.arange(256, device=dev, dtype=torch.uint8).view(16, 16, 1, 1).expand(16, 16, 2, 2)
    _bytes(ks)[:] = scale
    _bytes(vs)[:] = scale
    order = torch.randperm(256, device=dev)
    got = HipAttention.read_kv(k, v, order, dtype, ks, vs)
    for c, s, r in ((k, ks, got[0]), (v, vs, got[1])):
        want = _values(c, s).flatten(0, 1)[order].float().to(dtype)
        assert torch.equal(r.nan_to_num(12345.0), want.nan_to_num(12345.0)) and torch.equal(r.isnan(), want.isnan())


@pytest.mark.parametrize("layout", ["head", "token", "apart"])
@pytest.mark.parametrize("T,hkv,D", [(0, 2, 64), (1, 1, 32), (777, 8, 64), (2101, 3, 128), (1030, 2, 160)])
def test_read_kv_rows(hip_device, layout, T, hkv, D):
    caches = _random_pool(40, 16, hkv, D, hip_device, layout, seed=T)
    slots = torch.randint(0, 640, (T,), device=hip_device)
    got = HipAttention.read_kv(*caches[:2], slots, torch.bfloat16, *caches[2:])
    for i in (0, 1):
        assert torch.equal(got[i].double(), _values(caches[i], caches[i + 2]).flatten(0, 1)[slots])


# -- attention -------------------------------------------------------------------------------------
def _meta(w: workloads.Workload, dev, tables=None) -> AttentionMetadata:
    width = w.table_width()
    rows = [t + [0] * (width - len(t)) for t in w.tables]
    qsl = [0]
    for n in w.query_lens:
        qsl.append(qsl[-1] + n)
    t = lambda x: torch.tensor(x, dtype=torch.long, device=dev)  # noqa: E731
    return AttentionMetadata(t(w.slot_mapping()), t(rows), t(w.seq_lens), t(w.query_lens), t(qsl), max(w.seq_lens),
                             max(w.query_lens))  # fmt: skip


def _within_bound(got, q, caches, meta, seq_lens, query_lens, scale):
    want, mag = fp4.attention(q, _values(caches[0], caches[2]), _values(caches[1], caches[3]), meta.block_tables, seq_lens,
                              query_lens, scale)  # fmt: skip
    u = HALF_STEP[got.dtype]
    tiny = 2.0**-25 * (1 + 6 * max(seq_lens)) if got.dtype == torch.float16 else 1e-30
    bound = (u + 2.0**-9) * mag + 2 * u * want.abs() + tiny
    over = ((got.double() - want).abs() / bound).max().item()
    assert over <= 1, f"{over} times the bound"
    assert torch.isfinite(got).all()


def _run(w, dtype, dev, layout="head", seed=0, stale=True):
    caches = _random_pool(w.num_blocks, w.block_size, w.num_kv_heads, w.head_dim, dev, layout, seed)
    if stale:  # what no sequence holds may be anything: NaN scales
        used = torch.zeros(w.num_blocks * w.block_size, dtype=torch.bool, device=dev)
        for t, n in zip(w.tables, w.seq_lens):
            used[torch.tensor(workloads.slots_for(t, w.block_size, 0, n), device=dev)] = True
        for x in caches[2:]:
            _bytes(x)[~used.view(w.num_blocks, w.block_size)] = 255
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = torch.randn(w.num_tokens, w.num_heads, w.head_dim, generator=g, device=dev).to(dtype)
    meta = _meta(w, dev)
    out = HipAttention.forward(q, *caches[:2], meta, w.scale, None, *caches[2:])
    kinds = last_launch_kernels()
    torch.cuda.synchronize()
    _within_bound(out, q, caches, meta, w.seq_lens, w.query_lens, w.scale)
    return kinds


CASES = {**workloads.REFERENCE_CASES, "one_token": ([1], [0]), "page_ends": ([1] * 5, [14, 15, 16, 30, 31])}


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (14, 2), (24, 4)], ids=str)
@pytest.mark.parametrize("name", list(CASES))
def test_reference_cases(hip_device, name, heads, dtype, head_dim, layout):
    q, c = CASES[name]
    _run(workloads.custom(name, q, c, *heads, head_dim, 16, seed=3), dtype, hip_device, layout, seed=len(name))


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("draft", [2, 5, 12, 16])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_verify_tiles(hip_device, head_dim, draft, dtype):
    """One to four 16-row tiles per wave, segments split between units."""
    w = workloads.custom("verify", [draft] * 6, [40, 700, 1900, 3, 1200, 260], 32, 8, head_dim, 16, seed=draft)
    assert _run(w, dtype, hip_device, seed=draft) == ["decode", "reduce"]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("draft", [1, 2, 5, 12, 16])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_verify_tiles_of_token_pages(hip_device, head_dim, draft, dtype):
    """The same where a page keeps a token's heads together (other loads), a single query among them."""
    w = workloads.custom("verify", [draft] * 6, [40, 700, 1900, 3, 1200, 260], 32, 8, head_dim, 16, seed=draft)
    assert _run(w, dtype, hip_device, "token", seed=draft) == ["decode", "reduce"]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("scale", [-0.07, -0.0, 0.0])
def test_scales_of_other_signs(hip_device, scale, head_dim):
    """Decodes, drafts and prompt chunks under a negative scale (the smallest product weighs most) and none (a mean)."""
    dev = hip_device
    for q, c in (([1] * 5, [0, 5, 700, 1900, 31]), ([5] * 3, [1700, 2, 300]), ([200, 1, 60], [100, 900, 0]), ([1], [40])):
        w = workloads.custom("scale", q, c, 16, 4, head_dim, 16, seed=3)
        caches = _random_pool(w.num_blocks, 16, 4, head_dim, dev, "head", 8)
        x = torch.randn(w.num_tokens, 16, head_dim, generator=torch.Generator(device=dev).manual_seed(4), device=dev).bfloat16()
        meta = _meta(w, dev)
        out = HipAttention.forward(x, *caches[:2], meta, scale, None, *caches[2:])
        _within_bound(out, x, caches, meta, w.seq_lens, w.query_lens, scale)


@pytest.mark.parametrize("scale", [4.0, 1e3, 3e5])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("q,c", [([1] * 4, [300, 900, 3000, 31]), ([5] * 3, [1700, 40, 300]), ([200, 60], [100, 900])])
def test_large_scores(hip_device, q, c, dtype, scale):
    """Scores to 10^10: where one key's leads by more than fp32 can blur (128 products: 2^-17 of the sum of their
    magnitudes, here at most 128 * 6 * 200), that key's value comes out whole; no row is infinite or NaN."""
    dev = hip_device
    w = workloads.custom("large", q, c, 8, 2, 128, 16, seed=5)
    caches = _random_pool(w.num_blocks, 16, 2, 128, dev, "head", 6)
    x = torch.randn(w.num_tokens, 8, 128, generator=torch.Generator(device=dev).manual_seed(7), device=dev)
    x = (50 * x).clamp(-200, 200).to(dtype)
    meta = _meta(w, dev)
    out = HipAttention.forward(x, *caches[:2], meta, scale, None, *caches[2:])
    assert torch.isfinite(out).all()
    k, v = (_values(caches[i], caches[i + 2]).flatten(0, 1) for i in range(2))
    certain = t0 = 0
    for table, n, total in zip(w.tables, w.query_lens, w.seq_lens):
        at = torch.tensor(workloads.slots_for(table, 16, 0, total), device=dev)
        for i in range(n):
            see = at[: total - n + 1 + i]
            for h in range(8):
                best = (k[see, h // 4] @ x[t0 + i, h].double()).topk(2)
                lead = (best.values[0] - best.values[1]).item() - 2 * 128 * 6 * 200 * 2.0**-17
                if lead * scale > 200:
                    certain += 1
                    assert torch.equal(out[t0 + i, h].double(), v[see[best.indices[0]], h // 4])
        t0 += n
    assert certain > 0.8 * 8 * t0


@pytest.mark.parametrize("heads", [(1, 1), (64, 1), (40, 10), (12, 12)], ids=str)
def test_head_groups(hip_device, heads):
    w = workloads.custom("groups", [1, 3, 1, 20], [5000, 1200, 64, 300], *heads, 128, 16, seed=1)
    _run(w, torch.bfloat16, hip_device, "token", seed=2)


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_wide_groups_beside_chunks(hip_device, dtype, head_dim, layout):
    """GQA groups above 16: a decode row of several tiles in a mixed batch."""
    for heads in ((64, 1), (40, 2)):
        w = workloads.custom("wide", [1, 3, 1, 20], [5000, 1200, 64, 300], *heads, head_dim, 16, seed=1)
        assert _run(w, dtype, hip_device, layout, seed=2) == ["decode", "prefill", "reduce"]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_short_tables(hip_device, head_dim, dtype):
    w = workloads.custom("short", [1] * 7, [0, 15, 200, 511, 999, 64, 700], 32, 8, head_dim, 16, seed=6)
    assert _run(w, dtype, hip_device, seed=6) == ["decode"]


@pytest.mark.parametrize("layout", ["head", "token", "apart"])
def test_long_contexts_split(hip_device, layout):
    w = workloads.custom("long", [1] * 3 + [5], [12000, 9000, 300, 7000], 32, 8, 128, 16, seed=5)
    _run(w, torch.bfloat16, hip_device, layout, seed=5)


@pytest.mark.parametrize("D,BS", [(128, 32), (64, 64), (128, 48)])
def test_other_block_sizes(hip_device, D, BS):
    _run(workloads.custom("bs", [1, 40, 1, 9], [100, 70, 3000, 0], 32, 8, D, BS, seed=6), torch.bfloat16, hip_device)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("q,c", [([300, 1000], [0, 700]), ([130] * 3 + [1] * 9, [0, 33, 2000] + [100 * i for i in range(9)]),
                                 ([17, 1, 640], [2047, 0, 1]), ([200] * 2 + [1] * 150, [50, 900] + [1500] * 150)])  # fmt: skip
def test_prompt_chunks(hip_device, q, c, dtype):
    """Prompts, chunks over cached tokens, and both beside decodes: in one launch and (many decodes) in two."""
    kinds = _run(workloads.custom("chunks", q, c, 32, 8, 128, 16, seed=2), dtype, hip_device, seed=3)
    assert "prefill" in kinds
    _run(workloads.custom("chunks", q, c, 15, 3, 64, 16, seed=2), dtype, hip_device, "token", seed=3)


def test_shared_prefix(hip_device):
    """Tables that start with the same blocks (the cascade): 32-row groups, a ragged last one, and a single 16-row group."""
    from tests.test_hip_cascade import CASES as SHARED, shared_workload

    for name in ("g4_b16", "g4_b23_ragged", "g1_b5_sg16", "d64_bs16_b9", "g4_q3_rs12", "g4_b5_partial"):
        q, c, heads, D, BS, shared, width = SHARED[name]
        w = shared_workload(q, c, heads, D, BS, shared, width, seed=13)
        assert _run(w, torch.bfloat16, hip_device, seed=4)[0] == "share", name


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_shared_prefix_of_token_pages(hip_device, dtype):
    from tests.test_hip_cascade import CASES as SHARED, shared_workload

    for name in ("g4_b16", "d64_bs16_b9"):
        q, c, heads, D, BS, shared, width = SHARED[name]
        w = shared_workload(q, c, heads, D, BS, shared, width, seed=13)
        assert _run(w, dtype, hip_device, "token", seed=4)[0] == "share", name
        assert _run(w, dtype, hip_device, "head", seed=5)[0] == "share", name


@pytest.mark.parametrize("idx", [2, 3, 5])
def test_full_size_batches(hip_device, idx):
    """64 decodes of 1024-8192 keys, 512 decodes beside four prompt chunks, 32 sequences of five drafts."""
    _run(workloads.baseline_config(idx, seed=0), torch.bfloat16, hip_device, seed=idx, stale=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_every_code_reaches_the_output_exactly(hip_device, D, dtype):
    """Sequences of one key: the output is that key's V."""
    dev, hkv, B, BS = hip_device, 8, 8, 16
    caches = _random_pool(B, BS, hkv, D, dev, "head", seed=1)
    meta = AttentionMetadata(torch.empty(0, dtype=torch.long, device=dev), torch.arange(B, device=dev).view(B, 1),
                             torch.ones(B, dtype=torch.long, device=dev), torch.ones(B, dtype=torch.long, device=dev),
                             torch.arange(B + 1, device=dev), 1, 1)  # fmt: skip
    q = torch.randn(B, hkv, D, device=dev).to(dtype)
    out = HipAttention.forward(q, *caches[:2], meta, D**-0.5, k_scale=caches[2], v_scale=caches[3])
    assert torch.equal(out.double(), _values(caches[1], caches[3])[:, 0])


def test_missing_pages_empty_sequences_and_rows_behind(hip_device):
    """Block ids outside the pool are empty pages; a sequence of length 0 gives zeros; tokens behind the last sequence
    keep what the output held; a strided output and strided queries are taken as they are."""
    dev = hip_device
    w = workloads.custom("odd", [1, 1, 2, 1], [100, 40, 600, 0], 32, 8, 128, 16, seed=9)
    caches = _random_pool(w.num_blocks, 16, 8, 128, dev, "head", seed=9)
    meta = _meta(w, dev)
    meta.block_tables[0, 2] = -1
    meta.block_tables[2, 5] = w.num_blocks
    meta.seq_lens[1] = 0
    T = w.num_tokens + 3  # three rows that no sequence owns
    wide = torch.randn(T, 40, 128, device=dev).to(torch.bfloat16)
    q = wide[:, 4:36]
    room = torch.full((T, 34, 128), 7.0, device=dev, dtype=torch.bfloat16)
    out = room[:, 1:33]
    assert HipAttention.forward(q, *caches[:2], meta, w.scale, out, *caches[2:]) is out
    torch.cuda.synchronize()
    n = w.num_tokens
    _within_bound(out[:n], q[:n], caches, meta, [101, 0, 602, 1], w.query_lens, w.scale)
    assert not out[1].any()
    assert (room[n:] == 7).all() and (room[:, 0] == 7).all() and (room[:, 33] == 7).all()


def test_nan_blocks_stay_in_their_sequence(hip_device):
    """A NaN value block makes its 32 columns NaN for its kv head's rows that see it, a NaN key block whole rows; rows of
    other heads and sequences stay as they are. (A P of 0 times a NaN value is NaN, as in any P V product: rows of
    the same sequence and head that precede the value may have it too.)"""
    dev = hip_device
    w = workloads.custom("nan", [4, 1, 1], [60, 90, 300], 8, 2, 128, 16, seed=4)
    caches = _random_pool(w.num_blocks, 16, 2, 128, dev, "head", seed=4)
    meta = _meta(w, dev)
    q = torch.randn(w.num_tokens, 8, 128, device=dev).to(torch.bfloat16)
    clean = HipAttention.forward(q, *caches[:2], meta, w.scale, None, *caches[2:])
    slot = w.slot_mapping()[2]  # token 2 of the first sequence's four
    _bytes(caches[3])[slot // 16, slot % 16, 1, 2] = 255
    slot = w.slot_mapping()[5]  # the last sequence's token
    _bytes(caches[2])[slot // 16, slot % 16, 0, 3] = 255
    out = HipAttention.forward(q, *caches[:2], meta, w.scale, None, *caches[2:])
    assert out[2:4, 4:, 64:96].isnan().all() and out[5, :4].isnan().all()
    out[0:4, 4:, 64:96] = clean[0:4, 4:, 64:96]
    out[5, :4] = clean[5, :4]
    assert torch.equal(out, clean)


def test_graph_replays_match_eager(hip_device):
    """rope_and_cache and forward captured once and replayed with new inputs and metadata, eager work between."""
    dev = hip_device
    H, hkv, D, BS, NB, n, width = 32, 8, 128, 16, 600, 6, 90
    caches = _random_pool(NB + 1, BS, hkv, D, dev, "head", seed=2)
    cos, sin = _tables(1500, D, dev)
    long = lambda *s: torch.ones(*s, dtype=torch.long, device=dev)  # noqa: E731
    qkv = torch.zeros(n, (H + 2 * hkv) * D, device=dev, dtype=torch.bfloat16)
    pos, slots = long(n), long(n)
    meta = AttentionMetadata(slots, long(n, width), long(n), long(n), torch.arange(n + 1, device=dev), 1, 1)

    def step():
        q = HipAttention.rope_and_cache(qkv, pos, cos, sin, *caches[:2], slots, H, None, *caches[2:])
        return q, HipAttention.forward(q, *caches[:2], meta, D**-0.5, None, *caches[2:])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_out, out = step()
    rng = random.Random(5)
    for it in range(4):
        lens = [rng.randint(1, 1400) for _ in range(n)]
        ids = rng.sample(range(NB), sum(-(-x // BS) for x in lens))
        tables, at = [], 0
        for x in lens:
            tables.append(ids[at : at + -(-x // BS)])
            at += len(tables[-1])
        meta.block_tables.copy_(torch.tensor([t + [NB] * (width - len(t)) for t in tables]))
        meta.seq_lens.copy_(torch.tensor(lens))
        pos.copy_(torch.tensor(lens) - 1)
        slots.copy_(torch.tensor([t[-1] * BS + (x - 1) % BS for t, x in zip(tables, lens)]))
        qkv.copy_(torch.randn(qkv.shape, device=dev))
        graph.replay()
        got = q_out.clone(), out.clone()
        torch.cuda.synchronize()
        torch.randn(1 << 20, device=dev).sum()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), it
        _within_bound(got[1], got[0], caches, meta, lens, [1] * n, D**-0.5)


def test_other_stream(hip_device):
    """The calls run on the current stream: work queued there before them is seen, and what follows sees them."""
    dev = hip_device
    caches = _pool(8, 16, 2, 64, dev, "head")
    slots = torch.arange(5, device=dev)
    src = torch.randn(5, 2, 64, device=dev).to(torch.bfloat16)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device=dev)
        for _ in range(8):
            big = big @ big * 1e-2
        rows = src * 2 + (big[0, 0] * 0).nan_to_num().to(torch.bfloat16)
        HipAttention.write_kv(*caches[:2], rows, rows, slots, *caches[2:])
        k, v = HipAttention.read_kv(*caches[:2], slots, torch.bfloat16, *caches[2:])
        same = torch.equal(k, v)
    s.synchronize()
    assert same and torch.equal(k.cpu().double(), fp4.dequantize(*fp4.quantize((src * 2).cpu())))


def test_new_tensors_are_plain_ones(hip_device):
    """Outputs made by the calls: own storages, as any new tensor in and out of inference mode, empty ones too."""
    dev = hip_device
    caches = _random_pool(4, 16, 2, 64, dev, "head", 1)
    meta = AttentionMetadata(torch.tensor([2], device=dev), torch.tensor([[1]], device=dev), torch.tensor([3], device=dev),
                             torch.tensor([1], device=dev), torch.tensor([0, 1], device=dev), 3, 1)
    for inference in (False, True):
        with torch.inference_mode(inference):
            q = torch.randn(1, 4, 64, device=dev).bfloat16()
            slots = torch.arange(5, device=dev)
            made = [*HipAttention.read_kv(*caches[:2], slots, torch.bfloat16, *caches[2:]),
                    *HipAttention.read_kv(*caches[:2], slots[:0], torch.float32, *caches[2:]),
                    HipAttention.forward(q, *caches[:2], meta, 0.1, None, *caches[2:]),
                    *token_logprobs(torch.randn(3, 50, device=dev), slots[:3], 2)]
        for t in made:
            like = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
            assert t.is_contiguous() and t.device == dev and t.is_inference() == inference and not t.requires_grad
            assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == like.untyped_storage().nbytes()
        kept = made[0].clone()
        del made[1:]
        junk = [torch.full_like(kept, 9.0) for _ in range(8)]  # takes the freed blocks, not the one still held
        assert torch.equal(made[0], kept) and len(junk) == 8


def test_large_pool_offsets_pass_32_bits(hip_device):
    """Pages past 2^32 bytes of a cache: write, read and attention at the far end."""
    dev = hip_device
    hkv, D, BS = 8, 128, 64
    nb = (1 << 32) // (BS * hkv * D // 2) + 40
    caches = fp4_caches(nb, BS, hkv, D, dev)
    table = [nb - 1 - 3 * i for i in range(12)]
    L = 12 * BS - 5
    slots = torch.tensor(workloads.slots_for(table, BS, 0, L), device=dev)
    k, v = (torch.randn(L, hkv, D, device=dev).to(torch.bfloat16) for _ in range(2))
    HipAttention.write_kv(*caches[:2], k, v, slots, *caches[2:])
    rk, rv = HipAttention.read_kv(*caches[:2], slots, torch.bfloat16, *caches[2:])
    assert torch.equal(rk.cpu().double(), fp4.dequantize(*fp4.quantize(k.cpu())))
    for n in (1, 40):  # a decode and a chunk
        meta = AttentionMetadata(slots[-n:], torch.tensor([table], device=dev), torch.tensor([L], device=dev),
                                 torch.tensor([n], device=dev), torch.tensor([0, n], device=dev), L, n)  # fmt: skip
        q = torch.randn(n, 32, D, device=dev).to(torch.bfloat16)
        out = HipAttention.forward(q, *caches[:2], meta, D**-0.5, None, *caches[2:])
        # the oracle over the rows as read back, in pages of their own
        pages = [torch.zeros(12 * BS, hkv, D, dtype=torch.float64, device=dev) for _ in range(2)]
        pages[0][:L], pages[1][:L] = rk.double(), rv.double()
        want, mag = fp4.attention(q, *(p.view(12, BS, hkv, D) for p in pages), torch.arange(12, device=dev)[None], [L], [n],
                                  D**-0.5)  # fmt: skip
        assert ((out.double() - want).abs() <= (2.0**-8 + 2.0**-9) * mag + 2.0**-7 * want.abs()).all()


def test_refusals_on_the_device(hip_device):
    dev = hip_device
    k, v, ks, vs = fp4_caches(4, 16, 2, 64, dev)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(3, device=dev)

    def refused(match, **over):
        a = {"k_cache": k, "v_cache": v, "k": rows, "v": rows, "slots": slots, "k_scale": ks, "v_scale": vs, **over}
        with pytest.raises(ValueError, match=match):
            HipAttention.write_kv(**a)

    refused("scales must be", k_scale=ks[:, :8])
    refused("caches must be", v_cache=v[:2])
    refused("float8_e8m0fnu", v_scale=2.0)
    refused("rows", k=rows[..., :32], v=rows[..., :32])
    refused("one slot per token", slots=slots[:2])
    refused("int64", slots=slots.int())
    refused("device", k=rows.cpu())
    refused("device", k_scale=ks.cpu())
    refused("dtype", v=rows.half())
    refused("unsupported dtype", k=rows.double(), v=rows.double())
    with pytest.raises(ValueError, match="E8M0 scales"):
        HipAttention.write_kv(rows[None], rows[None], rows, rows, slots, ks, vs)
    with pytest.raises(ValueError, match="unsupported dtype"):
        HipAttention.read_kv(k, v, slots, torch.int8, ks, vs)
    meta = AttentionMetadata(slots, slots[None], slots[1:2], slots[1:2], slots[:2], 1, 1)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        HipAttention.forward(rows.float()[:1], k, v, meta, 1.0, None, ks, vs)
    with pytest.raises(ValueError, match="head_dim"):
        HipAttention.forward(rows[:1, :, :32], k, v, meta, 1.0, None, ks, vs)


def test_step_by_step_path_gives_the_same_bits(hip_device, monkeypatch):
    """The methods without the C++ calls on tensors (_kvhtorch), and what those leave to the methods."""
    from kvserve_amd import _lib

    dev = hip_device
    w = workloads.custom("calls", [1, 3, 40], [30, 500, 7], 32, 8, 64, 16, seed=1)
    caches = _random_pool(w.num_blocks, 16, 8, 64, dev, "head", seed=1)
    meta = _meta(w, dev)
    q = torch.randn(w.num_tokens, 32, 64, device=dev).to(torch.bfloat16)
    qkv = torch.randn(w.num_tokens, 48 * 64, device=dev).to(torch.bfloat16)
    k, v = qkv[:, : 8 * 64].view(-1, 8, 64), qkv[:, 8 * 64 : 16 * 64].view(-1, 8, 64)
    cos, sin = _tables(64, 64, dev)
    pos = torch.arange(w.num_tokens, device=dev)

    def everything():
        pools = [[_bytes(c).clone().view(c.dtype) for c in caches] for _ in range(2)]
        r = HipAttention.rope_and_cache(qkv, pos, cos, sin, *pools[0][:2], meta.slot_mapping, 32, None, *pools[0][2:])
        HipAttention.write_kv(*pools[1][:2], k, v, meta.slot_mapping, *pools[1][2:])
        rk, rv = HipAttention.read_kv(*pools[1][:2], meta.slot_mapping, torch.float32, *pools[1][2:])
        out = HipAttention.forward(q, *pools[0][:2], meta, 0.125, None, *pools[0][2:])
        return [r, rk, rv, out, *(_bytes(c) for p in pools for c in p)]

    calls = _lib.calls()
    a = [k, v, meta.slot_mapping]
    assert calls.write_kv_fp4(*caches[:2], *a, *caches[2:]) is True
    assert calls.write_kv_fp4(*caches[:2], *a, caches[2], 1.0) is None
    assert calls.read_kv_fp4(*caches[:2], meta.slot_mapping.int(), 2, *caches[2:]) is None
    assert calls.forward_fp4(q.float(), *caches[:2], meta.block_tables, meta.seq_lens, meta.query_start_loc, 40, 0.1, None,
                             *caches[2:]) is None  # fmt: skip
    got = everything()
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", None)
        want = everything()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("scale", [4.0, 1e3, 3e5])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("q,c", [([1] * 4, [300, 900, 3000, 31]), ([5] * 3, [1700, 40, 300]), ([200, 60], [100, 900])])
def test_large_scores_of_heads_of_64(hip_device, q, c, dtype, scale, layout):
    """As test_large_scores: 64 products blur by 2^-18 of at most 64 * 6 * 200. The scores' standard deviation is about
    600, a leader's mean distance some 600 / sqrt(2 ln n) = 180, and e^(-50 / 180) = 3 of 4 lead by the 50 of scale 4."""
    dev = hip_device
    w = workloads.custom("large", q, c, 8, 2, 64, 16, seed=5)
    caches = _random_pool(w.num_blocks, 16, 2, 64, dev, layout, 6)
    x = torch.randn(w.num_tokens, 8, 64, generator=torch.Generator(device=dev).manual_seed(7), device=dev)
    x = (50 * x).clamp(-200, 200).to(dtype)
    out = HipAttention.forward(x, *caches[:2], _meta(w, dev), scale, None, *caches[2:])
    assert torch.isfinite(out).all()
    k, v = (_values(caches[i], caches[i + 2]).flatten(0, 1) for i in range(2))
    certain = t0 = 0
    for table, n, total in zip(w.tables, w.query_lens, w.seq_lens):
        at = torch.tensor(workloads.slots_for(table, 16, 0, total), device=dev)
        for i in range(n):
            see = at[: total - n + 1 + i]
            for h in range(8):
                best = (k[see, h // 4] @ x[t0 + i, h].double()).topk(2)
                lead = (best.values[0] - best.values[1]).item() - 2 * 64 * 6 * 200 * 2.0**-18
                if lead * scale > 200:
                    certain += 1
                    assert torch.equal(out[t0 + i, h].double(), v[see[best.indices[0]], h // 4])
        t0 += n
    assert certain > 0.5 * 8 * t0


@pytest.mark.parametrize("rows,scales", [(("head", "token"), ("head", "token")), (("token", "head"), ("token", "head")),
                                         (("apart", "head"), ("head", "apart")), (("head", "head"), ("token", "token")),
                                         (("apart", "apart"), ("apart", "apart"))], ids=str)  # fmt: skip
@pytest.mark.parametrize("head_dim", [64, 128])
def test_keys_values_and_scales_in_pages_of_their_own(hip_device, head_dim, rows, scales):
    """Each of the four tensors has strides of its own: decodes over long and short tables, drafts, prompt chunks, a batch
    of both and a shared prefix."""
    dev = hip_device
    batches = [workloads.custom("own", q, c, 16, 4, head_dim, 16, seed=3) for q, c in (
        ([1] * 6, [0, 5, 700, 1900, 31, 5000]), ([1, 1], [40, 63]), ([5] * 3, [1700, 2, 300]), ([200, 60], [100, 900]),
        ([1, 1, 90], [700, 3000, 400]))]  # fmt: skip
    for w in batches:
        made = {name: _random_pool(w.num_blocks, 16, 4, head_dim, dev, name, 8) for name in {*rows, *scales}}
        caches = [made[rows[0]][0], made[rows[1]][1], made[scales[0]][2], made[scales[1]][3]]
        x = torch.randn(w.num_tokens, 16, head_dim, generator=torch.Generator(device=dev).manual_seed(4), device=dev).bfloat16()
        meta = _meta(w, dev)
        out = HipAttention.forward(x, *caches[:2], meta, w.scale, None, *caches[2:])
        _within_bound(out, x, caches, meta, w.seq_lens, w.query_lens, w.scale)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_value_scales_over_their_range(hip_device, head_dim, n):
    """Sequences of n tokens whose key is the same for each and whose value too: the output is that value, for every scale
    under which n of them add up in fp32 (40 * 6 * 2^120 do), the subnormal ones of bf16 too."""
    dev, hkv, BS = hip_device, 2, 64
    at = list(range(248))  # E8M0 bytes
    caches = _random_pool(len(at), BS, hkv, head_dim, dev, "head", seed=1)
    for c in (*caches[:2], caches[2]):  # every token's rows as the first's
        _bytes(c).copy_(_bytes(c)[:, :1].expand(-1, BS, -1, -1).clone())
    _bytes(caches[3]).copy_(torch.tensor(at, dtype=torch.uint8, device=dev).view(-1, 1, 1, 1).expand(caches[3].shape))
    B = len(at)
    meta = AttentionMetadata(torch.empty(0, dtype=torch.long, device=dev), torch.arange(B, device=dev).view(B, 1),
                             torch.full((B,), n, device=dev), torch.full((B,), n, device=dev),
                             torch.arange(B + 1, device=dev) * n, n, n)  # fmt: skip
    q = torch.randn(B * n, hkv, head_dim, device=dev).bfloat16()
    out = HipAttention.forward(q, *caches[:2], meta, head_dim**-0.5, k_scale=caches[2], v_scale=caches[3])
    want = _values(caches[1], caches[3])[:, 0].repeat_interleave(n, 0)
    # equal scores give P = 1 and exact sums; their quotient is off by two roundings to fp32, and bf16 holds the value
    # itself (2^-128 at least; its subnormals lie 2^-133 apart)
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("lens", [[96], [1500, 40], [7000] * 40])
def test_chunks_of_nan_keys_make_their_rows_nan(hip_device, head_dim, layout, lens):
    """Whole runs of NaN keys, as a diverged prompt leaves them: a piece of a split that sees nothing else included."""
    dev = hip_device
    w = workloads.custom("nan", [1] * len(lens), [n - 1 for n in lens], 8, 2, head_dim, 16, seed=4)
    caches = _random_pool(w.num_blocks, 16, 2, head_dim, dev, layout, seed=4)
    meta = _meta(w, dev)
    q = torch.randn(w.num_tokens, 8, head_dim, device=dev).to(torch.bfloat16)
    clean = HipAttention.forward(q, *caches[:2], meta, w.scale, None, *caches[2:])
    run = torch.tensor(w.tables[0][: lens[0] // 16 // 2], device=dev)
    _bytes(caches[2])[run, :, 1] = 255
    out = HipAttention.forward(q, *caches[:2], meta, w.scale, None, *caches[2:])
    assert out[0, 4:].isnan().all()
    out[0, 4:] = clean[0, 4:]
    assert torch.equal(out, clean)
