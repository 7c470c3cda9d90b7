"""Attention with a sliding window and sinks on the GPU, against the definition in 64 bits.

Whatever no token of a sequence sees is poisoned first: the table entries of pages that lie behind every window (ids out
of the pool, or of a page of NaNs), and the bytes of hidden tokens in pages that are read.

The bound is test_hip_fp4's: |got - want| <= (u + 2^-9) A + 2 u |want| with u the half step of the 16-bit type and
A = sum_j p_j |v_j|; E4M3 and MXFP4 values convert exactly to the 16-bit types. fp32 (the vector-ALU kernel): a score's D
products and its exponential's argument are off by at most (D + 4) 2^-24 sum |q k| scale (below 30 for the values here,
whatever D <= 128), numerator and denominator each by that and by the sums' rounding over up to 400 keys, in 64-key tiles:
2 * 132 * 30 * 2^-24 + 2 * 400 * 2^-24 < 2^-10, of A.
"""

from __future__ import annotations

import random

import pytest
import torch

from kvserve_amd import HipAttention, fp4_caches
from kvserve_amd.attention import AttentionMetadata
from oracle import fp4

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
E4M3 = torch.float8_e4m3fn


class Batch:
    """Sequences of q_lens new tokens behind ctx cached ones in a shuffled pool; `kv`: "own", "e4m3" or "fp4"."""

    def __init__(self, dev, q_lens, ctx, H, Hkv, D, bs, window, sinks, dtype=torch.bfloat16, kv="own", seed=0, poison=True):
        self.q_lens, self.ctx, self.H, self.Hkv, self.bs = q_lens, ctx, H, Hkv, bs
        self.window, self.sinks, self.scale = window, sinks, D**-0.5
        g = torch.Generator(device=dev).manual_seed(seed)
        rng = random.Random(seed)
        need = [-(-(n + c) // bs) for n, c in zip(q_lens, ctx)]
        nb = sum(need) + 3  # two spare pages, and one of NaNs (the last)
        ids = list(range(nb - 1))
        rng.shuffle(ids)
        k, v = (torch.randn((nb, bs, Hkv, D), generator=g, device=dev) for _ in range(2))
        self.kwargs = {}
        if kv == "e4m3":
            k, v = (x.clamp(-448, 448).mul(8).to(E4M3) for x in (k, v))
            self.kwargs = {"k_scale": 0.125, "v_scale": 0.125}
            self.kv64 = [x.float().double() * 0.125 for x in (k, v)]
        elif kv == "fp4":
            caches = fp4_caches(nb, bs, Hkv, D, dev)
            for c, x in zip(caches[:2], caches[2:]):
                c.view(torch.uint8).copy_(torch.randint(0, 256, c.shape, generator=g, device=dev, dtype=torch.uint8))
                x.view(torch.uint8).copy_(torch.randint(123, 127, x.shape, generator=g, device=dev, dtype=torch.uint8))
            k, v, ks, vs = caches
            self.kwargs = {"k_scale": ks, "v_scale": vs}
            self.kv64 = [fp4.dequantize(c.view(torch.uint8), x.view(torch.uint8)).double() for c, x in ((k, ks), (v, vs))]
        else:
            k, v = k.to(dtype), v.to(dtype)
            self.kv64 = [k.double(), v.double()]
        self.k, self.v = k, v
        tables = torch.zeros((len(need), max(need) + 1), dtype=torch.long)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = torch.tensor(ids[at : at + n])
            at += n
        self.true_tables = tables.clone()
        if poison:
            self._poison(tables, kv, nb - 1, rng)
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        i64 = lambda x: torch.tensor(x, dtype=torch.long, device=dev)  # noqa: E731
        self.meta = AttentionMetadata(i64([0] * starts[-1]), tables.to(dev), i64([n + c for n, c in zip(q_lens, ctx)]),
                                      i64(q_lens), i64(starts), 0, max(q_lens))  # fmt: skip
        self.starts = starts
        self.q = torch.randn((starts[-1], H, D), generator=g, device=dev).to(dtype)

    def _nan(self, kv, blk, off):
        for t in (self.k, self.v):
            if kv == "own":
                t[blk, off] = float("nan")
            elif kv == "e4m3":
                t.view(torch.uint8)[blk, off] = 0x7F
        if kv == "fp4":
            for t in self.kwargs.values():
                t.view(torch.uint8)[blk, off] = 255

    def _poison(self, tables, kv, nan_page, rng):
        for off in range(self.bs):
            self._nan(kv, nan_page, off)
        for i, (n, c) in enumerate(zip(self.q_lens, self.ctx)):
            lo = c + 1 - self.window  # the first row's first key
            for page in range(-(-(n + c) // self.bs)):
                toks = range(page * self.bs, (page + 1) * self.bs)
                hidden = [t for t in toks if (self.sinks <= t < lo) or t >= n + c]
                if len(hidden) == self.bs:
                    tables[i, page] = rng.choice([nan_page, -1, 10**12, nan_page + 1])
                else:
                    for t in hidden:
                        self._nan(kv, int(self.true_tables[i, page]), t % self.bs)

    def forward(self, **kw):
        return HipAttention.forward(self.q, self.k, self.v, self.meta, self.scale, window=self.window, sinks=self.sinks,
                                    **self.kwargs, **kw)  # fmt: skip

    def want(self):
        """(out, sum_j p_j |v_j|) in 64 bits."""
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.q.device)
        mag = torch.zeros_like(out)
        G = self.H // self.Hkv
        for i, (n, c) in enumerate(zip(self.q_lens, self.ctx)):
            pages = self.true_tables[i, : -(-(n + c) // self.bs)].to(self.q.device)
            k, v = (x[pages].flatten(0, 1)[: n + c] for x in self.kv64)
            j = torch.arange(n + c, device=self.q.device)
            p = c + torch.arange(n, device=self.q.device)[:, None]
            seen = (j <= p) & ((p - j < self.window) | (j < self.sinks))
            rows = slice(self.starts[i], self.starts[i + 1])
            for h in range(self.H):
                s = self.q[rows, h].double() @ k[:, h // G].t().contiguous() * self.scale
                w = torch.softmax(s.masked_fill(~seen, -float("inf")), dim=-1)
                out[rows, h] = w @ v[:, h // G].contiguous()
                mag[rows, h] = w @ v[:, h // G].abs().contiguous()
        return out, mag

    def check(self, got):
        want, mag = self.want()
        if self.q.dtype == torch.float32:
            bound = 2.0**-10 * mag
        else:
            u = HALF_STEP[self.q.dtype]
            bound = (u + 2.0**-9) * mag + 2 * u * want.abs() + 8 * 2.0**-25
        err = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        assert (err <= bound).all(), f"{float((err - bound).max()):.3e} past the bound, max error {float(err.max()):.3e}"


DECODES = [0, 1, 14, 15, 16, 31, 32, 33, 62, 63, 64, 65, 95, 127, 128, 200, 511, 900, 1500]


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (32, 0), (33, 31), (64, 33), (100, 100), (700, 5)])
def test_decode(hip_device, kv, D, window, sinks):
    """One new token a sequence, lengths around chunks and windows; the small windows in one workgroup a sequence."""
    dtype = torch.float16 if D == 64 else torch.bfloat16
    b = Batch(hip_device, [1] * len(DECODES), DECODES, 8, 2, D, 16, window, sinks, dtype, kv, seed=window + sinks)
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("H,Hkv,D,window,sinks", [(32, 8, 128, 1100, 4), (8, 8, 64, 2000, 0), (28, 4, 128, 1500, 70), (16, 1, 64, 1200, 1)])
def test_decode_long(hip_device, kv, H, Hkv, D, window, sinks):
    """Windows past one workgroup's keys: split over units and merged."""
    ctx = [5000, 0, 1099, 1100, 1101, 1200, 2047, 3333, 6000, 77, 2500, 1999]
    b = Batch(hip_device, [1] * len(ctx), ctx, H, Hkv, D, 32, window, sinks, torch.bfloat16, kv, seed=H)
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("q,H,Hkv,D", [(2, 32, 8, 128), (5, 32, 8, 128), (8, 16, 4, 64), (11, 32, 8, 64), (15, 32, 8, 128), (1, 48, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(3, 0), (40, 6), (1030, 40)])
def test_verify(hip_device, kv, q, H, Hkv, D, window, sinks):
    """Several new tokens a sequence, one to four tiles of rows; some sequences with fewer, one with none."""
    ctx = [0, 3, 30, 64, 500, 1029, 1100, 2600]
    q_lens = [q, 1, q, max(1, q - 1), q, q, 0, q]
    b = Batch(hip_device, q_lens, ctx, H, Hkv, D, 16, window, sinks, torch.float16, kv, seed=q)
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 3), (96, 40), (256, 0), (300, 130), (1000, 4)])
def test_chunks(hip_device, kv, D, window, sinks):
    """Prompt chunks alone: tiles that start before, in and behind the window, ragged ends."""
    b = Batch(hip_device, [130, 17, 333, 64, 700], [0, 40, 500, 1025, 0], 8, 2, D, 16, window, sinks, torch.bfloat16, kv,
              seed=window)  # fmt: skip
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("H,Hkv,D,dec", [(32, 8, 128, 3), (28, 4, 64, 40), (20, 4, 128, 3), (24, 1, 64, 5)])
@pytest.mark.parametrize("window,sinks", [(30, 1), (600, 64)])
def test_mixed(hip_device, kv, H, Hkv, D, dec, window, sinks):
    """Decodes beside chunks, groups of 4, 5, 7 and 24 heads, in one launch and apart."""
    ctx = [(37 * i) % 900 for i in range(dec)] + [700, 0]
    b = Batch(hip_device, [1] * dec + [211, 90], ctx, H, Hkv, D, 32, window, sinks, torch.bfloat16, kv, seed=dec)
    b.check(b.forward())


def test_many_decodes_beside_a_chunk(hip_device):
    """A decode part that goes ahead in its own launch, whose last workgroups plan the chunks."""
    rng = random.Random(5)
    ctx = [rng.randint(0, 2500) for _ in range(150)] + [2000, 100]
    b = Batch(hip_device, [1] * 150 + [300, 70], ctx, 16, 8, 64, 16, 1500, 33, seed=1)
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
def test_long_sinks_and_far_windows(hip_device, kv):
    """More sinks than the 64 chunks that a walk's page window holds, decoded and as a chunk far behind them."""
    for q_lens, ctx in (([1, 1, 3], [9000, 2100, 7000]), ([150, 1], [9000, 8000])):
        b = Batch(hip_device, q_lens, ctx, 4, 2, 128, 16, 100, 2500, torch.bfloat16, kv, seed=len(q_lens))
        b.check(b.forward())


@pytest.mark.parametrize("dtype,D,bs,H,Hkv", [(torch.float32, 64, 16, 4, 2), (torch.float32, 128, 10, 4, 4), (torch.bfloat16, 96, 16, 6, 2),
                                              (torch.float16, 128, 24, 4, 1), (torch.bfloat16, 64, 16, 65, 1)])  # fmt: skip
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 7), (130, 65)])
def test_vector_kernel(hip_device, dtype, D, bs, H, Hkv, window, sinks):
    """The shapes that the matrix kernels do not tile."""
    b = Batch(hip_device, [1, 9, 1, 20], [0, 0, 383, 200], H, Hkv, D, bs, window, sinks, dtype, seed=D)
    b.check(b.forward())


@pytest.mark.parametrize("q_lens,ctx", [([1, 1], [300, 20]), ([1, 1], [5000, 900]), ([200, 1], [900, 70])])
def test_reaching_window_is_the_plain_call(hip_device, q_lens, ctx):
    """A window that no sequence outgrows: the bits of the call without one."""
    b = Batch(hip_device, q_lens, ctx, 8, 2, 128, 16, 1, 0, poison=False)
    plain = HipAttention.forward(b.q, b.k, b.v, b.meta, b.scale)
    keys = b.meta.block_tables.shape[1] * b.bs
    for window, sinks in ((keys, 0), (keys - 40, 40), (2**40, 2**40)):
        b.window, b.sinks = window, sinks
        assert torch.equal(b.forward(), plain)
    b.window, b.sinks = keys - 1, 0  # the windowed kernels, with everything in the window
    b.check(b.forward())


@pytest.mark.parametrize("kv", ["own", "fp4"])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_signs_of_the_scale(hip_device, kv, scale):
    for q_lens, ctx in (([1, 4], [90, 300]), ([70], [200])):
        b = Batch(hip_device, q_lens, ctx, 4, 2, 64, 16, 33, 2, kv=kv)
        b.scale = scale
        b.check(b.forward())


def test_strided_tensors_and_out(hip_device):
    """q and out as slices of wider rows, caches with a head's tokens together; what lies beside stays as it was."""
    b = Batch(hip_device, [1, 40, 3], [100, 20, 300], 8, 2, 64, 16, 50, 4)
    plain = b.forward()
    wide = torch.zeros((44, 10, 64), dtype=b.q.dtype, device=hip_device)
    wide[:, 1:9] = b.q
    b.q = wide[:, 1:9]
    b.k, b.v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (b.k, b.v))
    out = torch.full((46, 10, 64), 7.0, dtype=b.q.dtype, device=hip_device)
    got = b.forward(out=out[:44, 1:9])
    b.check(got)
    assert torch.equal(got, plain)
    assert (out[44:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 9] == 7).all()


def test_graph_replays(hip_device):
    """Captured calls follow the lengths of each replay, eager work between them."""
    small = Batch(hip_device, [1] * 6, [10, 500, 40, 700, 0, 90], 8, 2, 128, 16, 64, 4, seed=1, poison=False)
    long = Batch(hip_device, [1] * 6, [10, 5000, 40, 3000, 0, 1900], 8, 2, 128, 16, 1400, 4, seed=2, poison=False)
    mixed = Batch(hip_device, [1, 60, 1], [900, 100, 40], 8, 2, 128, 16, 100, 40, seed=3, poison=False)
    batches = [small, long, mixed]
    for b in batches:
        b.forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [b.forward() for b in batches]
    for step in range(3):
        for b in batches:
            b.meta.seq_lens -= (b.meta.seq_lens > b.meta.query_lens + 3 * step).long() * step  # shorter, same pages
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        eager = [b.forward() for b in batches]
        torch.cuda.synchronize()
        for a, e, b in zip(got, eager, batches):
            assert torch.equal(a, e)
            assert torch.isfinite(a).all()
    for b in batches:
        b.ctx = (b.meta.seq_lens - b.meta.query_lens).tolist()
        b.check(b.forward())


def test_no_sequences_and_refusals(hip_device):
    b = Batch(hip_device, [1], [30], 4, 2, 64, 16, 8, 0)
    empty = b.q[:0]
    assert HipAttention.forward(empty, b.k, b.v, b.meta, b.scale, window=8).shape == empty.shape
    for window, sinks in ((0, 0), (-1, 0), (2.5, 0), (8, -1), (None, 1)):
        with pytest.raises(ValueError):
            HipAttention.forward(b.q, b.k, b.v, b.meta, b.scale, window=window, sinks=sinks)
    with pytest.raises(ValueError):
        HipAttention.forward(b.q.cpu(), b.k, b.v, b.meta, b.scale, window=8)
    with pytest.raises(ValueError):
        HipAttention.forward(b.q.float(), b.k, b.v, b.meta, b.scale, window=8)


@pytest.mark.parametrize("kv", ["own", "e4m3", "fp4"])
@pytest.mark.parametrize("q_lens,ctx,H,D,window,sinks", [
    ([3000], [0], 32, 128, 512, 0), ([2000], [0], 32, 128, 500, 4), ([5000], [0], 32, 128, 2048, 0), ([512], [3001], 32, 128, 1000, 70),
    ([2900, 900, 1], [100, 3000, 2000], 32, 64, 300, 33), ([1000, 900] + [1] * 12, [2000, 3000] + [1700] * 12, 40, 128, 1024, 64),
])  # fmt: skip
def test_prompts_that_fill_the_launch(hip_device, kv, q_lens, ctx, H, D, window, sinks):
    """Tiles of two and of three to a wave, whole to a unit and split between units."""
    b = Batch(hip_device, q_lens, ctx, H, 8, D, 16, window, sinks, torch.bfloat16, kv, seed=len(q_lens) + window)
    b.check(b.forward())


@pytest.mark.parametrize("q_lens,ctx,H,window,sinks", [([4000], [0], 32, 300, 0), ([3001], [500], 32, 2000, 4), ([300, 900], [0, 3000], 56, 700, 70)])
def test_prompts_over_heads_of_64(hip_device, q_lens, ctx, H, window, sinks):
    b = Batch(hip_device, q_lens, ctx, H, 8, 64, 16, window, sinks, torch.float16, seed=window)
    b.check(b.forward())
