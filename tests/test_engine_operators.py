"""The engine with normed and partly rotated heads, sliding windows with sinks and projections in 4 bits: norm_rope_and_cache,
the windowed attention and linear4 as the steps of a model run them together, against the whole model in 64 bits.

On the CPU plain torch runs the same stages; on the GPU the HIP backend runs eagerly, in piecewise graphs and in decode
graphs, over pools of every format."""

from __future__ import annotations

import math
from dataclasses import replace

import pytest
import torch

from kvserve_amd import HipAttention, Weight4
from kvserve_amd.attention import FP4, FP8
from kvserve_amd.engine import LLAMA_3_2_1B, ModelConfig, build_model
from kvserve_amd.engine.model import rope_inv_freq
from kvserve_amd.engine.runner import Batcher, ModelRunner, Sequence
from oracle import fp4, fp8
from tests.engine_backends import TorchRefAttention

ALL = ModelConfig(
    vocab_size=1024, hidden_size=512, intermediate_size=640, num_layers=3, num_heads=8, num_kv_heads=2, head_dim=64,
    rope_scaling=LLAMA_3_2_1B.rope_scaling, tie_word_embeddings=True, qk_norm=True, rotary_dim=32, rope_interleaved=True,
    sliding_window=24, attention_sinks=3, full_layers=(1,),
)  # fmt: skip
CONFIGS = {
    "all": ALL,
    "halves": replace(ALL, rope_interleaved=False, attention_sinks=0),
    "window": replace(ALL, qk_norm=False, rotary_dim=None, rope_interleaved=False, full_layers=()),
    "norms": replace(ALL, rotary_dim=None, sliding_window=None, attention_sinks=0),
}
PROMPTS = [[(31 * i + 7 * n) % 1000 for i in range(n)] for n in (5, 37, 130, 1, 16, 25)]
STEPS = 5


class WindowedTorch(TorchRefAttention):
    """write_kv and forward with a window, sequence by sequence in fp32."""

    @staticmethod
    def forward(q, k_cache, v_cache, meta, scale, out=None, window=None, sinks=0) -> torch.Tensor:
        res = torch.empty_like(q)
        group = q.shape[1] // k_cache.shape[2]
        for s, n in enumerate(meta.seq_lens.tolist()):
            first, last = meta.query_start_loc[s : s + 2].tolist()
            pages = meta.block_tables[s, : -(-n // k_cache.shape[1])]
            k, v = (c[pages].flatten(0, 1)[:n].float().repeat_interleave(group, 1) for c in (k_cache, v_cache))
            p = torch.arange(n - (last - first), n)[:, None]
            j = torch.arange(n)[None]
            seen = (j <= p) if window is None else (j <= p) & ((p - j < window) | (j < sinks))
            score = torch.einsum("qhd,khd->hqk", q[first:last].float(), k) * scale
            prob = score.masked_fill(~seen[None], -math.inf).softmax(-1)
            res[first:last] = torch.einsum("hqk,khd->qhd", prob, v).to(q.dtype)
        return res


def _model(cfg, device, dtype, backend, group=None, **kw):
    model = build_model(cfg, device, dtype, 256, backend=backend, std=0.06, seed=5, weight4_group=group, **kw)
    gen = torch.Generator(device="cpu").manual_seed(11)
    for lw in model.w.layers:
        lw.k_scale, lw.v_scale = 1 / 16, 1 / 64  # of an E4M3 pool
        if cfg.qk_norm:
            for name in ("q_norm", "k_norm"):  # scores of a spread of 4 or so
                setattr(lw, name, (1 + torch.rand(cfg.head_dim, generator=gen)).to(device, dtype))
    return model


def _rounded(x: torch.Tensor, scale: float, pool) -> torch.Tensor:
    """x [n, heads, D] as a pool of that type holds it."""
    if pool == FP8:
        return fp8.dequantize(fp8.quantize(x, scale), scale).double()
    return fp4.dequantize(*fp4.quantize(x)).double() if pool == FP4 else x


def _exact(model, tokens: list[int], pool=None) -> torch.Tensor:
    """The model's logits [len(tokens), vocab] in 64 bits, the whole sequence at once, over keys and values as the pool
    rounds them."""
    cfg, w = model.cfg, model.w
    f = lambda t: (t.dequantize(torch.float64) if isinstance(t, Weight4) else t.double()).cpu()  # noqa: E731
    norm = lambda x, g: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * (1.0 if g is None else f(g))  # noqa: E731
    n, D = len(tokens), cfg.head_dim
    rot = cfg.rotary_dim or D
    angle = torch.arange(n)[:, None].double() * rope_inv_freq(cfg).double()
    pairs = torch.arange(rot).view(-1, 2) if cfg.rope_interleaved else torch.arange(rot).view(2, -1).t()

    def turn(x):  # [n, heads, D]
        y = x.clone()
        for i, (a, b) in enumerate(pairs.tolist()):
            c, s = angle[:, i, None].cos(), angle[:, i, None].sin()
            y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        return y

    p, j = torch.arange(n)[:, None], torch.arange(n)[None]
    x = f(w.embed)[torch.tensor(tokens)]
    for i, lw in enumerate(w.layers):
        qkv = (norm(x, lw.attn_norm) @ f(lw.wqkv).t()).view(n, -1, D)
        q, k, v = qkv.split([cfg.num_heads, cfg.num_kv_heads, cfg.num_kv_heads], 1)
        if cfg.qk_norm:
            q, k = norm(q, lw.q_norm), norm(k, lw.k_norm)
        q, k = turn(q), turn(k)
        k, v = _rounded(k, lw.k_scale, pool), _rounded(v, lw.v_scale, pool)
        k, v = (t.repeat_interleave(cfg.num_heads // cfg.num_kv_heads, 1) for t in (k, v))
        seen = j <= p
        if cfg.sliding_window is not None and i not in cfg.full_layers:
            seen = seen & ((p - j < cfg.sliding_window) | (j < cfg.attention_sinks))
        score = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(D)
        o = torch.einsum("hqk,khd->qhd", score.masked_fill(~seen, -math.inf).softmax(-1), v).flatten(1)
        x = x + o @ f(lw.wo).t()
        g, u = (norm(x, lw.mlp_norm) @ f(lw.w_gate_up).t()).chunk(2, -1)
        x = x + (g * torch.sigmoid(g) * u) @ f(lw.w_down).t()
    return norm(x, w.final_norm) @ f(w.lm_head).t()


def _run(runner, cfg) -> list[tuple[list[int], torch.Tensor]]:
    """(tokens, logits of their last STEPS positions) of the prompts, generated in steps together."""
    rows = [[] for _ in PROMPTS]
    seqs = [Sequence(list(p)) for p in PROMPTS]
    orig = runner.model.logits
    for _ in range(STEPS):
        got = []
        runner.model.logits = lambda h: got.append(orig(h)) or got[-1]
        runner.execute([(s, s.pending) for s in seqs])
        for r, row in zip(rows, got[-1]):
            r.append(row)
    runner.model.logits = orig
    return [(s.tokens[:-1], torch.stack(r)) for s, r in zip(seqs, rows)]


def _error(model, got, pool=None) -> float:
    """rms of the logits' errors over their rms"""
    err = ref = 0.0
    for tokens, rows in got:
        want = _exact(model, tokens, pool)[-STEPS:]
        err += float((rows.double().cpu() - want).square().sum())
        ref += float(want.square().sum())
    return math.sqrt(err / ref)


@pytest.mark.parametrize("group", [None, 32])
@pytest.mark.parametrize("name", CONFIGS)
def test_cpu_matches_64_bits(name, group):
    """fp32 stages: 2^-24 at some hundred terms and steps, far below 1e-4."""
    dtype = torch.float32 if group is None else torch.bfloat16
    model = _model(CONFIGS[name], "cpu", dtype, WindowedTorch, group)
    if group is not None:  # the packed weights in fp32 stages
        model.dtype = torch.float32
        model.w.embed, model.w.final_norm = model.w.embed.float(), model.w.final_norm.float()
        model.w.lm_head = model.w.embed
        for lw in model.w.layers:
            lw.attn_norm, lw.mlp_norm = lw.attn_norm.float(), lw.mlp_norm.float()
            if lw.q_norm is not None:
                lw.q_norm, lw.k_norm = lw.q_norm.float(), lw.k_norm.float()
    assert _error(model, _run(ModelRunner(model, num_blocks=96, max_model_len=256), model.cfg)) < 1e-4


def test_every_option_moves_the_logits():
    """... by far more than the errors that the tests below allow."""
    tokens = PROMPTS[2]
    base = _model(ALL, "cpu", torch.float32, WindowedTorch)
    want = _exact(base, tokens)
    for over in ({"qk_norm": False}, {"rotary_dim": None}, {"rope_interleaved": False}, {"sliding_window": None, "attention_sinks": 0},
                 {"attention_sinks": 0}, {"full_layers": ()}, {"sliding_window": 20}):  # fmt: skip
        base.cfg = replace(ALL, **over)
        other = _exact(base, tokens)
        assert float((other - want).norm() / want.norm()) > 0.08, over


def test_chunks_give_the_whole_prompts_tokens():
    out = []
    for budget in (2048, 7):
        r = ModelRunner(_model(ALL, "cpu", torch.float32, WindowedTorch), num_blocks=96, max_model_len=256, token_budget=budget)
        b = Batcher(r)
        seqs = [b.submit(p, 4) for p in PROMPTS]
        b.drain()
        out.append([s.generated for s in seqs])
    assert out[0] == out[1]


def test_refusals():
    for over in ({"sliding_window": 0}, {"sliding_window": None}, {"attention_sinks": -1}):
        with pytest.raises(ValueError):
            _model(replace(ALL, **over), "cpu", torch.float32, WindowedTorch)
    with pytest.raises(ValueError):
        ALL.to_hf_dict()
    with pytest.raises(ValueError):
        _model(ALL, "cpu", torch.float32, WindowedTorch, fused_rope=True)
    with pytest.raises(ValueError):  # 4 bits of fp32 weights
        _model(ALL, "cpu", torch.float32, WindowedTorch, 32)


# Rounding to bf16, rms 2^-9 / sqrt(3) relative each, some 12 times a layer along a token's path and once more for the logits:
# sqrt(3 * 12 + 2) 2^-9 / sqrt(3) = 0.7%, and the layers pass it on with a gain of 2 or so; 4% allowed. A pool rounds keys and
# values that are off by that d = 1% or so, and where one crosses a boundary it moves by a step s: rms sqrt(d s) of the
# element, 3.5% for E4M3's s of an eighth, 5.5% for MXFP4's of 0.3. Scores spread by 2.3, so a probability moves by 2.3 times
# that, and an attention output by both together, 9% and 14%, in each of three layers, where it adds less than half to the
# stream: 7% and 12%, and half as much again allowed.
POOLS = {"bf16": (None, 0.04), "e4m3": (FP8, 0.04 + 0.11), "mxfp4": (FP4, 0.04 + 0.18)}


@pytest.mark.gpu
@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("name", CONFIGS)
def test_gpu_matches_64_bits(hip_device, name, pool):
    """4-bit projections (groups of 128), eager steps and graphs."""
    dtype, tol = POOLS[pool]
    model = _model(CONFIGS[name], hip_device, torch.bfloat16, HipAttention, 128)
    errs = []
    for graphs in (False, True):
        r = ModelRunner(model, num_blocks=96, max_model_len=256, kv_cache_dtype=dtype, decode_graphs=graphs,
                        piecewise_graphs=graphs, max_graph_batch=8, max_piecewise_tokens=256)  # fmt: skip
        errs.append(_error(model, _run(r, model.cfg), dtype))
        del r
    assert max(errs) < tol, errs
    assert abs(errs[0] - errs[1]) < 0.02  # the same arithmetic, sums in other orders


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_fused_path_matches_the_separate_one(hip_device, dtype):
    """norm_rope_and_cache against norm, rotation and write_kv one by one, 16-bit projections."""
    errs = []
    for fused in (True, False):
        model = _model(ALL, hip_device, dtype, HipAttention, fused_rope=fused)
        errs.append(_error(model, _run(ModelRunner(model, num_blocks=96, max_model_len=256), model.cfg)))
    assert max(errs) < (0.04 if dtype == torch.bfloat16 else 0.005), errs
