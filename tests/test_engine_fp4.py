"""The engine over an MXFP4 KV pool, with log probabilities of what it generates and of its prompts: the quantising RoPE
and cache write, the attention over the packed pages and the pass over the logits as a serving step runs them together.

On the CPU the pool's tensors go through a backend that writes with the 64-bit definition of the format and attends over
the values it decodes; on the GPU the HIP backend runs eagerly, in piecewise graphs and in decode graphs."""

from __future__ import annotations

import math

import pytest
import torch

from kvserve_amd import HipAttention, fp4_caches, token_logprobs
from kvserve_amd.attention import FP4
from kvserve_amd.engine import LLAMA_3_1_8B, LLAMA_3_2_1B, ModelConfig
from kvserve_amd.engine.model import build_model
from kvserve_amd.engine.runner import Batcher, KVPool, ModelRunner, Sequence
from oracle import fp4, torch_reference
from tests.engine_backends import TorchRefAttention

SMALL = ModelConfig(
    vocab_size=2048, hidden_size=512, intermediate_size=1536, num_layers=4, num_heads=8, num_kv_heads=2, head_dim=64,
    rope_scaling=LLAMA_3_2_1B.rope_scaling, tie_word_embeddings=True,
)  # fmt: skip
TINY = ModelConfig(vocab_size=300, hidden_size=64, intermediate_size=96, num_layers=2, num_heads=4, num_kv_heads=2,
                   head_dim=32, tie_word_embeddings=True)  # fmt: skip

PROMPTS = [[(31 * i + 7) % 300 for i in range(n)] for n in (5, 37, 130, 1, 16)]


class OracleFP4Attention(TorchRefAttention):
    """write_kv stores the format's 64-bit quantisation, forward attends in fp32 over the decoded caches."""

    name = "torch-fp4"

    @staticmethod
    def write_kv(k_cache, v_cache, k, v, slots, k_scale, v_scale) -> None:
        for cache, scales, x in ((k_cache, k_scale, k), (v_cache, v_scale, v)):
            code, s = (t.to(cache.device) for t in fp4.quantize(x))
            bs = cache.shape[1]
            cache.view(torch.uint8)[slots // bs, slots % bs] = code
            scales.view(torch.uint8)[slots // bs, slots % bs] = s

    @staticmethod
    def forward(q, k_cache, v_cache, meta, scale, out=None, k_scale=None, v_scale=None) -> torch.Tensor:
        kd, vd = (fp4.dequantize(c.view(torch.uint8), s.view(torch.uint8)).float()
                  for c, s in ((k_cache, k_scale), (v_cache, v_scale)))  # fmt: skip
        res = torch_reference.forward(q.float(), kd, vd, meta.block_tables, meta.seq_lens, meta.query_lens, scale,
                                      meta.q_gather, meta.q_valid).to(q.dtype)  # fmt: skip
        if out is not None:
            out.copy_(res)
            return out
        return res


def _runner(cfg, device, dtype, backend, **kw):
    kw.setdefault("kv_cache_dtype", FP4)
    model = build_model(cfg, device, dtype, 512, backend=backend, std=0.06)
    return ModelRunner(model, num_blocks=96, max_model_len=512, **kw)


def _all_logits(runner, tokens: list[int]) -> torch.Tensor:
    """fp32 logits of every position of one prompt, from forward passes of its own within the runner's budget."""
    seq, got = Sequence(list(tokens)), []
    while seq.pending:
        got.append(runner.model.logits(runner._forward([(seq, min(seq.pending, runner.token_budget))], eager=True)))
    runner.release(seq)
    return torch.cat(got)


def test_pool_holds_packed_pages_and_sizes_them():
    r = _runner(TINY, "cpu", torch.float32, OracleFP4Attention)
    assert len(r.kv_caches) == 2
    for k, v, ks, vs in r.kv_caches:
        assert k.shape == v.shape == (97, 16, 2, 16) and ks.shape == vs.shape == (97, 16, 2, 1)
        assert k.dtype == FP4 and ks.dtype == torch.float8_e8m0fnu
        assert k.stride() == fp4_caches(97, 16, 2, 32, "cpu")[0].stride()
    model = build_model(TINY, "cpu", torch.float32, 512)
    per_block = 2 * 2 * 16 * 2 * (16 + 1)
    assert KVPool.blocks_in(model, per_block * 10 / 2**30, 16, FP4) == 10
    dense = 2 * LLAMA_3_1_8B.head_dim
    assert dense / (LLAMA_3_1_8B.head_dim / 2 + LLAMA_3_1_8B.head_dim / 32) == pytest.approx(3.7647, abs=1e-4)


def test_head_sizes_off_32_are_refused():
    cfg = ModelConfig(vocab_size=64, hidden_size=32, intermediate_size=32, num_layers=1, num_heads=2, num_kv_heads=1,
                      head_dim=16, tie_word_embeddings=True)  # fmt: skip
    with pytest.raises(ValueError, match="32s"):
        _runner(cfg, "cpu", torch.float32, OracleFP4Attention)


def test_chunks_over_the_packed_pool_give_the_whole_prompts_tokens():
    """A row's bytes depend on that row alone, so chunked steps attend over the same cache as one step."""
    out = {}
    for budget in (2048, 7):
        r = _runner(TINY, "cpu", torch.float32, OracleFP4Attention, token_budget=budget)
        b = Batcher(r)
        seqs = [b.submit(p, 6) for p in PROMPTS]
        b.drain()
        out[budget] = [s.generated for s in seqs]
        assert r.pool.free_blocks == 96
    assert out[2048] == out[7]


@pytest.mark.parametrize("budget", [2048, 11])
def test_score_on_the_cpu_matches_log_softmax(budget):
    r = _runner(TINY, "cpu", torch.float32, TorchRefAttention, kv_cache_dtype=None, token_budget=budget)
    got = r.score(PROMPTS, top=3)
    assert r.pool.free_blocks == 96
    for p, lp in zip(PROMPTS, got):
        want = _all_logits(r, p).double().log_softmax(-1)[:-1]
        assert lp.logprobs.shape == (len(p) - 1,) and lp.top_ids.shape == (len(p) - 1, 3)
        if len(p) > 1:
            # fp32 logits of two passes: hidden states differ by rounding, 2^-24 times some thousand terms
            torch.testing.assert_close(lp.logprobs.double(), want.gather(1, torch.tensor(p[1:])[:, None])[:, 0],
                                       atol=1e-3, rtol=0)  # fmt: skip
            torch.testing.assert_close(lp.entropy.double(), -(want.exp() * want).sum(-1), atol=1e-3, rtol=0)
            torch.testing.assert_close(lp.top_logprobs.double(), want.topk(3).values, atol=1e-3, rtol=0)


def test_generated_tokens_carry_their_log_probabilities():
    r = _runner(TINY, "cpu", torch.float32, TorchRefAttention, kv_cache_dtype=None)
    seqs = [Sequence(list(p)) for p in PROMPTS]
    for step in range(3):
        r.execute([(s, s.pending) for s in seqs], logprobs=2)
    r.execute([(s, s.pending) for s in seqs])  # not asked for: nothing added
    for s in seqs:
        assert len(s.logprobs) == 3 and len(s.generated) == 4
        want = _all_logits(r, s.tokens).log_softmax(-1)
        for i, (own, top) in enumerate(s.logprobs):
            tok = s.generated[i]
            assert own == pytest.approx(want[s.prompt_len - 1 + i, tok].item(), abs=1e-3)
            assert len(top) == 2 and top[tok] == own == max(top.values())


@pytest.mark.parametrize("kw", [{"num_blocks": 3}, {"num_blocks": 40, "max_seqs": 4}, {"num_blocks": 40, "token_budget": 5}])
def test_score_takes_what_the_pool_holds(kw):
    """More prompts than blocks, sequences or tokens of a step: in turns, each as if alone."""
    model = build_model(TINY, "cpu", torch.float32, 512, backend=TorchRefAttention, std=0.06)
    prompts = [[(7 * i + j) % 300 for j in range(1 + 5 * i % 37)] for i in range(30)]
    r = ModelRunner(model, block_size=16, max_model_len=512, **kw)
    got = r.score(prompts)
    assert r.pool.free_blocks == kw["num_blocks"]
    big = ModelRunner(model, num_blocks=40, block_size=16, max_model_len=512)
    for p, lp in zip(prompts, got):
        torch.testing.assert_close(lp.logprobs, big.score([p])[0].logprobs, atol=1e-3, rtol=0)


def test_score_of_a_prompt_past_the_pool():
    model = build_model(TINY, "cpu", torch.float32, 512, backend=TorchRefAttention, std=0.06)
    for budget in (2048, 7):
        r = ModelRunner(model, num_blocks=3, block_size=16, max_model_len=512, token_budget=budget)
        with pytest.raises(RuntimeError, match="exhausted"):
            r.score([[3] * 20, [1] * 49, [2] * 5])
        assert r.pool.free_blocks == 3


def test_refusals_leave_the_pool_whole():
    r = _runner(TINY, "cpu", torch.float32, TorchRefAttention, kv_cache_dtype=None)
    with pytest.raises(ValueError, match="at least one token"):
        r.score([[1, 2], []])
    with pytest.raises(ValueError, match="max_model_len"):
        r.score([[1, 2], [1] * 513])
    for n in (-1, 65):
        with pytest.raises(ValueError, match="logprobs must be"):
            r.execute([(Sequence([1, 2]), 2)], logprobs=n)
    assert r.pool.free_blocks == 96


@pytest.mark.parametrize("over,dtype,block,match", [
    ({}, torch.float32, 16, "bf16 or fp16"), ({"head_dim": 96}, torch.bfloat16, 16, "head sizes"),
    ({"head_dim": 32}, torch.float16, 16, "head sizes"), ({}, torch.bfloat16, 24, "blocks in 16s"),
    ({"num_heads": 65, "num_kv_heads": 1}, torch.bfloat16, 16, "query heads"),
])  # fmt: skip
def test_pools_that_the_backend_cannot_attend_over_are_refused(over, dtype, block, match):
    """At construction, not at the first step; the same model's 16-bit pool is as before."""
    cfg = ModelConfig(**{"vocab_size": 64, "hidden_size": 64, "intermediate_size": 32, "num_layers": 1, "num_heads": 4,
                         "num_kv_heads": 2, "head_dim": 64, "tie_word_embeddings": True, **over})  # fmt: skip
    model = build_model(cfg, "cpu", dtype, 64, backend=HipAttention)
    with pytest.raises(ValueError, match=match):
        ModelRunner(model, num_blocks=4, block_size=block, max_model_len=64, kv_cache_dtype=FP4)
    ModelRunner(model, num_blocks=4, block_size=block, max_model_len=64)


@pytest.mark.parametrize("group,head_dim,dtype", [(1, 64, torch.float16), (8, 128, torch.bfloat16), (64, 64, torch.bfloat16)])
def test_pools_that_the_backend_takes(group, head_dim, dtype):
    cfg = ModelConfig(vocab_size=64, hidden_size=64, intermediate_size=32, num_layers=1, num_heads=group, num_kv_heads=1,
                      head_dim=head_dim, tie_word_embeddings=True)  # fmt: skip
    model = build_model(cfg, "cpu", dtype, 64, backend=HipAttention)
    r = ModelRunner(model, num_blocks=4, block_size=32, max_model_len=64, kv_cache_dtype=FP4)
    assert r.kv_caches[0][0].shape == (5, 32, 1, head_dim // 2)


# -- on the GPU --------------------------------------------------------------------------------


def _logits_of(r, call):
    got = {}
    orig = r.model.logits
    r.model.logits = lambda h: got.setdefault("l", orig(h))
    try:
        call()
    finally:
        r.model.logits = orig
    return got["l"]


@pytest.mark.gpu
@pytest.mark.parametrize("fused_rope", [True, False])
def test_prefill_logits_match_the_definition(hip_device, fused_rope):
    """bf16 prefill over the packed pool against attention over the decoded 64-bit quantisation: within 5% of the
    logits' scale, as over the other cache types. (The two paths round K in bf16 before the cache or not at all, which
    moves single codes by a step of up to a sixth of their block's largest: four layers of 2^-3 at the worst and far
    less over sums of hundreds of keys.)"""
    logits = {}
    for name, backend in (("hip", HipAttention), ("torch", OracleFP4Attention)):
        model = build_model(SMALL, hip_device, torch.bfloat16, 512, backend=backend, seed=3,
                            fused_rope=fused_rope if name == "hip" else None)  # fmt: skip
        r = ModelRunner(model, num_blocks=96, max_model_len=512, kv_cache_dtype=FP4, decode_graphs=False,
                        piecewise_graphs=False)  # fmt: skip
        logits[name] = _logits_of(r, lambda r=r: r.prefill([Sequence(list(p)) for p in PROMPTS]))
    assert (logits["hip"] - logits["torch"]).abs().max() <= 0.05 * logits["torch"].abs().max()


@pytest.mark.gpu
def test_graphs_match_eager_steps(hip_device):
    """Decode graphs and piecewise steps over the packed pool give the eager steps' logits within 3% of their scale
    (bf16; the batch's padding moves the split of the key axis), step after step."""
    kw = dict(max_graph_batch=8, token_budget=256, max_piecewise_tokens=64)
    runners = [_runner(SMALL, hip_device, torch.bfloat16, HipAttention, **kw),
               _runner(SMALL, hip_device, torch.bfloat16, HipAttention, decode_graphs=False, piecewise_graphs=False, **kw)]
    seqs = [[Sequence(list(p)) for p in PROMPTS] for _ in runners]
    for r, s in zip(runners, seqs):
        r.prefill(s)
    late = [Sequence(list(PROMPTS[1])) for _ in runners]
    for step in range(6):
        outs = []
        for r, s, x in zip(runners, seqs, late):
            plan = [(q, 1) for q in s]
            if step == 2:
                plan.append((x, x.pending))
            outs.append(_logits_of(r, lambda r=r, plan=plan: r.execute(plan)))
        for g, e in zip(seqs[0] + late[:1], seqs[1] + late[1:]):  # both see the eager run's tokens
            g.tokens[-1] = e.tokens[-1]
        diff = (outs[0] - outs[1]).abs().max().item()
        assert diff <= 3e-2 * outs[1].abs().max().item(), (step, diff)
    assert runners[0].paths["decode_graph"] == 5 and runners[0].paths["piecewise"] >= 1, runners[0].paths


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [FP4, None], ids=["mxfp4", "16-bit"])
def test_log_probabilities_of_a_run(hip_device, kv):
    """Generation with log probabilities through graphs, and the same tokens scored as a prompt afterwards: each
    sequence's own log probabilities agree with the score of its text. Both come from bf16 logits of hidden states that
    differ by bf16 rounding over the layers (a decode step and a prefill of the same row), bounded as the graphs are:
    3% of the logits' scale, twice (the token's logit and the normaliser)."""
    r = _runner(SMALL, hip_device, torch.bfloat16, HipAttention, kv_cache_dtype=kv, max_graph_batch=8,
                token_budget=128, max_piecewise_tokens=64)  # fmt: skip
    b = Batcher(r)
    seqs = [b.submit(p, 5) for p in PROMPTS]
    tables = []
    while b.busy:
        b.step(logprobs=4)
        tables.append(r.pool.free_blocks)
    assert r.pool.free_blocks == 96 and min(tables) < 96 and r.paths["decode_graph"] >= 3
    scored = r.score([s.tokens for s in seqs], top=4)
    assert r.pool.free_blocks == 96
    for s, lp in zip(seqs, scored):
        assert len(s.logprobs) == 5 and lp.logprobs.shape == (len(s.tokens) - 1,)
        top = _all_logits(r, s.tokens).abs().max().item()
        for i, (own, best) in enumerate(s.logprobs):
            row = s.prompt_len - 1 + i
            assert abs(own - lp.logprobs[row].item()) <= 0.06 * top
            assert len(best) == 4 and best[s.generated[i]] == own == max(best.values())
            assert lp.entropy[row].item() <= math.log(SMALL.vocab_size) + 1e-4


@pytest.mark.gpu
def test_score_is_the_pass_over_the_heads_logits(hip_device):
    """One chunk: score's rows are token_logprobs of the very logits of that step, bit for bit."""
    r = _runner(SMALL, hip_device, torch.bfloat16, HipAttention, decode_graphs=False, piecewise_graphs=False)
    p = PROMPTS[2]
    got = r.score([p], top=5)[0]
    seq = Sequence(list(p))
    logits = r.model.logits(r._forward([(seq, len(p))], eager=True)).to(torch.bfloat16)
    want = token_logprobs(logits, torch.tensor(p[1:] + [0], device=hip_device), 5)
    for a, b in zip(got, want):
        assert torch.equal(a, b[:-1])


@pytest.mark.gpu
@pytest.mark.parametrize("live", [1, 3])
def test_score_beside_live_sequences(hip_device, live):
    """Sequences being generated keep their rows of the resident tables: prompts to score take turns on the others."""
    r = _runner(SMALL, hip_device, torch.bfloat16, HipAttention, decode_graphs=False, piecewise_graphs=False, max_seqs=4)
    seqs = [Sequence(list(p)) for p in PROMPTS[:live]]
    r.execute([(s, s.pending) for s in seqs])
    free = r.pool.free_blocks
    prompts = [PROMPTS[i % len(PROMPTS)][i:] + [7, 8] for i in range(10)]
    got = r.score(prompts, top=2)
    assert r.pool.free_blocks == free
    alone = _runner(SMALL, hip_device, torch.bfloat16, HipAttention, decode_graphs=False, piecewise_graphs=False)
    for p, lp in zip(prompts, got):
        # logits of two batches, bounded as the graphs are: 3% of their scale, twice (the token's and the normaliser)
        top = _all_logits(alone, p).abs().max().item()
        assert (lp.logprobs - alone.score([p])[0].logprobs).abs().max().item() <= 0.06 * top
    r.execute([(s, s.pending) for s in seqs])
    assert all(len(s.generated) == 2 for s in seqs)


# -- the model's pass over the head's logits without a GPU ------------------------------------------


def _cpu_token_logprobs(logits, tokens, top):
    """PagedLlama.token_logprobs where the head gives these logits."""
    model = build_model(TINY, "cpu", torch.float32, 512, backend=TorchRefAttention)
    model._linear = lambda x, w: logits
    return model.token_logprobs(torch.zeros(len(logits), TINY.hidden_size), tokens, top)[1]


def test_cpu_log_probabilities_of_special_rows():
    """As kvserve_amd.token_logprobs has them: NaN for a row with a NaN or a +inf or of -inf alone, and for a token
    outside the vocabulary; a logit of -inf adds nothing to the entropy; NaN counts as -inf in the order."""
    inf, nan = math.inf, math.nan
    x = torch.tensor([[0.0, nan, 2.0, 1.0], [0.0, inf, 2.0, 1.0], [-inf] * 4, [-inf, 0.0, -inf, 0.0], [0.0] * 4, [0.0] * 4])
    lp = _cpu_token_logprobs(x, torch.tensor([0, 1, 2, 0, 4, -1]), 4)
    for row in range(3):
        assert lp.logprobs[row].isnan() and lp.entropy[row].isnan() and lp.top_logprobs[row].isnan().all()
    assert lp.top_ids[:4].tolist() == [[2, 3, 0, 1], [1, 2, 3, 0], [0, 1, 2, 3], [1, 3, 0, 2]]
    # log 2 and log 4 in fp32: two roundings of exponentials and a logarithm
    assert lp.logprobs[3] == -inf and abs(lp.entropy[3].item() - math.log(2)) <= 2.0**-22
    assert lp.top_logprobs[3, 2:].tolist() == [-inf, -inf]
    assert lp.logprobs[4:].isnan().all() and (lp.entropy[4:] - math.log(4)).abs().max() <= 2.0**-21


def test_cpu_alternatives_are_ordered_by_their_logits():
    """Log probabilities of neighbouring logits round to one value beside a far larger one; the order is the logits'."""
    x = torch.zeros(2, 40)
    x[:, 7] = 100.0
    x[0, 20], x[0, 30] = 1.0, 1.0 + 2.0**-23
    lp = _cpu_token_logprobs(x, torch.tensor([7, 7]), 5)
    assert lp.top_logprobs[0, 1] == lp.top_logprobs[0, 2]
    assert lp.top_ids.tolist() == [[7, 30, 20, 0, 1], [7, 0, 1, 2, 3]]


@pytest.mark.parametrize("top", [-1, 65, 301])
def test_cpu_refuses_other_numbers_of_alternatives(top):
    r = _runner(TINY, "cpu", torch.float32, TorchRefAttention, kv_cache_dtype=None)
    with pytest.raises(ValueError, match="top must be 0 .. 64"):
        r.score([[1, 2, 3]], top=top)
    assert r.pool.free_blocks == 96
