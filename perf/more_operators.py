"""The steps of a layer with windowed attention, normed heads and 4-bit weights, as they are timed.

  rope    `HipAttention.norm_rope_and_cache` of a step's fused projection: the norms of every query and key head, the
          rotation of (part of) each head, and the write of keys and values into the paged cache.
  attend  `HipAttention.forward` with a sliding window and sinks: decoding sequences, drafts to verify, prompt chunks.
  linear  `linear4`: rows against a weight held in 4 bits with a scale and a zero point for every group along k.
  mlp     `linear4_silu_mul`: the gate and up projections of such a weight with SiLU(gate) * up.

`run` computes each operator in elementary torch operations where `own` is false, and calls the framework's operators
where it is true.

Sizes are those of the two Llama shapes the engine is configured for (1B: hidden 2048, 32 query heads over 8 kv heads of
64, MLP of 8192; 8B: hidden 4096, 32 over 8 of 128, MLP of 14336) and of the benchmark's workloads; the drawn ones spread
around them. Lengths follow from the case alone, values and physical block orders from the seed.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
SHAPES = {"1b": (32, 8, 64), "8b": (32, 8, 128)}  # query heads, kv heads, head size
K_SCALE, V_SCALE = 0.03125, 0.015625  # of E4M3 caches
EPS = 1e-6


# -- the cases -------------------------------------------------------------------------------------


def _attend(name: str | None = None, **kw) -> dict:
    """`decodes` sequences of `q` query tokens over lo .. hi cached tokens, then `chunks` sequences computing chunk_lo ..
    chunk_hi prompt tokens over ctx_lo .. ctx_hi cached ones. A token sees the last `window` tokens, itself among them,
    and the first `sinks`. `cache`: "own" (the queries' type) or "e4m3"."""
    c = {
        "kind": "attend", "dtype": "bf16", "cache": "own", "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16,
        "window": 4096, "sinks": 0, "decodes": 0, "q": 1, "lo": 0, "hi": 0, "chunks": 0, "chunk_lo": 0, "chunk_hi": 0,
        "ctx_lo": 0, "ctx_hi": 0, "lens": 0,
    }  # fmt: skip
    c.update(kw)
    return {"name": name, **c} if name else c


def _rope(name: str | None = None, **kw) -> dict:
    """The first `rotary` elements of each head are rotated, pairs (i, i + rotary / 2) or (2i, 2i + 1) where `interleaved`;
    `factor`: positions stretched for a longer context, with the attention factor in the tables."""
    c = {"kind": "rope", "dtype": "bf16", "model": "8b", "tokens": 1, "rotary": 128, "interleaved": False, "factor": 1.0}
    c.update(kw)
    return {"name": name, **c} if name else c


def _linear(name: str | None = None, kind: str = "linear", **kw) -> dict:
    """`rows` of x against a weight [n, k] in groups of `group`; kind "mlp": n = 2 * the MLP's width, gate rows first."""
    c = {"kind": kind, "dtype": "bf16", "rows": 1, "n": 4096, "k": 4096, "group": 128}
    c.update(kw)
    return {"name": name, **c} if name else c


def listed() -> list[dict]:
    return [
        # the rows of one decode step of a small model, eight users: bound by latency
        _rope("rope_1b_b8", model="1b", tokens=8, rotary=64),
        # a full step of prompts and decodes, half of each head rotated in neighbouring pairs, a stretched context
        _rope("rope_8b_2047_part", tokens=2047, rotary=64, interleaved=True, factor=8.0),
        # a small model answering a few short chats, some shorter than the window
        _attend("decode_1b_b8", dtype="fp16", head_dim=64, window=128, sinks=4, decodes=8, lo=63, hi=511),
        # a busy server's decode step over long contexts: most of each cache lies behind the window
        _attend("decode_8b_b64", window=4096, sinks=4, decodes=64, lo=1023, hi=16383),
        # speculative decoding over an E4M3 cache: five draft tokens verified per sequence
        _attend("verify_8b_b32_q5_e4m3", cache="e4m3", window=1024, decodes=32, q=5, lo=500, hi=12000),
        # a continuous-batching step: decodes, and chunks of two long prompts over what is cached
        _attend("mixed_8b", window=2048, sinks=64, decodes=24, lo=255, hi=8191, chunks=2, chunk_lo=900, chunk_hi=1024,
                ctx_lo=4000, ctx_hi=10000),
        # a long prompt computed in one step (the most arithmetic of the attention)
        _attend("prompt_8b_8191", window=1024, chunks=1, chunk_lo=8191, chunk_hi=8191),
        # a single user's decode step: one row against the output projection
        _linear("linear_1x4096x4096", rows=1, n=4096, k=4096),
        # a small model's down projection for an odd number of users, smaller groups
        _linear("linear_33x2048x8192_fp16", dtype="fp16", rows=33, n=2048, k=8192, group=64),
        # a chunk of a prompt through the fused QKV projection
        _linear("linear_500x6144x4096", rows=500, n=6144, k=4096),
        # the largest weight of a layer at eight users: what a decode step spends most on
        _linear("mlp_8x28672x4096", kind="mlp", rows=8, n=28672, k=4096),
        # the same for a batch that still shares each weight among few rows
        _linear("mlp_64x28672x4096", kind="mlp", rows=64, n=28672, k=4096),
    ]  # fmt: skip


def _log(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5)))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rope", "rope", "decode", "decode", "verify", "mixed", "chunks", "linear", "linear", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rope":
        model = rng.choice(["1b", "8b"])
        D = SHAPES[model][2]
        return _rope(dtype=dtype, model=model, tokens=_log(rng, 1, 4096), rotary=rng.choice([D, D, D // 2, D // 4]),
                     interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 32.0]))  # fmt: skip
    if kind in ("linear", "mlp"):
        group = rng.choice([32, 64, 128, 128])
        shapes = [(4096, 4096), (4096, 14336), (6144, 4096), (2048, 2048), (2048, 8192)]
        if kind == "mlp":
            n, k = rng.choice([(28672, 4096), (16384, 2048), (32 * _log(rng, 4, 800), 128 * _log(rng, 2, 32))])
        else:
            n, k = rng.choice(shapes + [(_log(rng, 100, 8200), group * rng.randint(3, 5000 // group))])
        rows = _log(rng, 1, min(640, 12_500_000_000 // (n * k)))
        return _linear(kind=kind, dtype=dtype, rows=rows, n=n, k=k, group=group)
    c = {"dtype": dtype, "cache": rng.choice(["own", "own", "e4m3"]), "head_dim": rng.choice([64, 128, 128]),
         "block": rng.choice([16, 16, 32]), "window": _log(rng, 32, 4096),
         "sinks": rng.choice([0, 4, rng.randint(1, 128)]), "lens": rng.randrange(1 << 20)}  # fmt: skip
    c["heads"], c["kv_heads"] = rng.choice([(32, 8), (32, 8), (32, 8), (32, 4), (16, 16)])
    most = 4_000_000 // c["kv_heads"]  # cached tokens of a batch at most
    seen = 2_000_000 // c["kv_heads"]  # tokens that a batch's windows hold at most
    if kind in ("decode", "verify"):
        n = _log(rng, 1, min(256, seen // (c["window"] + c["sinks"])))
        hi = min(_log(rng, 64, 16384), most // n)
        c.update(decodes=n, q=1 if kind == "decode" else rng.randint(2, 8), lo=rng.randint(1, hi), hi=hi)
    else:
        if kind == "mixed":
            n = _log(rng, 1, 48)
            hi = min(_log(rng, 64, 8192), most // n)
            c.update(decodes=n, lo=rng.randint(1, hi), hi=hi)
        c.update(chunks=_log(rng, 1, 4), ctx_hi=rng.choice([0, _log(rng, 1, 9000)]))
        pairs = 8_000_000 // c["chunks"]  # (query, key) pairs of a sequence at most
        c["chunk_hi"] = max(20, min(_log(rng, 20, 4000), pairs // (c["window"] + c["sinks"])))
        c["chunk_lo"] = rng.randint(20, c["chunk_hi"])
    return _attend(**c)


# -- inputs ----------------------------------------------------------------------------------------


def _normal(gen: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _channels(gen: torch.Generator, *shape: int) -> torch.Tensor:
    """Keys and activations have channels that are larger than others by a factor, the same for every token."""
    return torch.exp(0.7 * _normal(gen, *shape))


def _cache(gen: torch.Generator, blocks: int, block: int, kv_heads: int, head_dim: int, dtype: torch.dtype,
           factor, scale: float) -> torch.Tensor:  # fmt: skip
    """A cache as earlier steps left it."""
    c = torch.empty((blocks, block, kv_heads, head_dim), dtype=dtype, device=DEVICE)
    step = max(1, (1 << 26) // (block * kv_heads * head_dim))
    for b in range(0, blocks, step):
        x = _normal(gen, min(step, blocks - b), block, kv_heads, head_dim) * factor
        c[b : b + step] = (x / scale).clamp(-448, 448).to(dtype) if dtype == E4M3 else x.to(dtype)
    return c


def _prepare_rope(case: dict, seed: int) -> dict:
    """A step's tokens: consecutive positions of one prompt, in pages of a shuffled pool."""
    H, Hkv, D = SHAPES[case["model"]]
    T, bs, R, dtype = case["tokens"], 16, case["rotary"], DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    blocks = -(-T // bs) + 4
    order = list(range(blocks))
    random.Random(seed).shuffle(order)
    at = torch.arange(T, device=DEVICE)
    x = _normal(gen, T, H + 2 * Hkv, D)
    x[:, H : H + Hkv] *= _channels(gen, Hkv, D)
    angle = torch.arange(4 * T, device=DEVICE).double()[:, None] / case["factor"] * 500000.0 ** -(
        torch.arange(0, R, 2, device=DEVICE).double() / R
    )
    stretch = 0.1 * math.log(case["factor"]) + 1.0
    return {
        "case": case, "heads": H, "qkv": x.to(dtype).flatten(1), "positions": at + T * random.Random(seed + 1).randint(0, 3),
        "cos": (torch.cos(angle) * stretch).float(), "sin": (torch.sin(angle) * stretch).float(),
        "q_norm": (1.0 + 0.3 * _normal(gen, D)).to(dtype), "k_norm": (1.0 + 0.3 * _normal(gen, D)).to(dtype),
        "k_cache": _cache(gen, blocks, bs, Hkv, D, dtype, 1.0, 1.0), "v_cache": _cache(gen, blocks, bs, Hkv, D, dtype, 1.0, 1.0),
        "slots": torch.tensor(order, device=DEVICE)[at // bs] * bs + at % bs,
    }  # fmt: skip


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(query lengths, cached lengths) of an attend case, decoding sequences first."""
    rng = random.Random(case["lens"])
    q, ctx = [], []
    for _ in range(case["decodes"]):
        q.append(case["q"])
        ctx.append(rng.randint(case["lo"], case["hi"]))
    for _ in range(case["chunks"]):
        q.append(rng.randint(case["chunk_lo"], case["chunk_hi"]))
        ctx.append(rng.randint(case["ctx_lo"], case["ctx_hi"]))
    return q, ctx


def _prepare_attend(case: dict, seed: int) -> dict:
    q, ctx = _lengths(case)
    H, Hkv, D, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    need = [-(-(n + c) // bs) for n, c in zip(q, ctx)]
    blocks = sum(need) + 8
    ids = list(range(blocks))
    random.Random(seed).shuffle(ids)
    tables = torch.zeros((len(q), max(need)), dtype=torch.long)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = torch.tensor(ids[at : at + n])
        at += n
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    dtype = DTYPES[case["dtype"]]
    kv = E4M3 if case["cache"] == "e4m3" else dtype
    k = _cache(gen, blocks, bs, Hkv, D, kv, _channels(gen, Hkv, D), K_SCALE)
    v = _cache(gen, blocks, bs, Hkv, D, kv, 1.0, V_SCALE)
    # what the calls read of a step's metadata, under the names it has there
    meta = SimpleNamespace(
        block_tables=tables.to(DEVICE), seq_lens=torch.tensor([n + c for n, c in zip(q, ctx)], device=DEVICE),
        query_start_loc=torch.tensor(starts, device=DEVICE), max_query_len=max(q),
        max_seq_len=max(n + c for n, c in zip(q, ctx)),
    )  # fmt: skip
    scales = {"k_scale": K_SCALE, "v_scale": V_SCALE} if kv == E4M3 else {}
    return {"case": case, "k": k, "v": v, "scales": scales, "meta": meta, "scale": D**-0.5,
            "q": _normal(gen, starts[-1], H, D).to(dtype)}  # fmt: skip


def _prepare_linear(case: dict, seed: int) -> dict:
    n, k, group, dtype = case["n"], case["k"], case["group"], DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 25) // k)
    for r in range(0, n, step):
        c = (7.5 + 2.7 * _normal(gen, min(step, n - r), k)).round().clamp(0, 15).to(torch.uint8)
        codes[r : r + step] = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = (0.008 * torch.exp(0.3 * _normal(gen, n, k // group))).to(dtype)
    zeros = torch.randint(5, 11, (n, k // group), generator=gen, device=DEVICE, dtype=torch.uint8)
    s = {"case": case, "codes": codes, "scales": scales, "zeros": zeros,
         "x": (_normal(gen, case["rows"], k) * _channels(gen, k)).to(dtype)}  # fmt: skip
    if own:
        from kvserve_amd import Weight4

        s["weight"] = Weight4.pack(codes, scales, zeros)
    return s


# -- one pass --------------------------------------------------------------------------------------


def _run_rope(s: dict) -> dict:
    if own:
        from kvserve_amd import HipAttention

        q = HipAttention.norm_rope_and_cache(s["qkv"], s["positions"], s["cos"], s["sin"], s["k_cache"], s["v_cache"],
                                             s["slots"], s["heads"], s["q_norm"], s["k_norm"], EPS,
                                             s["case"]["interleaved"])  # fmt: skip
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    H, (_, bs, Hkv, D) = s["heads"], s["k_cache"].shape
    dtype, half = s["qkv"].dtype, s["cos"].shape[1]
    x = s["qkv"].float().unflatten(1, (-1, D))
    v = x[:, H + Hkv :]
    x = x[:, : H + Hkv]
    weight = torch.cat((s["q_norm"].expand(H, D), s["k_norm"].expand(Hkv, D))).float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    cos, sin = (s[n][s["positions"]][:, None] for n in ("cos", "sin"))
    rot, rest = x[..., : 2 * half], x[..., 2 * half :]
    if s["case"]["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    x = torch.cat((rot, rest), dim=-1).to(dtype)
    blk, off = s["slots"] // bs, s["slots"] % bs
    s["k_cache"][blk, off] = x[:, H:]
    s["v_cache"][blk, off] = v.to(dtype)
    return {"q": x[:, :H].contiguous(), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rows(cache: torch.Tensor, tables: torch.Tensor, keys: torch.Tensor, scale: float) -> torch.Tensor:
    """fp32 rows [n, Hkv, keys, D] of the sequences' tokens `keys` [n, keys]."""
    bs = cache.shape[1]
    blk, off = tables.gather(1, keys // bs), keys % bs
    if cache.dtype == E4M3:
        rows = cache.view(torch.uint8)[blk, off].view(E4M3).float() * scale
    else:
        rows = cache[blk, off].float()
    return rows.transpose(1, 2).contiguous()


def _plain_block(s: dict, first: int, last: int, begin: int, longest: int) -> torch.Tensor:
    """Attention of query tokens begin .. begin + longest - 1 of sequences first .. last - 1 (padded where they have
    fewer): [n, longest, H, D]."""
    meta, case = s["meta"], s["case"]
    H, Hkv, W, S = case["heads"], case["kv_heads"], case["window"], case["sinks"]
    G, D = H // Hkv, case["head_dim"]
    tables, lens, start = meta.block_tables[first:last], meta.seq_lens[first:last, None], meta.query_start_loc[first:last]
    n_q = (meta.query_start_loc[first + 1 : last + 1] - start)[:, None]
    at = begin + torch.arange(longest, device=DEVICE)
    rows = s["q"][(start[:, None] + at).clamp(max=len(s["q"]) - 1)].float()  # [n, longest, H, D]
    n = len(tables)
    q = rows.view(n, longest, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(n, Hkv, longest * G, D)
    pos = lens - n_q + at  # [n, longest]
    # the sinks, then the tokens that one of the rows has in its window
    base = (pos[:, :1] + 1 - W).clamp(min=S)
    reach = min(W + longest - 1, meta.max_seq_len)
    keys = torch.cat((torch.arange(S, device=DEVICE).expand(n, S), base + torch.arange(reach, device=DEVICE)), dim=1)
    seen = (keys[:, None] <= pos[..., None]) & ((keys[:, None] < S) | (keys[:, None] > pos[..., None] - W))
    seen = (seen & (at < n_q)[..., None]).repeat_interleave(G, dim=1)[:, None]  # [n, 1, longest G, keys]
    keys = torch.minimum(keys, lens - 1)
    p = torch.matmul(q, _rows(s["k"], tables, keys, K_SCALE).transpose(-1, -2).contiguous()) * s["scale"]
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp_(p.sub_(top.masked_fill(top == -math.inf, 0.0)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _rows(s["v"], tables, keys, V_SCALE)) / total.masked_fill(total == 0, 1.0)
    return out.view(n, Hkv, longest, G, D).permute(0, 2, 1, 3, 4).reshape(n, longest, H, D)


def _run_attend(s: dict) -> dict:
    case = s["case"]
    if own:
        from kvserve_amd import HipAttention

        return {"out": HipAttention.forward(s["q"], s["k"], s["v"], s["meta"], s["scale"], **s["scales"],
                                            window=case["window"], sinks=case["sinks"])}  # fmt: skip
    parts, n_dec = [], case["decodes"]
    step = max(1, (1 << 20) // ((case["window"] + case["sinks"] + 8) * case["kv_heads"]))
    for i in range(0, n_dec, step):
        parts.append(_plain_block(s, i, min(i + step, n_dec), 0, case["q"]).flatten(0, 1))
    q, _ = _lengths(case)
    for i in range(n_dec, len(q)):
        for b in range(0, q[i], 256):
            parts.append(_plain_block(s, i, i + 1, b, min(256, q[i] - b))[0])
    return {"out": torch.cat(parts).to(s["q"].dtype)}


def _plain_product(s: dict) -> torch.Tensor:
    """x W^T in fp32."""
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=-1).flatten(1)  # [n, k]
    w = codes.float().unflatten(1, (-1, s["case"]["group"]))
    w = ((w - s["zeros"].float()[..., None]) * s["scales"].float()[..., None]).flatten(1)
    return torch.matmul(s["x"].float(), w.t())


def _run_linear(s: dict) -> dict:
    if own:
        from kvserve_amd import linear4

        return {"y": linear4(s["x"], s["weight"])}
    return {"y": _plain_product(s).to(s["x"].dtype)}


def _run_mlp(s: dict) -> dict:
    if own:
        from kvserve_amd import linear4_silu_mul

        return {"y": linear4_silu_mul(s["x"], s["weight"])}
    gate, up = _plain_product(s).chunk(2, dim=-1)
    return {"y": (gate / (1 + torch.exp(-gate)) * up).to(s["x"].dtype)}


# -- from the definitions, in 64 bits --------------------------------------------------------------


def _exact_rope(case: dict, seed: int) -> dict:
    s = _prepare_rope(case, seed)
    H, Hkv, D = SHAPES[case["model"]]
    R = case["rotary"]
    heads = s["qkv"].double().view(case["tokens"], -1, D)
    angles = (s["cos"].double()[s["positions"]].unsqueeze(1), s["sin"].double()[s["positions"]].unsqueeze(1))

    def turned(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * weight.double()
        i = torch.arange(R // 2, device=DEVICE)
        lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
        y = x.clone()
        y[..., lo] = angles[0] * x[..., lo] - angles[1] * x[..., hi]
        y[..., hi] = angles[1] * x[..., lo] + angles[0] * x[..., hi]
        return y

    out = {"q": turned(heads[:, :H], s["q_norm"])}
    for name, rows in (("k_cache", turned(heads[:, H : H + Hkv], s["k_norm"])), ("v_cache", heads[:, H + Hkv :])):
        flat = s[name].double().flatten(0, 1)
        flat[s["slots"]] = rows
        out[name] = flat.view(s[name].shape)
    return out


def _exact_attend(case: dict, seed: int):
    q, ctx = _lengths(case)
    if sum(n * (n + c) for n, c in zip(q, ctx)) * case["heads"] * case["head_dim"] > 2e12:
        return None
    s = _prepare_attend(case, seed)
    G, bs, tables = case["heads"] // case["kv_heads"], case["block"], s["meta"].block_tables
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    t0 = 0
    for i, (n, have) in enumerate(zip(q, ctx)):
        pages = tables[i, : -(-(n + have) // bs)]
        k, v = (x.view(torch.uint8)[pages].view(x.dtype).float().flatten(0, 1)[: n + have].double() for x in (s["k"], s["v"]))
        if case["cache"] == "e4m3":
            k, v = k * K_SCALE, v * V_SCALE
        ahead = torch.arange(n + have, device=DEVICE) - (have + torch.arange(n, device=DEVICE))[:, None]  # key - query
        hidden = (ahead > 0) | ((ahead <= -case["window"]) & (torch.arange(n + have, device=DEVICE) >= case["sinks"]))
        for h in range(case["heads"]):
            kt = k[:, h // G].t().contiguous()
            w = (s["q"][t0 : t0 + n, h].double().contiguous() @ kt) * s["scale"]
            out[t0 : t0 + n, h] = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // G].contiguous()
        t0 += n
    return {"out": out}


def _exact_product(case: dict, seed: int) -> torch.Tensor:
    s = _prepare_linear(case, seed)
    x, y = s["x"].double(), torch.empty((case["rows"], case["n"]), dtype=torch.float64, device=DEVICE)
    group = torch.arange(case["k"], device=DEVICE) // case["group"]
    for r in range(0, case["n"], 2048):
        w = torch.empty((min(2048, case["n"] - r), case["k"]), dtype=torch.float64, device=DEVICE)
        w[:, 0::2] = (s["codes"][r : r + 2048] % 16).double()
        w[:, 1::2] = (s["codes"][r : r + 2048] // 16).double()
        w = (w - s["zeros"][r : r + 2048].double()[:, group]) * s["scales"][r : r + 2048].double()[:, group]
        y[:, r : r + 2048] = x @ w.t().contiguous()
    return y


def _exact_linear(case: dict, seed: int) -> dict:
    return {"y": _exact_product(case, seed)}


def _exact_mlp(case: dict, seed: int) -> dict:
    y = _exact_product(case, seed)
    gate, up = y[:, : case["n"] // 2], y[:, case["n"] // 2 :]
    return {"y": gate * torch.sigmoid(gate) * up}


# -- what a pass cannot do without -----------------------------------------------------------------


def _work_rope(case: dict) -> dict:
    H, Hkv, D = SHAPES[case["model"]]
    T, R = case["tokens"], case["rotary"]
    # the projection in, its rows out, a table row per token, the norms' weights, positions and slots
    return {"bytes": 2 * T * (H + 2 * Hkv) * D * 2 + T * (R * 4 + 16) + 4 * D, "flops": T * (H + Hkv) * (4 * D + 3 * R)}


def _work_attend(case: dict) -> dict:
    q, ctx = _lengths(case)
    H, Hkv, D, W, S = (case[n] for n in ("heads", "kv_heads", "head_dim", "window", "sinks"))

    def upto(p: int) -> int:
        """Keys that the tokens at positions 0 .. p - 1 see, all told."""
        return p * (p + 1) // 2 if p <= W + S else (W + S) * (W + S + 1) // 2 + (p - W - S) * (W + S)

    keys = sum(min(n + c, W + n - 1 + S) for n, c in zip(q, ctx))  # rows that some token of a sequence sees
    seen = sum(upto(n + c) - upto(c) for n, c in zip(q, ctx))
    eb = 1 if case["cache"] == "e4m3" else 2
    return {"bytes": 2 * Hkv * D * eb * keys + 2 * sum(q) * H * D * 2 + 8 * (keys // case["block"] + 2 * len(q) + 1),
            "flops": 4 * H * D * seen}  # fmt: skip


def _work_linear(case: dict) -> dict:
    m, n, k, groups = case["rows"], case["n"], case["k"], case["k"] // case["group"]
    out = n // 2 if case["kind"] == "mlp" else n
    return {"bytes": n * k // 2 + n * groups * 3 + 2 * m * (k + out), "flops": 2 * m * n * k}


# -- the cases' common face ------------------------------------------------------------------------


_KINDS = {
    "rope": (_prepare_rope, _run_rope, _exact_rope, _work_rope),
    "attend": (_prepare_attend, _run_attend, _exact_attend, _work_attend),
    "linear": (_prepare_linear, _run_linear, _exact_linear, _work_linear),
    "mlp": (_prepare_linear, _run_mlp, _exact_mlp, _work_linear),
}


def prepare(case: dict, seed: int) -> dict:
    return _KINDS[case["kind"]][0](case, seed)


def run(state: dict):
    return _KINDS[state["case"]["kind"]][1](state)


def exact(case: dict, seed: int):
    return _KINDS[case["kind"]][2](case, seed)


def work(case: dict) -> dict:
    return _KINDS[case["kind"]][3](case)
