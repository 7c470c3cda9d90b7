"""The operators over a KV cache held in 4 bits, and the log probabilities of given tokens, as they are timed.

  write    `HipAttention.write_kv` of a step's K and V rows into a 4-bit cache, and `read_kv` of the same slots
           (what attention will see of them).
  rope     `HipAttention.rope_and_cache` of a step's fused projection into a 4-bit cache, and `read_kv`.
  read     `HipAttention.read_kv`: the rows of a cached prefix as 16-bit values.
  attend   `HipAttention.forward` over a 4-bit cache: decoding sequences, drafts to verify, prompt chunks.
  logprobs `token_logprobs`: log probability and entropy per row of logits, with the k largest alternatives.

The cache format is MXFP4: E2M1 elements two to a byte (element 2i in the low half) and one power of two (E8M0) for
every 32 consecutive elements of a row. `run` computes each operator in elementary torch operations where `own` is
false, and calls the framework's operators where it is true.

Sizes are those of the two Llama shapes the engine is configured for (1B: 32 query heads over 8 kv heads of 64; 8B: 32
over 8 of 128; both 128256 tokens of vocabulary) and of the benchmark's workloads. Lengths follow from the case alone,
values and physical block orders from the seed.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32  # elements of a row that share a scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SHAPES = {"1b": (32, 8, 64), "8b": (32, 8, 128)}  # query heads, kv heads, head size


# -- the cases -------------------------------------------------------------------------------------


def _attend(name: str | None = None, **kw) -> dict:
    """`decodes` sequences of `q` query tokens over lo .. hi cached tokens, then `chunks` sequences computing chunk_lo ..
    chunk_hi prompt tokens over ctx_lo .. ctx_hi cached ones. `pages`: whether a page holds each head's tokens
    together ("head") or each token's heads ("token")."""
    c = {
        "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16, "pages": "head",
        "decodes": 0, "q": 1, "lo": 0, "hi": 0, "chunks": 0, "chunk_lo": 0, "chunk_hi": 0, "ctx_lo": 0, "ctx_hi": 0,
        "lens": 0,
    }  # fmt: skip
    c.update(kw)
    return {"name": name, **c} if name else c


def listed() -> list[dict]:
    return [
        # the rows of one decode step of a small model, eight users: the smallest call
        {"name": "write_1b_b8", "kind": "write", "model": "1b", "dtype": "bf16", "tokens": 8, "pages": "head"},
        # the rows of a full step of prompts and decodes
        {"name": "write_8b_2048", "kind": "write", "model": "8b", "dtype": "bf16", "tokens": 2048, "pages": "head"},
        # a decode step's projection, an odd number of users, fp16, pages in the 16-bit caches' order
        {"name": "rope_1b_33_fp16", "kind": "rope", "model": "1b", "dtype": "fp16", "tokens": 33, "pages": "token"},
        # a full step's projection rotated and written
        {"name": "rope_8b_2048", "kind": "rope", "model": "8b", "dtype": "bf16", "tokens": 2048, "pages": "head"},
        # a short cached prefix handed to something that takes 16 bits
        {"name": "read_1b_777_fp16", "kind": "read", "model": "1b", "dtype": "fp16", "tokens": 777, "pages": "token"},
        # a long document's keys and values handed over
        {"name": "read_8b_32768", "kind": "read", "model": "8b", "dtype": "bf16", "tokens": 32768, "pages": "head"},
        # a small model answering a few short chats: bound by launches and latency
        _attend("decode_1b_b8", head_dim=64, decodes=8, lo=63, hi=511),
        # a busy server's decode step over long contexts
        _attend("decode_8b_b64", decodes=64, lo=1023, hi=8191),
        # speculative decoding: five draft tokens verified per sequence
        _attend("verify_8b_b32_q5_fp16", dtype="fp16", decodes=32, q=5, lo=2048, hi=4096),
        # a continuous-batching step: decodes, and chunks of two long prompts over what is cached (the most arithmetic)
        _attend("mixed_8b", decodes=24, lo=255, hi=4095, chunks=2, chunk_lo=900, chunk_hi=1024, ctx_lo=4000, ctx_hi=10000),
        # a decode step's sampled tokens with the five likeliest alternatives
        {"name": "logprobs_b8_top5", "kind": "logprobs", "dtype": "bf16", "rows": 8, "vocab": 128256, "top": 5},
        # a prompt scored, with the twenty likeliest alternatives at each place
        {"name": "logprobs_1023_top20", "kind": "logprobs", "dtype": "bf16", "rows": 1023, "vocab": 128256, "top": 20},
    ]  # fmt: skip


def _log(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5)))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["write", "rope", "read", "decode", "decode", "verify", "mixed", "chunks", "logprobs", "logprobs"])
    pages = rng.choice(["head", "head", "token"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind in ("write", "rope", "read"):
        return {"kind": kind, "model": rng.choice(["1b", "8b"]), "dtype": dtype,
                "tokens": _log(rng, 1, 32768 if kind == "read" else 4096), "pages": pages}  # fmt: skip
    if kind == "logprobs":
        vocab = rng.choice([128256, _log(rng, 257, 160000)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "vocab": vocab,
                "rows": _log(rng, 1, min(2048, 65_000_000 // vocab)), "top": rng.choice([0, 1, 5, rng.randint(2, 20)])}  # fmt: skip
    c = {"dtype": dtype, "head_dim": rng.choice([64, 128, 128]), "block": rng.choice([16, 16, 32]), "pages": pages,
         "lens": rng.randrange(1 << 20)}  # fmt: skip
    c["heads"], c["kv_heads"] = rng.choice([(32, 8), (32, 8), (32, 8), (32, 4), (16, 16)])
    most = 2_000_000 // c["kv_heads"]  # cached tokens of a batch at most
    if kind in ("decode", "verify"):
        n = _log(rng, 1, 256)
        hi = min(_log(rng, 64, 16384), most // n)
        c.update(decodes=n, q=1 if kind == "decode" else rng.randint(2, 8), lo=rng.randint(1, hi), hi=hi)
    else:
        if kind == "mixed":
            n = _log(rng, 1, 48)
            hi = min(_log(rng, 64, 8192), most // n)
            c.update(decodes=n, lo=rng.randint(1, hi), hi=hi)
        c.update(chunks=_log(rng, 1, 4), ctx_hi=rng.choice([0, _log(rng, 1, 9000)]))
        c["chunk_hi"] = _log(rng, 20, 1500)
        pairs = 12_000_000 // c["chunks"]  # (query, key) pairs of a sequence at most
        c["chunk_hi"] = max(20, min(c["chunk_hi"], pairs // (c["ctx_hi"] + c["chunk_hi"])))
        c["chunk_lo"] = rng.randint(20, c["chunk_hi"])
    return _attend(**c)


# -- the format ------------------------------------------------------------------------------------


def _largest(dtype: torch.dtype) -> float:
    """The largest value that both the format and a row's type hold."""
    return 1.5 * 2.0 ** (15 if dtype == torch.float16 else 127)


def _quantise(x: torch.Tensor, largest: float) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows [..., D] as E2M1 bytes [..., D / 2] and E8M0 bytes [..., D / 32]."""
    x = x.clamp(-largest, largest).unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1, keepdim=True)
    # the exponent under which nothing is off by more than half a step: one more from a mantissa of 1.75 on
    s = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 253)
    y = x * ((254 - s) << 23).view(torch.float32)  # x / 2^(s - 127), exact
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)  # ties go to the even code
    for i, edge in enumerate((0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > edge) if i % 2 else (a >= edge)
    code |= torch.signbit(x).to(torch.uint8) << 3
    code = code.flatten(-2)
    s = torch.where(top.isnan(), 255, s).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), s


def _values(code: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """The fp32 values [..., D] of E2M1 bytes [..., D / 2] with E8M0 bytes [..., D / 32]."""
    one = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=code.device)
    pair = torch.stack((one.repeat(16), one.repeat_interleave(16)), dim=1)  # of a byte
    x = pair[code.int()].flatten(-2)
    f = (s.int() << 23).view(torch.float32).masked_fill(s == 255, math.nan)
    return (x.unflatten(-1, (-1, BLOCK)) * f.unsqueeze(-1)).flatten(-2)


# -- inputs ----------------------------------------------------------------------------------------


def _normal(gen: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _channels(gen: torch.Generator, kv_heads: int, head_dim: int) -> torch.Tensor:
    """Keys have channels that are larger than others by a factor, the same for every token."""
    return torch.exp(0.7 * _normal(gen, kv_heads, head_dim))


def _pool(blocks: int, block: int, kv_heads: int, width: int, pages: str) -> torch.Tensor:
    """Zero bytes of shape [blocks, block, kv_heads, width], each head's (or each token's) together in a page."""
    if pages == "token":
        return torch.zeros((blocks, block, kv_heads, width), dtype=torch.uint8, device=DEVICE)
    return torch.zeros((blocks, kv_heads, block, width), dtype=torch.uint8, device=DEVICE).permute(0, 2, 1, 3)


def _caches(gen: torch.Generator, blocks: int, block: int, kv_heads: int, head_dim: int, pages: str, filled: bool) -> dict:
    """K and V bytes with their scales, as earlier steps left them (`filled`) or zeros."""
    c = {}
    for name in ("k", "v"):
        c[name] = _pool(blocks, block, kv_heads, head_dim // 2, pages)
        c[name + "_scale"] = _pool(blocks, block, kv_heads, head_dim // BLOCK, pages)
        factor = _channels(gen, kv_heads, head_dim) if name == "k" else 1.0
        step = max(1, (1 << 25) // (block * kv_heads * head_dim))
        for b in range(0, blocks if filled else 0, step):
            n = min(step, blocks - b)
            code, s = _quantise(_normal(gen, n, block, kv_heads, head_dim) * factor, _largest(torch.bfloat16))
            c[name][b : b + n], c[name + "_scale"][b : b + n] = code, s
    return c


def _typed(c: dict) -> dict:
    """The arguments k_cache, v_cache, k_scale, v_scale of the framework's calls: the same memory under its types."""
    return {
        "k_cache": c["k"].view(torch.float4_e2m1fn_x2), "v_cache": c["v"].view(torch.float4_e2m1fn_x2),
        "k_scale": c["k_scale"].view(torch.float8_e8m0fnu), "v_scale": c["v_scale"].view(torch.float8_e8m0fnu),
    }  # fmt: skip


def _prepare_rows(case: dict, seed: int) -> dict:
    """A step's tokens: consecutive positions of one prompt, in pages of a shuffled pool."""
    H, Hkv, D = SHAPES[case["model"]]
    T, bs = case["tokens"], 16
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    blocks = -(-T // bs) + 4
    order = list(range(blocks))
    random.Random(seed).shuffle(order)
    table = torch.tensor(order, device=DEVICE)
    at = torch.arange(T, device=DEVICE)
    c = _caches(gen, blocks, bs, Hkv, D, case["pages"], case["kind"] == "read")
    s = {"case": case, "caches": c, "args": _typed(c), "slots": table[at // bs] * bs + at % bs, "heads": H,
         "dtype": DTYPES[case["dtype"]]}  # fmt: skip
    if case["kind"] == "read":
        return s
    qkv = _normal(gen, T, H + 2 * Hkv, D)
    qkv[:, H : H + Hkv] *= _channels(gen, Hkv, D)
    s["qkv"] = qkv.to(s["dtype"]).flatten(1)
    if case["kind"] == "write":  # k and v as a layer hands them over: v a view of the fused projection's rows
        s["k"] = s["qkv"][:, H * D : (H + Hkv) * D].unflatten(1, (Hkv, D)).contiguous()
        s["v"] = s["qkv"][:, (H + Hkv) * D :].unflatten(1, (Hkv, D))
        return s
    start = T * random.Random(seed + 1).randint(0, 3)
    angle = torch.arange(4 * T, device=DEVICE).double()[:, None] * 500000.0 ** -(
        torch.arange(0, D, 2, device=DEVICE).double() / D
    )
    s["cos"], s["sin"] = (f(angle).float().repeat(1, 2) for f in (torch.cos, torch.sin))
    s["positions"] = at + start
    return s


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
    c = _caches(gen, blocks, bs, Hkv, D, case["pages"], True)
    # what the calls read of a step's metadata, under the names it has there
    meta = SimpleNamespace(
        block_tables=tables.to(DEVICE), seq_lens=torch.tensor([n + c for n, c in zip(q, ctx)], device=DEVICE),
        query_start_loc=torch.tensor(starts, device=DEVICE), max_query_len=max(q),
        max_seq_len=max(n + c for n, c in zip(q, ctx)),
    )  # fmt: skip
    return {"case": case, "caches": c, "args": _typed(c), "meta": meta, "scale": D**-0.5,
            "q": _normal(gen, starts[-1], H, D).to(DTYPES[case["dtype"]])}  # fmt: skip


def _prepare_logprobs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    T, V = case["rows"], case["vocab"]
    logits = torch.empty((T, V), dtype=DTYPES[case["dtype"]], device=DEVICE)
    tokens = torch.empty(T, dtype=torch.long, device=DEVICE)
    for r in range(0, T, 128):
        x = 2.0 * _normal(gen, min(128, T - r), V)
        # a few likely words in each row, from nearly certain to one among many
        near = torch.randint(V, (len(x), 8), generator=gen, device=DEVICE)
        x.scatter_add_(1, near, 6.0 + 4.0 * _normal(gen, len(x), 8))
        logits[r : r + 128] = x
        gumbel = -torch.log(torch.empty_like(x).exponential_(generator=gen))
        tokens[r : r + 128] = (x + gumbel).argmax(1)
    return {"case": case, "logits": logits, "tokens": tokens, "top": case["top"]}


# -- one pass --------------------------------------------------------------------------------------


def _store(c: dict, name: str, rows: torch.Tensor, slots: torch.Tensor, largest: float) -> None:
    code, s = _quantise(rows, largest)
    bs = c[name].shape[1]
    c[name][slots // bs, slots % bs] = code
    c[name + "_scale"][slots // bs, slots % bs] = s


def _fetch(c: dict, name: str, slots: torch.Tensor) -> torch.Tensor:
    bs = c[name].shape[1]
    return _values(c[name][slots // bs, slots % bs], c[name + "_scale"][slots // bs, slots % bs])


def _read(s: dict) -> dict:
    if own:
        from kvserve_amd import HipAttention

        k, v = HipAttention.read_kv(s["args"]["k_cache"], s["args"]["v_cache"], s["slots"], s["dtype"],
                                    s["args"]["k_scale"], s["args"]["v_scale"])  # fmt: skip
        return {"k": k, "v": v}
    return {n: _fetch(s["caches"], n, s["slots"]).to(s["dtype"]) for n in ("k", "v")}


def _write(s: dict) -> dict:
    if own:
        from kvserve_amd import HipAttention

        HipAttention.write_kv(k=s["k"], v=s["v"], slots=s["slots"], **s["args"])
    else:
        for n in ("k", "v"):
            _store(s["caches"], n, s[n].float(), s["slots"], _largest(s["dtype"]))
    return _read(s)


def _rope(s: dict) -> dict:
    if own:
        from kvserve_amd import HipAttention

        q = HipAttention.rope_and_cache(s["qkv"], s["positions"], s["cos"], s["sin"], slots=s["slots"],
                                        num_heads=s["heads"], **s["args"])  # fmt: skip
    else:
        H, (Hkv, half) = s["heads"], (s["caches"]["k"].shape[2], s["caches"]["k"].shape[3])
        x = s["qkv"].float().unflatten(1, (-1, 2 * half))
        cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
        rot, v = x[:, : H + Hkv], x[:, H + Hkv :]
        rot = rot * cos + torch.cat((-rot[..., half:], rot[..., :half]), dim=-1) * sin
        q = rot[:, :H].to(s["dtype"])
        _store(s["caches"], "k", rot[:, H:], s["slots"], _largest(s["dtype"]))
        _store(s["caches"], "v", v, s["slots"], _largest(s["dtype"]))
    return {"q": q, **_read(s)}


def _softmax_av(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor, scale: float) -> torch.Tensor:
    """q [n, Hkv, R, D] over k, v [n, Hkv, L, D] where seen [n, 1, R, L]; rows that see nothing give zeros."""
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp_(p.sub_(top.masked_fill(top == -math.inf, 0.0)))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _plain_group(s: dict, first: int, last: int, longest: int) -> torch.Tensor:
    """Attention of sequences first .. last - 1 as one batch padded to `longest` query tokens: [n, longest, H, D]."""
    meta, c = s["meta"], s["caches"]
    H, Hkv = s["case"]["heads"], s["case"]["kv_heads"]
    G = H // Hkv
    tables = meta.block_tables[first:last]
    lens, begin = meta.seq_lens[first:last], meta.query_start_loc[first:last]
    n_q = meta.query_start_loc[first + 1 : last + 1] - begin
    at = torch.arange(longest, device=DEVICE)
    rows = s["q"][(begin[:, None] + at).clamp(max=len(s["q"]) - 1)].float()  # [n, longest, H, D]
    n, D = len(tables), rows.shape[-1]
    q = rows.view(n, longest, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(n, Hkv, longest * G, D)
    limit = (lens - n_q)[:, None] + at + 1  # keys that a query token sees
    limit = torch.where(at < n_q[:, None], limit, 0).repeat_interleave(G, dim=1)[:, None, :, None]
    L = tables.shape[1] * c["k"].shape[1]
    seen = torch.arange(L, device=DEVICE) < limit
    k, v = (_values(c[m][tables], c[m + "_scale"][tables]).flatten(1, 2).transpose(1, 2) for m in ("k", "v"))
    inside = (torch.arange(L, device=DEVICE) < lens[:, None])[:, None, :, None]
    out = _softmax_av(q, k, v.masked_fill(~inside, 0.0), seen, s["scale"])
    return out.view(n, Hkv, longest, G, D).permute(0, 2, 1, 3, 4).reshape(n, longest, H, D)


def _attention(s: dict) -> dict:
    if own:
        from kvserve_amd import HipAttention

        return {"out": HipAttention.forward(s["q"], meta=s["meta"], scale=s["scale"], **s["args"])}
    case, n_dec = s["case"], s["case"]["decodes"]
    parts = []
    if n_dec:
        parts.append(_plain_group(s, 0, n_dec, case["q"]).flatten(0, 1))
    if case["chunks"]:
        out = _plain_group(s, n_dec, n_dec + case["chunks"], case["chunk_hi"])
        n_q = s["meta"].query_start_loc.diff()[n_dec:]
        keep = torch.arange(case["chunk_hi"], device=DEVICE) < n_q[:, None]
        parts.append(out[keep])
    return {"out": torch.cat(parts).to(s["q"].dtype)}


def _logprobs(s: dict) -> dict:
    if own:
        from kvserve_amd import token_logprobs

        r = token_logprobs(s["logits"], s["tokens"], s["top"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    mean = (e * (x - top).masked_fill(x == -math.inf, 0.0)).sum(-1, keepdim=True) / total
    # the largest first, ties to the lowest id: the value's place in the order of fp32, then the id from the end
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key += x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device)
    ids = x.shape[1] - 1 - (torch.topk(key, s["top"], dim=-1).values & 0xFFFFFFFF)
    return {"logprobs": (x.gather(1, s["tokens"][:, None]) - lse).squeeze(1),
            "entropy": (torch.log(total) - mean).squeeze(1), "top_logprobs": x.gather(1, ids) - lse, "top_ids": ids}  # fmt: skip


# -- from the definitions, in 64 bits --------------------------------------------------------------


def _power64(e: torch.Tensor) -> torch.Tensor:
    """2^e from its bits: exact, as torch.ldexp on a GPU is not."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored64(x: torch.Tensor, largest: float) -> torch.Tensor:
    """What the format keeps of 64-bit rows: the nearest value of the block's grid, ties to the even code."""
    x = x.clamp(-largest, largest).unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # the maximum is m 2^e, m in [0.5, 1)
    unit = _power64((e - 3 + (m >= 0.875).to(e.dtype)).clamp(-125, 126))
    y = (x / unit).abs()
    # the step of the grid at y: 0.5 below 2, 1 below 4, 2 from there
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return ((torch.round(y / step) * step).clamp(max=6.0) * unit * torch.sign(x)).flatten(-2)


def _decoded64(code: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """The values of E2M1 bytes in 64 bits, from sign, exponent and mantissa bits."""
    nib = torch.stack((code & 15, code >> 4), dim=-1).flatten(-2).to(torch.int16)
    e, m = (nib >> 1) & 3, (nib & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * _power64((e - 1).clamp(min=0)))
    val = torch.where(nib >= 8, -mag, mag)
    return val * _power64(s.int() - 127).repeat_interleave(BLOCK, -1)


def _exact_rows(case: dict, seed: int) -> dict:
    s = _prepare_rows(case, seed)
    H, Hkv, D = SHAPES[case["model"]]
    if case["kind"] == "read":
        blk, off = s["slots"] // 16, s["slots"] % 16
        c = s["caches"]
        return {n: _decoded64(c[n][blk, off], c[n + "_scale"][blk, off]) for n in ("k", "v")}
    x = s["qkv"].double().unflatten(1, (-1, D))
    q, k, v = x.split([H, Hkv, Hkv], dim=1)
    out = {}
    if case["kind"] == "rope":
        c, w = (s[n][s["positions"]].double()[:, None, : D // 2] for n in ("cos", "sin"))

        def turn(a: torch.Tensor) -> torch.Tensor:
            lo, hi = a.chunk(2, dim=-1)
            return torch.cat((lo * c - hi * w, hi * c + lo * w), dim=-1)

        q, k = turn(q), turn(k)
        out["q"] = q
    return {**out, "k": _stored64(k, _largest(s["dtype"])), "v": _stored64(v, _largest(s["dtype"]))}


def _exact_attend(case: dict, seed: int):
    q, ctx = _lengths(case)
    if sum(n * (n + c) for n, c in zip(q, ctx)) * case["heads"] * case["head_dim"] > 2e12:
        return None
    s = _prepare_attend(case, seed)
    c, tables, bs = s["caches"], s["meta"].block_tables, case["block"]
    G = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    t0 = 0
    for i, (n, have) in enumerate(zip(q, ctx)):
        pages = tables[i, : -(-(n + have) // bs)]
        k, v = (_decoded64(c[m][pages], c[m + "_scale"][pages]).flatten(0, 1)[: n + have] for m in ("k", "v"))
        later = torch.arange(n + have, device=DEVICE) > have + torch.arange(n, device=DEVICE)[:, None]
        for h in range(case["heads"]):
            kt = k[:, h // G].t().contiguous()
            w = (s["q"][t0 : t0 + n, h].double().contiguous() @ kt) * s["scale"]
            out[t0 : t0 + n, h] = torch.softmax(w.masked_fill(later, -math.inf), dim=-1) @ v[:, h // G].contiguous()
        t0 += n
    return {"out": out}


def _exact_logprobs(case: dict, seed: int) -> dict:
    s = _prepare_logprobs(case, seed)
    got: dict[str, list] = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_ids": []}
    for x, tok in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = x.double()
        lp = torch.log_softmax(x, dim=-1)
        got["logprobs"].append(lp.gather(1, tok[:, None]).squeeze(1))
        got["entropy"].append(-(lp.exp() * lp).nan_to_num(0.0).sum(-1))
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
        got["top_logprobs"].append(lp.gather(1, order))
        got["top_ids"].append(order)
    return {n: torch.cat(parts) for n, parts in got.items()}


# -- what a pass cannot do without -----------------------------------------------------------------


def _work_rows(case: dict) -> dict:
    H, Hkv, D = SHAPES[case["model"]]
    T, eb = case["tokens"], DTYPES[case["dtype"]].itemsize
    packed, wide = 2 * T * Hkv * (D // 2 + D // BLOCK), 2 * T * Hkv * D * eb
    if case["kind"] == "read":
        return {"bytes": packed + wide + 8 * T, "flops": 2 * T * Hkv * D}
    # the rows in, the packed rows out, and the rows as read back
    n = {"bytes": wide + packed + wide + 8 * T, "flops": 8 * T * Hkv * D}
    if case["kind"] == "rope":
        n["bytes"] += T * (2 * H * D * eb + 2 * D * 4 + 8)
        n["flops"] += 3 * T * (H + Hkv) * D
    return n


def _work_attend(case: dict) -> dict:
    q, ctx = _lengths(case)
    H, Hkv, D, T = case["heads"], case["kv_heads"], case["head_dim"], sum(q)
    blocks = sum(-(-(n + c) // case["block"]) for n, c in zip(q, ctx))
    seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(q, ctx))
    return {"bytes": 2 * Hkv * (D // 2 + D // BLOCK) * (sum(ctx) + T) + 2 * T * H * D * 2 + 8 * (blocks + 2 * len(q) + 1),
            "flops": 4 * H * D * seen}  # fmt: skip


def _work_logprobs(case: dict) -> dict:
    T, V, eb = case["rows"], case["vocab"], DTYPES[case["dtype"]].itemsize
    return {"bytes": T * (V * eb + 8 + 8 + 12 * case["top"]), "flops": 5 * T * V}


# -- the cases' common face ------------------------------------------------------------------------


_KINDS = {
    "write": (_prepare_rows, _write, _exact_rows, _work_rows),
    "rope": (_prepare_rows, _rope, _exact_rows, _work_rows),
    "read": (_prepare_rows, _read, _exact_rows, _work_rows),
    "attend": (_prepare_attend, _attention, _exact_attend, _work_attend),
    "logprobs": (_prepare_logprobs, _logprobs, _exact_logprobs, _work_logprobs),
}


def prepare(case: dict, seed: int) -> dict:
    return _KINDS[case["kind"]][0](case, seed)


def run(state: dict):
    return _KINDS[state["case"]["kind"]][1](state)


def exact(case: dict, seed: int):
    return _KINDS[case["kind"]][2](case, seed)


def work(case: dict) -> dict:
    return _KINDS[case["kind"]][3](case)
